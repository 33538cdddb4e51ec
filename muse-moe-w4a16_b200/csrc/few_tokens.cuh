// Launch interface of the few-token products (few_tokens.cu).
#pragma once

#include "w4.cuh"

namespace muse {

// The most tokens of these calls.
constexpr int kFewTokens = 32;
// A forward product of 16-bit weights [n, k] that is streamed: few tokens, or a small weight, where set-up
// and exchange cost the tensor-core kernels more than the stream's mma.sync does. Device times of whole
// blocks, both products streamed / both on the tensor cores, us:
//   block           8 tokens     9            16           17           32
//   2048 x 768      8.3 / 12.6   10.5 / 12.7  11.6 / 12.7  12.2 / 12.7  14.2 / 12.7
//   4096 x 1024     10.5 / 14.3  13.4 / 14.3  14.2 / 14.2  15.9 / 14.3  17.8 / 14.3
//   4096 x 2048     15.1 / 19.3  19.2 / 19.3  18.5 / 19.0  19.9 / 19.1  19.7 / 19.1
//   7168 x 2048     19.6 / 24.3  22.3 / 24.3  22.4 / 24.4  25.6 / 24.4  27.1 / 24.5
// From 9 to 16 tokens the stream is level or ahead at all of these, from 17 on behind at most: one limit
// for both, which costs up to a quarter where it is farthest off (4096 x 1024 at 32 tokens).
inline bool streams_dense(int tokens, int n, int k) {
  return tokens <= 8 || (tokens <= kFewTokens && (long long)n * k <= (8LL << 20));
}
// A product with an NVFP4 weight that is streamed: likewise (streamed / tensor cores, us on the device):
//   rows x columns  8 tokens    16           17           32
//   2048 x 2048     4.1 / 8.5   6.0 / 8.5    6.3 / 8.5    7.0 / 8.6
//   4096 x 4096     7.4 / 10.4  9.8 / 10.4   10.3 / 10.4  10.6 / 10.4
//   5120 x 4096     8.8 / 12.7  11.6 / 12.7  14.3 / 12.7  15.8 / 12.8
//   8192 x 7168     13.1 / 20.1 17.0 / 20.1  22.5 / 20.2  23.7 / 20.2
// Above 16 tokens they cross between 16 and 20 M codes.
inline bool streams_w4(int tokens, int rows, int cols) {
  return tokens <= 16 || (tokens <= kFewTokens && (long long)rows * cols <= (20LL << 20));
}

struct FewArgs {
  const uint8_t* wq;      // NVFP4: prepared tiles and the global scale
  const float* gs;
  const uint16_t* add;
  long long ld_add;
  uint16_t* out;
  long long ldo;
  float* ab;              // gated 16-bit weights: pre-activations to keep, or null
  int tokens, n_out, up_row;
  int stages;             // stages of K: 128 codes or 64 16-bit columns
  int ranks, stages_per_rank, depth;  // cluster size, stages of one rank, ring depth
  uint32_t m16, m64;
  int* error_flag;
};

int launch_few_w4(const LinearArgs& l, int dtype, bool gated, int* error_flag, cudaStream_t st);
// A forward product of the feed-forward block (modes kStore and kGate, both operands along k).
int launch_few_dense(const DenseGemm& g, cudaStream_t st);

}  // namespace muse
