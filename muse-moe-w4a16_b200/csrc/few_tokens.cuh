// Launch interface of the few-token products (few_tokens.cu).
#pragma once

#include "w4.cuh"

namespace muse {

// The most tokens of these calls.
constexpr int kFewTokens = 32;
// A forward product of 16-bit weights [n, k] that is streamed: few tokens, or a weight so small that the
// other kernel's second launch for its split K costs more than it gains (24 x 2048 x 768 block: 16.4
// against 19.6 us a call; 32 x 7168 x 2048: 28.8 against 23.5).
inline bool streams_dense(int tokens, int n, int k) {
  return tokens <= 8 || (tokens <= kFewTokens && (long long)n * k <= (8LL << 20));
}
// A product with an NVFP4 weight that is streamed: likewise (24 x 4096 x 4096: 10.4 against 11.7 us, 17 x
// 7168 x 4096: 15.6 against 13.8).
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
