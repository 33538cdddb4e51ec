// In-register dequantisation of prepared NVFP4 code words (layout.cuh) and the launch interface
// of the many-token 4-bit product (swap_gemm.cu).
#pragma once

#include "dense.cuh"
#include "layout.cuh"
#include "ptx.cuh"

namespace muse {

// A prepared tile: 128 rows' codes of 128 k, then their scales.
constexpr int kLinearTileBytes = kTileCodeBytes + kTileScaleBytes;

struct LinearArgs {
  const uint8_t* wq;         // prepared tiles
  const float* gs;
  const uint16_t* x;
  long long ldx;
  const uint16_t* add;
  long long ld_add;
  uint16_t* out;
  long long ldo;
  float* ab;                 // gated 16-bit weights: fp32 pre-activations to keep, [tokens, 2 n_out], or null
  int tokens, cols, n_out;   // n_out: columns of y
  int k_chunks;              // 128-code chunks of K
  int padded_rows;           // weight rows, padded to 128
  uint32_t m16, m64;         // 16 and 64 (see dequant_word)
};

// The product for more than a few tokens, and how it runs.
int launch_linear_gemm(const LinearArgs& a, int dtype, bool gated, int* error_flag, cudaStream_t st);
PlanInfo linear_gemm_plan(int tokens, int padded_rows, int k_chunks);

__device__ __forceinline__ uint32_t mul2_bf16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t mul2_f16(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Two e4m3 scales -> a pair register per scale. bf16: (s * 2^118, twice); fp16: (s * 2^5, twice).
// Exact: four significant bits, and 448 * 2^118 and 448 * 2^5 are in range.
template <bool kHalf>
__device__ __forceinline__ void expand_scales(uint32_t two, uint32_t& s0, uint32_t& s1) {
  uint32_t h;
  asm("{\n\t.reg .b16 t;\n\tcvt.u16.u32 t, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
  if (kHalf) {
    const uint32_t v = mul2_f16(h, 0x50005000u);  // 2^5
    s0 = __byte_perm(v, v, 0x1010);
    s1 = __byte_perm(v, v, 0x3232);
  } else {
    const float2 f = unpack16(kFp16, h);
    constexpr float kUp = 332306998946228968225951765070086144.0f;  // 2^118
    s0 = pack16(kBf16, f.x * kUp, f.x * kUp);
    s1 = pack16(kBf16, f.y * kUp, f.y * kUp);
  }
}

// One permuted code word -> four pairs (natural element order) times the scale register.
// The masked bits read as bf16 are e2m1 * 2^-126; with the scale the result is e2m1 * e4m3 * 2^-8,
// six significant bits: exact. The logic pipe is the busiest one here, so two of the shifts are
// multiplies by m16 = 16 and m64 = 64, which the compiler cannot see. For fp16 the three magnitude bits move up by three (e2m1 * 2^-14);
// times s * 2^5, then times 2^9: e2m1 * e4m3, exact (every step is a multiple of 2^-24).
template <bool kHalf>
__device__ __forceinline__ void dequant_word(uint32_t w, uint32_t scale, uint32_t m16, uint32_t m64, uint32_t (&out)[4]) {
  constexpr uint32_t kMask = 0x81C081C0u;
  uint32_t v[4] = {w & kMask, (w * m16) & kMask, ptx::rotl(w, 10) & kMask,
                   ((w * m64) & 0x80C080C0u) | ((w >> 2) & 0x01000100u)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (kHalf) {
      const uint32_t u = (v[i] & 0x80008000u) | ((v[i] << 3) & 0x0E000E00u);
      out[i] = mul2_f16(mul2_f16(u, scale), 0x60006000u);  // 2^9
    } else {
      out[i] = mul2_bf16(v[i], scale);
    }
  }
}
template <bool kHalf> constexpr float kUnscale = kHalf ? 1.f : 256.f;
// The global scale, from L2: this kernel may have started before the one that writes it ended, which a
// load through the read-only path does not allow for.
template <bool kHalf>
__device__ __forceinline__ float load_scale(const float* gs) { return __ldcg(gs) * kUnscale<kHalf>; }

__device__ __forceinline__ uint16_t round16(int dtype, float v) { return (uint16_t)(pack16(dtype, v, v) & 0xFFFF); }
// (from L2: an addend may be the output that the kernel before wrote in place)
__device__ __forceinline__ float load16(int dtype, const uint16_t* p) {
  return unpack16(dtype, (uint32_t)__ldcg(p)).x;
}

}  // namespace muse
