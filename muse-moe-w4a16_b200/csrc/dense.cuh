// Internal interface of the dense 16-bit matrix products (dense_gemm.cu): the gated
// feed-forward block's forward and backward products.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "common.cuh"

namespace muse {

constexpr int kMaxRows = 1 << 28;   // tokens of one call

// Element type of a dense operator's tensors (the ABI's `dtype`).
enum DenseType : int { kBf16 = 0, kFp16 = 1 };

// One operand of D[m, n] = sum_k A[m, k] B[n, k], 16-bit, `ld` elements between rows of the
// memory. K-major: memory rows are m (or n) and run along k; else memory rows are k and run
// along m (or n) -- the transposed products of a backward pass, read in place.
struct DenseOperand {
  const void* ptr;
  long long ld;
  bool k_major;
};

// What becomes of the fp32 accumulators.
enum DenseMode : int {
  kStore,  // out[m, n] = acc (+ add[m, n]), 16-bit
  kGate,   // B holds gate rows [0, I) and up rows [I, 2I): out[m, i] = silu(a) * b, 16-bit, and
           // (if ab) ab[m, i] = a, ab[m, I + i] = b in fp32 for the backward pass
  kDGate,  // acc = dh: out[m, i] = da, out[m, I + i] = db, h_out[m, i] = silu(a) * b (16-bit), with
           // a, b read from ab
};

struct DenseGemm {
  DenseOperand a, b;
  int m, n, k;           // n: accumulator columns (2I for kGate, I for kDGate)
  int dtype;             // DenseType
  int mode;              // DenseMode
  void* out;
  long long ldo;
  const void* add;       // kStore: 16-bit addend or null
  long long ld_add;
  float* ab;             // kGate: written if not null; kDGate: read. [m, 2I], 16-byte aligned
  void* h_out;           // kDGate: [m, I]
  float* partials;       // split-K scratch (dense_scratch_bytes of it) or null if that is 0
  int* error_flag;
};

// Scratch bytes of the fp32 partial sums for these sizes (0: K is not split).
size_t dense_scratch_bytes(int m, int n, int k, int mode, bool b_k_major);
int launch_dense_gemm(const DenseGemm& g, cudaStream_t stream);

// Tensor map of an operand with `extent` m (or n) and k: boxes of 64 k x box rows (K-major) or of
// 64 m x 64 k, 128-byte swizzle, zeros out of bounds.
int make_operand_map(CUtensorMap* map, const DenseOperand& o, int extent, int k, int dtype, int box);

// Map of gated weights [gate rows; up rows] (K-major) as [inter / 8][2][8] rows: a box is 64 k x eight
// gate and the eight matching up rows x eight such groups, 128 rows in that order.
int make_gated_map(CUtensorMap* map, const DenseOperand& o, int inter, int k, int dtype);

// How a product runs (muse_moe_linear_plan, muse_moe_ffn_plan), in the order of their plan's entries.
struct PlanInfo {
  long long kernel, tile, tiles, whole, splits, per_group;
};
inline int put_plan(const PlanInfo& p, int* out) {
  if (p.tiles > (1 << 30)) return MUSE_ERR_UNSUPPORTED_SHAPE;   // more than any launch takes
  const long long v[6] = {p.kernel, p.tile, p.tiles, p.whole, p.splits, p.per_group};
  for (int i = 0; i < 6; ++i) out[i] = (int)v[i];
  return MUSE_OK;
}
PlanInfo dense_plan(int m, int n, int k, int mode, bool b_k_major);
PlanInfo swap_dense_plan(int m, int n, int k);

// The forward products (modes kStore and kGate, both operands along k) with the weights on the MMA's
// M side (swap_gemm.cu), and both forms' estimated times in SM clocks.
double dense_cost(int m, int n, int k, int mode, bool b_k_major);
double swap_dense_cost(int m, int n, int k);
int launch_swap_dense(const DenseGemm& g, cudaStream_t stream);

// ---- 16-bit conversions shared by the dense kernels

// Logistic function and silu with the fast division (2 steps of 2^-24; its range ends at 2^126, where
// the result is below 2^-118 and becomes 0): the exact one's slow path is a branch per element.
__device__ __forceinline__ float sigmoid_f(float a) { return __fdividef(1.f, 1.f + __expf(-a)); }
__device__ __forceinline__ float silu_f(float a) { return __fdividef(a, 1.f + __expf(-a)); }

__device__ __forceinline__ uint32_t pack16(int dtype, float lo, float hi) {
  uint32_t r;
  if (dtype == kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float2 unpack16(int dtype, uint32_t v) {
  if (dtype == kBf16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
  float lo, hi;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.f32.f16 %0, l;\n\tcvt.f32.f16 %1, h;\n\t}"
      : "=f"(lo), "=f"(hi) : "r"(v));
  return make_float2(lo, hi);
}

// ---- programmatic dependent launch: the kernels of one call are launched with the attribute
// (launch_chained) and wait here before they touch global memory, so a kernel's set-up overlaps
// the one before it. Every thread that reads or writes global memory waits, and does so before its
// bounded waits: what the kernel before wrote is visible only after the wait, even where it releases
// nothing early and its CTAs have left. Ahead of it weights are at most drawn into L2.

__device__ __forceinline__ void chain_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void chain_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
inline int launch_chained(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                          int cluster, Args... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = block;
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  c.attrs = at;
  c.numAttrs = cluster > 1 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&c, kernel, Params(args)...);
}

}  // namespace muse
