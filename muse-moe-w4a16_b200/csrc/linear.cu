// y = x . W^T with an NVFP4 weight (E2M1 codes, an e4m3 scale per 16 of them along K, one fp32
// scale): the dense projections and the 4-bit shared expert beside the routed experts.
//
//   y[t, n] = gs * sum_k x[t, k] * e2m1[n, k] * e4m3[n, k / 16]     (+ add[t, n])
//   gated:  y[t, i] = silu(a) * b,  a, b = the products with gate row i and up row i
//
// The weight is kept in the tile order of layout.cuh (rows padded to 128, K to 128 with zero
// codes), the routed experts' own format, so that sixteen rows of a 128-code chunk are 1 KiB in
// a row and a code pair drops into a bf16x2 with one logic op.
#undef MUSE_TRACE  // these kernels record no stamps
#include "kernels.cuh"
#include "w4.cuh"

namespace muse {
namespace {

// ---------------------------------------------------------------------------- repack

// One CTA per (128-row tile, 128-code chunk), thread = tile row. Rows and codes past the
// matrix are zero codes with zero scales. gate_up > 0: rows of gate and up interleave by 16 as
// in a w13 tile; `gate_up` is I, padded to 64 rows per half on its own.
__global__ void __launch_bounds__(kTileM)
prepare_linear_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int cols,
                      int gate_up, uint8_t* __restrict__ codes_out, uint8_t* __restrict__ scales_out) {
  const int kc = blockIdx.x, m = blockIdx.y, r = threadIdx.x;
  const int k_chunks = gridDim.x;
  int src = m * kTileM + r;
  bool row_ok = src < rows;
  if (gate_up > 0) {
    const int j = 64 * m + 16 * (r >> 5) + (r & 15);  // output column
    row_ok = j < gate_up;
    src = (r & 16) ? gate_up + j : j;
  }
  const size_t tile = (size_t)m * k_chunks + kc;
  uint8_t* dst = codes_out + tile * kTileCodeBytes + (size_t)r * kRowCodeBytes;
  uint8_t* sdst = scales_out + tile * kTileScaleBytes + (size_t)r * kRowScaleBytes;
  const uint8_t* c = codes + (size_t)src * (cols / 2) + (size_t)kc * kRowCodeBytes;
  const uint8_t* s = scales + (size_t)src * (cols / 16) + (size_t)kc * kRowScaleBytes;
  const int blocks = row_ok ? min(8, cols / 16 - kc * 8) : 0;  // 16-code blocks inside the matrix
  // rows are cols / 2 bytes apart, a multiple of 8: 8-byte loads
  for (int i = 0; i < 4; ++i) {
    uint2 lo = make_uint2(0, 0), hi = make_uint2(0, 0);
    if (2 * i < blocks) lo = *reinterpret_cast<const uint2*>(c + 16 * i);
    if (2 * i + 1 < blocks) hi = *reinterpret_cast<const uint2*>(c + 16 * i + 8);
    *reinterpret_cast<uint4*>(dst + 16 * code_slot(r, i)) =
        make_uint4(permute_codes(lo.x), permute_codes(lo.y), permute_codes(hi.x), permute_codes(hi.y));
  }
  for (int i = 0; i < 8; ++i) sdst[i] = i < blocks ? s[i] : 0;
}

// ---------------------------------------------------------------------------- few tokens

// mma.sync m16n8k16, fp32 accumulators: 16 weight rows x 8 tokens x 16 k.
template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if (kHalf)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

constexpr int kFewWarps = 8;
// Chunks in flight per warp: the token rows share the ring, so more tokens leave room for fewer.
template <int kNT> constexpr int kDepthOf = kNT == 1 ? 4 : kNT == 2 ? 3 : 2;

// A CTA of eight warps computes 16 * kMT weight rows for up to 8 * kNT tokens; the warps take the
// 128-code chunks of K in turn and a cluster of CTAs splits them further, so that a matrix of few
// rows still fills the chip. A lane copies the code pieces that it multiplies into its own part
// of the warp's ring (cp.async, several chunks deep): no barrier inside the K loop. Sums over warps
// and cluster ranks are taken in a fixed order, through shared and distributed shared memory.
// Bound by the weights' bytes while tokens are few (measured figures at launch_few).
template <int kMT, int kNT, bool kHalf, bool kGated>
__global__ void __launch_bounds__(32 * kFewWarps)
linear_few(const LinearArgs a) {
  static_assert(!kGated || kMT % 2 == 0, "gate and up tiles come in pairs");
  constexpr int kFewDepth = kDepthOf<kNT>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int row0 = (blockIdx.x / ranks) * 16 * kMT;  // first (padded) weight row
  const int m_tile = row0 / kTileM, r0 = row0 % kTileM;
  const int tok0 = blockIdx.y * a.tile_tokens;
  const int toks = min(a.tile_tokens, a.tokens - tok0);
  const int x_bytes = a.tile_tokens * 256;
  const int stage_bytes = kMT * 1152 + x_bytes;
  const uint32_t ring = ptx::smem_u32(smem) + warp * kFewDepth * stage_bytes;
  uint8_t* ring_p = smem + warp * kFewDepth * stage_bytes;

  const int first = rank * kFewWarps + warp, step = ranks * kFewWarps;
  const int n_chunks = first < a.k_chunks ? (a.k_chunks - first + step - 1) / step : 0;
  auto load_w = [&](int i) {
    const size_t tile = (size_t)m_tile * a.k_chunks + first + i * step;
    const uint32_t dst = ring + (i % kFewDepth) * stage_bytes;
    const uint8_t* q = a.wq + tile * kTileCodeBytes;
#pragma unroll
    for (int m = 0; m < 2 * kMT; ++m) {
      const int r = r0 + 8 * m + g;
      cp_async16(dst + (m * 32 + lane) * 16, q + r * kRowCodeBytes + 16 * code_slot(r, t), true);
    }
    if (lane < 8 * kMT)
      cp_async16(dst + kMT * 1024 + lane * 16, a.wsf + tile * kTileScaleBytes + r0 * kRowScaleBytes + lane * 16, true);
  };
  auto load_x = [&](int i) {
    const int k0 = (first + i * step) * kChunkK;
    const uint32_t dst = ring + (i % kFewDepth) * stage_bytes + kMT * 1152;
    for (int p = lane; p < a.tile_tokens * 16; p += 32) {
      const int tok = p >> 4, q = p & 15, k = k0 + q * 8;
      const bool ok = tok < toks && k < a.cols;
      const uint16_t* src = ok ? a.x + (size_t)(tok0 + tok) * a.ldx + k : a.x;
      cp_async16(dst + ((q & 3) * a.tile_tokens * 4 + tok * 4 + (q >> 2)) * 16, src, ok);
    }
  };
  // The weights are written by prepare only, never by the kernel before this one, so their first
  // chunks are fetched ahead of the wait for it.
  chain_release();
#pragma unroll
  for (int i = 0; i < kFewDepth - 1; ++i)
    if (i < n_chunks) load_w(i);
  chain_wait();
#pragma unroll
  for (int i = 0; i < kFewDepth - 1; ++i) {
    if (i < n_chunks) load_x(i);
    cp_commit();
  }

  float acc[kMT][kNT][4];
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;

  for (int i = 0; i < n_chunks; ++i) {
    cp_wait<kFewDepth - 2>();
    __syncwarp();
    const uint8_t* st = ring_p + (i % kFewDepth) * stage_bytes;
    if (i + kFewDepth - 1 < n_chunks) {
      load_w(i + kFewDepth - 1);
      load_x(i + kFewDepth - 1);
    }
    cp_commit();
    uint4 code[kMT][2];
    uint32_t sc[kMT][2][2];
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        code[m][h] = *reinterpret_cast<const uint4*>(st + ((2 * m + h) * 32 + lane) * 16);
        const uint32_t two = *reinterpret_cast<const uint16_t*>(st + kMT * 1024 + (16 * m + 8 * h + g) * 8 + 2 * t);
        expand_scales<kHalf>(two, sc[m][h][0], sc[m][h][1]);
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint4 b[kNT];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
        b[n] = make_uint4(0, 0, 0, 0);
        if (8 * n + g < toks)
          b[n] = *reinterpret_cast<const uint4*>(st + kMT * 1152 + (j * a.tile_tokens * 4 + (8 * n + g) * 4 + t) * 16);
      }
#pragma unroll
      for (int m = 0; m < kMT; ++m) {
        uint32_t lo[4], hi[4];
        const uint32_t wl = j == 0 ? code[m][0].x : j == 1 ? code[m][0].y : j == 2 ? code[m][0].z : code[m][0].w;
        const uint32_t wh = j == 0 ? code[m][1].x : j == 1 ? code[m][1].y : j == 2 ? code[m][1].z : code[m][1].w;
        dequant_word<kHalf>(wl, sc[m][0][j >> 1], a.m16, a.m64, lo);
        dequant_word<kHalf>(wh, sc[m][1][j >> 1], a.m16, a.m64, hi);
#pragma unroll
        for (int n = 0; n < kNT; ++n) {
          mma16816<kHalf>(acc[m][n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
          mma16816<kHalf>(acc[m][n], lo[2], hi[2], lo[3], hi[3], b[n].z, b[n].w);
        }
      }
    }
  }
  cp_wait<0>();
  __syncthreads();

  // warp partials: part[warp][row][token]
  constexpr int kRows = 16 * kMT, kToks = 8 * kNT;
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < kMT; ++m)
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        part[(warp * kRows + 16 * m + g + (i >> 1) * 8) * kToks + 8 * n + 2 * t + (i & 1)] = acc[m][n][i];
  __syncthreads();
  float* sums = part + kFewWarps * kRows * kToks;  // [token][row]
  for (int i = threadIdx.x; i < kRows * kToks; i += 32 * kFewWarps) {
    const int tok = i / kRows, row = i % kRows;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) s += part[(w * kRows + row) * kToks + tok];
    sums[tok * kRows + row] = s;
  }
  if (ranks > 1) {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  } else {
    __syncthreads();
  }
  if (rank == 0) {
    const float gs = __ldg(a.gs) * kUnscale<kHalf>;
    constexpr int kOut = kGated ? kRows / 2 : kRows;
    constexpr int dtype = kHalf ? kFp16 : kBf16;
    auto total = [&](int tok, int row) {
      float s = sums[tok * kRows + row];
      const uint32_t at = ptx::smem_u32(&sums[tok * kRows + row]);
      for (uint32_t k = 1; k < ranks; ++k) {
        uint32_t addr;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(at), "r"(k));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
        s += v;
      }
      return s * gs;
    };
    const int col0 = kGated ? row0 / 2 : row0;
    for (int i = threadIdx.x; i < kOut * kToks; i += 32 * kFewWarps) {
      const int tok = i / kOut, o = i % kOut;
      if (tok >= toks || col0 + o >= a.n_out) continue;
      float v;
      if (kGated) {
        const int r = (o >> 4) * 32 + (o & 15);
        v = silu_f(total(tok, r)) * total(tok, r + 16);
      } else {
        v = total(tok, o);
      }
      if (a.add) v += load16(dtype, a.add + (size_t)(tok0 + tok) * a.ld_add + col0 + o);
      a.out[(size_t)(tok0 + tok) * a.ldo + col0 + o] = round16(dtype, v);
    }
  }
  // a rank's sums are read by rank 0: stay until it is done
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int kMT, int kNT, bool kHalf, bool kGated>
int launch_few(LinearArgs a, cudaStream_t st) {
  a.tile_tokens = a.tokens < 8 * kNT ? a.tokens : 8 * kNT;
  const int ctas = a.padded_rows / (16 * kMT);
  const int y = (a.tokens + a.tile_tokens - 1) / a.tile_tokens;
  int cluster = 1;
  while (cluster < 8 && (long long)ctas * y * cluster < 2 * 148 && a.k_chunks >= 2 * kFewWarps * cluster) cluster *= 2;
  const size_t ring = (size_t)kFewWarps * kDepthOf<kNT> * (kMT * 1152 + a.tile_tokens * 256);
  const size_t red = (size_t)(kFewWarps + 1) * 16 * kMT * 8 * kNT * 4;
  const size_t smem = ring > red ? ring : red;
  static bool set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(linear_few<kMT, kNT, kHalf, kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  return launch_chained(linear_few<kMT, kNT, kHalf, kGated>, dim3(ctas * cluster, y), dim3(32 * kFewWarps), smem, st,
                        cluster, a);
}

template <int kMT, int kNT>
int launch_few_typed(const LinearArgs& a, int dtype, bool gated, cudaStream_t st) {
  if (gated)
    return dtype == kFp16 ? launch_few<(kMT < 2 ? 2 : kMT), kNT, true, true>(a, st)
                          : launch_few<(kMT < 2 ? 2 : kMT), kNT, false, true>(a, st);
  return dtype == kFp16 ? launch_few<kMT, kNT, true, false>(a, st)
                        : launch_few<kMT, kNT, false, false>(a, st);
}

// Up to this many tokens the mma.sync kernel streams the weights; beyond, the tcgen05 kernel.
constexpr int kFewTokens = 8;

int padded(int v, int to) { return (v + to - 1) / to * to; }

int check_linear(int rows, int cols, int gated) {
  if (rows <= 0 || cols <= 0 || (gated != 0 && gated != 1) || (gated && rows % 2)) return MUSE_ERR_INVALID_ARGUMENT;
  if (cols % kBlock || rows > (1 << 24) || cols > (1 << 24)) return MUSE_ERR_UNSUPPORTED_SHAPE;
  return MUSE_OK;
}
int padded_rows_of(int rows, int gated) { return gated ? 2 * padded(rows / 2, 64) : padded(rows, kTileM); }

bool misaligned(const void* p, unsigned to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

}  // namespace
}  // namespace muse

using namespace muse;

extern "C" int muse_moe_linear_prepared_size(int rows, int cols, int gated, size_t* code_bytes, size_t* scale_bytes) {
  if (!code_bytes || !scale_bytes) return MUSE_ERR_INVALID_ARGUMENT;
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  const size_t n = (size_t)padded_rows_of(rows, gated) * padded(cols, kChunkK);
  *code_bytes = n / 2;
  *scale_bytes = n / kBlock;
  return MUSE_OK;
}

extern "C" int muse_moe_prepare_linear(const uint8_t* w, const uint8_t* w_sf, int rows, int cols, int gated,
                                       uint8_t* w_out, uint8_t* w_sf_out, muse_stream_t stream) {
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  if (!w || !w_sf || !w_out || !w_sf_out || misaligned(w, 8) || misaligned(w_out, 16) || misaligned(w_sf_out, 16))
    return MUSE_ERR_INVALID_ARGUMENT;
  const dim3 grid(padded(cols, kChunkK) / kChunkK, padded_rows_of(rows, gated) / kTileM);
  if (grid.y > 65535) return MUSE_ERR_UNSUPPORTED_SHAPE;
  prepare_linear_kernel<<<grid, kTileM, 0, (cudaStream_t)stream>>>(w, w_sf, rows, cols, gated ? rows / 2 : 0, w_out,
                                                                   w_sf_out);
  return last_launch_status();
}

extern "C" int muse_moe_linear_workspace_size(int tokens, int rows, int cols, int gated, size_t* bytes) {
  if (!bytes) return MUSE_ERR_INVALID_ARGUMENT;
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  if (tokens < 0) return MUSE_ERR_INVALID_ARGUMENT;
  *bytes = tokens > kFewTokens
               ? linear_gemm_scratch_bytes(tokens, padded_rows_of(rows, gated), padded(cols, kChunkK) / kChunkK)
               : 0;
  return MUSE_OK;
}

extern "C" int muse_moe_linear_w4(const void* x, long long ldx, int dtype, int tokens, int rows, int cols, int gated,
                                  const uint8_t* wp, const uint8_t* w_sfp, const float* w_gs, const void* add,
                                  long long ld_add, void* out, long long ldo, void* workspace,
                                  size_t workspace_bytes, muse_stream_t stream) {
  int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  const int n_out = gated ? rows / 2 : rows;
  if (tokens < 0 || (dtype != kBf16 && dtype != kFp16)) return MUSE_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return MUSE_OK;
  if (!x || !wp || !w_sfp || !w_gs || !out || misaligned(x, 16) || ldx % 8 || misaligned(wp, 16) ||
      misaligned(w_sfp, 16) || (tokens > 1 && (ldx < cols || ldo < n_out || (add && ld_add < n_out))))
    return MUSE_ERR_INVALID_ARGUMENT;
  LinearArgs a{};
  a.wq = wp;
  a.wsf = w_sfp;
  a.gs = w_gs;
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx;
  a.add = static_cast<const uint16_t*>(add);
  a.ld_add = ld_add;
  a.out = static_cast<uint16_t*>(out);
  a.ldo = ldo;
  a.tokens = tokens;
  a.m16 = 16;
  a.m64 = 64;
  a.cols = cols;
  a.n_out = n_out;
  a.k_chunks = padded(cols, kChunkK) / kChunkK;
  a.padded_rows = padded_rows_of(rows, gated);
  const cudaStream_t st = (cudaStream_t)stream;
  if (tokens <= 4) return launch_few_typed<1, 1>(a, dtype, gated, st);
  if (tokens <= kFewTokens) return launch_few_typed<2, 1>(a, dtype, gated, st);
  const size_t scratch = linear_gemm_scratch_bytes(tokens, a.padded_rows, a.k_chunks);
  if (scratch > 0 && (!workspace || misaligned(workspace, 16))) return MUSE_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < scratch) return MUSE_ERR_WORKSPACE_TOO_SMALL;
  int* flag = nullptr;
  if ((rc = device_status_ptr(&flag))) return rc;
  return launch_linear_gemm(a, dtype, gated, static_cast<float*>(workspace), flag, st);
}
