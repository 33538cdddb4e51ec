// Products with few tokens (up to 32): y = x . W^T as a stream over the weights, which are either
// prepared NVFP4 tiles or 16-bit rows.
//
// A CTA takes 128 weight rows (gated 16-bit weights: 64 gate rows and the 64 matching up rows) and a
// cluster of CTAs splits K. One thread copies whole stages into a ring of shared memory -- NVFP4:
// the 9 KiB tile of 128 k by two bulk copies; 16 bits: 64 k by TMA -- together with the tokens'
// columns (TMA, rows past the last token read as zeros). Each of eight warps multiplies its
// own 16 rows by mma.sync m16n8k16: tokens are the 8-wide side, so one token wastes no weight
// traffic, and at 32 tokens the matrix pipe still keeps up with HBM. Lanes read operands as 16-byte
// pieces along k: the order of k inside a stage is the lanes', the same for both operands, so no
// shuffle is needed. There is no reduction inside a CTA; the ranks' sums meet once, in rank order,
// through distributed shared memory, each rank finishing its share of the rows.
// Bound by the weights' bytes; the smallest sizes by launch, first-byte and cluster latency.
#undef MUSE_TRACE  // these kernels record no stamps
#include "few_tokens.cuh"

#include "kernels.cuh"
#include "pair.cuh"

namespace muse {
namespace {

constexpr int kWarps = 8;                     // consumers, 16 rows each
constexpr int kThreads = 32 * (kWarps + 1);   // and the producer
constexpr int kMaxDepth = 16;
constexpr int kPitch = kTileM + 4;            // floats of one token's sums: conflict-free fragment stores

struct Ctl {
  uint64_t full[kMaxDepth], empty[kMaxDepth];
};

template <bool kW4> constexpr int kStageK = kW4 ? kChunkK : 64;
template <bool kW4> constexpr int kWeightBytes = kW4 ? kTileCodeBytes + kTileScaleBytes : kTileM * 128;
template <bool kW4, int kNT> constexpr int kStageBytes = kWeightBytes<kW4> + (kW4 ? 2 : 1) * kNT * 1024;

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

__device__ __forceinline__ uint4 lds16(const uint8_t* p) { return *reinterpret_cast<const uint4*>(p); }
// 16-byte piece p of row r of a 128-byte-swizzled box.
__device__ __forceinline__ uint4 box_piece(const uint8_t* box, int r, int p) {
  return lds16(box + r * 128 + ((p ^ (r & 7)) << 4));
}
__device__ __forceinline__ void prefetch_tile(const CUtensorMap* map, int c0, int c1) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1)
               : "memory");
}

template <bool kW4, int kNT, bool kHalf, bool kGated>
__global__ void __launch_bounds__(kThreads)
few_tokens(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const FewArgs a) {
  constexpr int kK = kStageK<kW4>, kWBytes = kWeightBytes<kW4>, kStage = kStageBytes<kW4, kNT>;
  constexpr int dtype = kHalf ? kFp16 : kBf16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Ctl& ctl = *reinterpret_cast<Ctl*>(smem + a.depth * kStage);
  float* sums = reinterpret_cast<float*>(&ctl + 1);   // [token][kPitch]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), ranks = a.ranks;
  const int m_tile = blockIdx.x / ranks;
  const int first = rank * a.stages_per_rank;
  const int n_stages = min(a.stages_per_rank, a.stages - first);   // may be <= 0 for a last rank

  if (threadIdx.x == 0) {
    for (int s = 0; s < a.depth; ++s) {
      ptx::mbar_init(&ctl.full[s], 1);
      ptx::mbar_init(&ctl.empty[s], kWarps);
    }
    ptx::fence_barrier_init();
  }
  __syncthreads();
  chain_release();

  bool ok = true;
  float acc[kNT][4];
#pragma unroll
  for (int n = 0; n < kNT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  if (warp == kWarps) {
    if (ptx::elect_one()) {
      auto load_w = [&](int i, uint64_t* bar) {
        uint8_t* dst = smem + (i % a.depth) * kStage;
        if (kW4) {
          const size_t tile = (size_t)m_tile * a.stages + first + i;
          ptx::bulk_g2s(dst, a.wq + tile * kTileCodeBytes, kTileCodeBytes, bar);
          ptx::bulk_g2s(dst + kTileCodeBytes, a.wsf + tile * kTileScaleBytes, kTileScaleBytes, bar);
        } else if (kGated) {
          ptx::tma_load_2d(dst, &map_w, (first + i) * kK, m_tile * 64, bar);
          ptx::tma_load_2d(dst + kWBytes / 2, &map_w, (first + i) * kK, a.up_row + m_tile * 64, bar);
        } else {
          ptx::tma_load_2d(dst, &map_w, (first + i) * kK, m_tile * kTileM, bar);
        }
      };
      auto load_x = [&](int i, uint64_t* bar) {
        uint8_t* dst = smem + (i % a.depth) * kStage + kWBytes;
        ptx::tma_load_2d(dst, &map_x, (first + i) * kK, 0, bar);
        if (kW4) ptx::tma_load_2d(dst + kNT * 1024, &map_x, (first + i) * kK + 64, 0, bar);
      };
      const int head = min(n_stages, a.depth);
      // Ahead of the wait for the kernel before: prepared weights (written by prepare only) are
      // copied, 16-bit weights, which that kernel might have written, only drawn into L2.
      for (int i = 0; i < head; ++i) {
        if (kW4) {
          ptx::mbar_arrive_expect_tx(&ctl.full[i], kStage);
          load_w(i, &ctl.full[i]);
        } else if (kGated) {
          prefetch_tile(&map_w, (first + i) * kK, m_tile * 64);
          prefetch_tile(&map_w, (first + i) * kK, a.up_row + m_tile * 64);
        } else {
          prefetch_tile(&map_w, (first + i) * kK, m_tile * kTileM);
        }
      }
      chain_wait();
      for (int i = 0; i < n_stages; ++i) {
        const int slot = i % a.depth;
        if (i >= a.depth && !ptx::mbar_wait(&ctl.empty[slot], ((i / a.depth) & 1) ^ 1)) {
          ok = false;
          break;
        }
        if (!kW4 || i >= a.depth) {
          ptx::mbar_arrive_expect_tx(&ctl.full[slot], kStage);
          load_w(i, &ctl.full[slot]);
        }
        load_x(i, &ctl.full[slot]);
      }
    }
  } else {
    const int g = lane >> 2, t = lane & 3, r0 = warp * 16 + g;
    int slot = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n_stages; ++i) {
      if (!warp_wait(&ctl.full[slot], phase)) {
        ok = false;
        break;
      }
      const uint8_t* w = smem + slot * kStage;
      const uint8_t* xb = w + kWBytes;
      if (kW4) {
        const uint4 c0 = lds16(w + r0 * kRowCodeBytes + 16 * code_slot(r0, t));
        const uint4 c1 = lds16(w + (r0 + 8) * kRowCodeBytes + 16 * code_slot(r0 + 8, t));
        uint32_t s0[2], s1[2];
        expand_scales<kHalf>(*reinterpret_cast<const uint16_t*>(w + kTileCodeBytes + r0 * kRowScaleBytes + 2 * t), s0[0], s0[1]);
        expand_scales<kHalf>(*reinterpret_cast<const uint16_t*>(w + kTileCodeBytes + (r0 + 8) * kRowScaleBytes + 2 * t), s1[0],
                             s1[1]);
        const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // lane t's codes are k = 32 t .. 32 t + 31, word j eight of them
          uint4 b[kNT];
#pragma unroll
          for (int n = 0; n < kNT; ++n) b[n] = box_piece(xb + (t >> 1) * kNT * 1024, 8 * n + g, (t & 1) * 4 + j);
          uint32_t lo[4], hi[4];
          dequant_word<kHalf>(w0[j], s0[j >> 1], a.m16, a.m64, lo);
          dequant_word<kHalf>(w1[j], s1[j >> 1], a.m16, a.m64, hi);
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            mma16816<kHalf>(acc[n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
            mma16816<kHalf>(acc[n], lo[2], hi[2], lo[3], hi[3], b[n].z, b[n].w);
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {   // lane t's pieces are k = 16 t .. 16 t + 15
          const uint4 lo = box_piece(w, r0, 2 * t + j), hi = box_piece(w, r0 + 8, 2 * t + j);
#pragma unroll
          for (int n = 0; n < kNT; ++n) {
            const uint4 b = box_piece(xb, 8 * n + g, 2 * t + j);
            mma16816<kHalf>(acc[n], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
            mma16816<kHalf>(acc[n], lo.z, hi.z, lo.w, hi.w, b.z, b.w);
          }
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&ctl.empty[slot]);
      if (++slot == a.depth) {
        slot = 0;
        phase ^= 1;
      }
    }
#pragma unroll
    for (int n = 0; n < kNT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int tok = 8 * n + 2 * t + (i & 1);
        if (tok < a.tokens) sums[tok * kPitch + r0 + (i >> 1) * 8] = acc[n][i];
      }
    chain_wait();   // add is read and the outputs are written below
  }
  if (!ok) give_up(a.error_flag);
  __syncwarp();
  if (ranks > 1)
    cluster_sync();
  else
    __syncthreads();

  // Outputs of the tile: kOut per token, this rank's share of them.
  constexpr int kOut = kGated ? kTileM / 2 : kTileM;
  const int share = kOut / ranks;
  const float scale = kW4 ? __ldg(a.gs) * kUnscale<kHalf> : 1.f;
  uint32_t base[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < ranks) base[k] = map_rank(sums, k);
  auto total = [&](int tok, int row) {
    float s = 0.f, v[8];
    const uint32_t off = (tok * kPitch + row) * 4;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < ranks) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[k]) : "r"(base[k] + off) : "memory");
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < ranks) s += v[k];
    return s * scale;
  };
  if (warp < kWarps) {
    for (int i = threadIdx.x; i < share * a.tokens; i += 32 * kWarps) {
      const int tok = i / share, o = rank * share + (i - tok * share);
      const int col = m_tile * kOut + o;
      if (col >= a.n_out) continue;
      float v;
      if (kGated) {
        const int gate = kW4 ? (o >> 4) * 32 + (o & 15) : o;
        const float ga = total(tok, gate), up = total(tok, gate + (kW4 ? 16 : 64));
        if (!kW4 && a.ab) {
          a.ab[(size_t)tok * 2 * a.n_out + col] = ga;
          a.ab[(size_t)tok * 2 * a.n_out + a.n_out + col] = up;
        }
        v = silu_f(ga) * up;
      } else {
        v = total(tok, o);
      }
      if (a.add) v += load16(dtype, a.add + (size_t)tok * a.ld_add + col);
      a.out[(size_t)tok * a.ldo + col] = round16(dtype, v);
    }
  }
  if (ranks > 1) {   // the other ranks read this one's sums
    __syncwarp();
    cluster_sync();
  }
}

// CTAs to aim for: about two on every SM keep enough copies in flight.
constexpr int kTargetCtas = 2 * 148;
constexpr size_t kCtaBytes = 112 * 1024;   // shared memory of one: two on an SM

template <bool kW4, int kNT, bool kHalf, bool kGated>
int launch(FewArgs a, int m_tiles, const CUtensorMap& mx, const CUtensorMap& mw, cudaStream_t st) {
  constexpr int kStage = kStageBytes<kW4, kNT>;
  a.ranks = 1;
  while (a.ranks < 8 && m_tiles * a.ranks * 2 <= kTargetCtas && a.stages >= 4 * a.ranks) a.ranks *= 2;
  a.stages_per_rank = (a.stages + a.ranks - 1) / a.ranks;
  const size_t rest = 1024 + sizeof(Ctl) + (size_t)4 * kPitch * a.tokens;
  a.depth = (int)((kCtaBytes - rest) / kStage);
  if (a.depth > kMaxDepth) a.depth = kMaxDepth;
  if (a.depth > a.stages_per_rank) a.depth = a.stages_per_rank;
  const size_t smem = rest + (size_t)a.depth * kStage;
  static bool set[64] = {};  // per device: the attribute belongs to its context
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(few_tokens<kW4, kNT, kHalf, kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kCtaBytes);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  return launch_chained(few_tokens<kW4, kNT, kHalf, kGated>, dim3(m_tiles * a.ranks), dim3(kThreads), smem, st, a.ranks,
                        mx, mw, a);
}

template <bool kW4, int kNT>
int launch_typed(const FewArgs& a, int dtype, bool gated, int m_tiles, const CUtensorMap& mx, const CUtensorMap& mw,
                 cudaStream_t st) {
  if (dtype == kFp16)
    return gated ? launch<kW4, kNT, true, true>(a, m_tiles, mx, mw, st) : launch<kW4, kNT, true, false>(a, m_tiles, mx, mw, st);
  return gated ? launch<kW4, kNT, false, true>(a, m_tiles, mx, mw, st) : launch<kW4, kNT, false, false>(a, m_tiles, mx, mw, st);
}

template <bool kW4>
int launch_sized(const FewArgs& a, int dtype, bool gated, int m_tiles, const CUtensorMap& mx, const CUtensorMap& mw,
                 cudaStream_t st) {
  if (a.tokens <= 8) return launch_typed<kW4, 1>(a, dtype, gated, m_tiles, mx, mw, st);
  if (a.tokens <= 16) return launch_typed<kW4, 2>(a, dtype, gated, m_tiles, mx, mw, st);
  return launch_typed<kW4, 4>(a, dtype, gated, m_tiles, mx, mw, st);
}

// Rows of an x box: the token tile, so that rows past the last token are filled with zeros.
int box_tokens(int tokens) { return tokens <= 8 ? 8 : tokens <= 16 ? 16 : 32; }

}  // namespace

int launch_few_w4(const LinearArgs& l, int dtype, bool gated, int* error_flag, cudaStream_t st) {
  FewArgs a{};
  a.wq = l.wq;
  a.wsf = l.wsf;
  a.gs = l.gs;
  a.add = l.add;
  a.ld_add = l.ld_add;
  a.out = l.out;
  a.ldo = l.ldo;
  a.tokens = l.tokens;
  a.n_out = l.n_out;
  a.stages = l.k_chunks;
  a.m16 = l.m16;
  a.m64 = l.m64;
  a.error_flag = error_flag;
  CUtensorMap mx;
  const int rc = make_operand_map(&mx, DenseOperand{l.x, l.ldx, true}, l.tokens, l.cols, dtype, box_tokens(l.tokens));
  if (rc) return rc;
  return launch_sized<true>(a, dtype, gated, l.padded_rows / kTileM, mx, mx, st);
}

int launch_few_dense(const DenseGemm& g, cudaStream_t st) {
  const bool gated = g.mode == kGate;
  FewArgs a{};
  a.add = static_cast<const uint16_t*>(g.add);
  a.ld_add = g.ld_add;
  a.out = static_cast<uint16_t*>(g.out);
  a.ldo = g.ldo;
  a.ab = gated ? g.ab : nullptr;
  a.tokens = g.m;
  a.n_out = gated ? g.n / 2 : g.n;
  a.up_row = a.n_out;
  a.stages = (g.k + 63) / 64;
  a.error_flag = g.error_flag;
  CUtensorMap mx, mw;
  int rc = make_operand_map(&mx, g.a, g.m, g.k, g.dtype, box_tokens(g.m));
  if (!rc) rc = make_operand_map(&mw, g.b, g.n, g.k, g.dtype, gated ? 64 : kTileM);
  if (rc) return rc;
  const int rows = gated ? 64 : kTileM;
  return launch_sized<false>(a, g.dtype, gated, (a.n_out + rows - 1) / rows, mx, mw, st);
}

}  // namespace muse
