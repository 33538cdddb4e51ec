// Products with few tokens (up to 32): y = x . W^T as a stream over the weights, which are either
// prepared NVFP4 tiles or 16-bit rows.
//
// A CTA takes 128 weight rows (gated 16-bit weights: 64 gate rows and the 64 matching up rows) and a
// cluster of CTAs splits K. One thread copies the weights into a ring of shared memory, 128 codes
// or 64 16-bit columns to a stage (one bulk copy of a tile, or a TMA box), and the same columns of
// x (TMA; rows past the last token read as zeros). Eight warps multiply 16 rows each (9 to 16 tokens:
// 32 rows and half of the k) by mma.sync m16n8k16: tokens are the 8-wide side, so one token wastes no
// weight traffic. Lanes read both operands as 16-byte pieces along k -- the order of k inside a stage
// is the lanes' -- so nothing is shuffled. A CTA pushes its sums to the ranks that own the outputs
// (16-byte stores to distributed shared memory, one cluster barrier), which add them in rank order.
// Sixteen warps with half of a stage each measured slower (13.0 against 8.7 us at 1 x 7168 x 4096
// gated).
// 16 bits are bound by the weights' bytes (the block of 1 x 7168 x 2048: 20.1 us, 4.4 TB/s over both
// products). NVFP4 is bound by latency: 1 x 7168 x 4096 gated takes 9.0 us, 1.8 TB/s, with a CTA's seven
// stages in flight from the start; its warps issue in 37 % of the cycles they are resident, the logic
// pipe is 33 % busy, and they wait at the barriers, for the first bytes and for one another's sums. So do
// the smallest sizes (1 x 1024 x 1024: 3.3 us).
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

// A stage is 128 codes or 64 16-bit columns of the tile's rows.
template <bool kW4> constexpr int kStageK = kW4 ? kChunkK : 64;
template <bool kW4> constexpr int kWeightBytes = kW4 ? kLinearTileBytes : kTileM * 128;
// x: boxes of 64 columns x 8 kNT tokens.
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
template <bool kW4, int kNT, bool kHalf, bool kGated>
__global__ void __launch_bounds__(kThreads)
few_tokens(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const FewArgs a) {
  constexpr int kK = kStageK<kW4>, kWBytes = kWeightBytes<kW4>, kStage = kStageBytes<kW4, kNT>;
  constexpr int dtype = kHalf ? kFp16 : kBf16;
  constexpr int kOut = kGated ? kTileM / 2 : kTileM;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int toks = a.tokens, ranks = a.ranks;
  float* recv = reinterpret_cast<float*>(smem + a.depth * kStage);  // [rank][token][128 / ranks]
  float* sums = recv + toks * kTileM;                 // [token][kPitch], rows in the order of their owners
  Ctl& ctl = *reinterpret_cast<Ctl*>(sums + toks * kPitch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();
  const int m_tile = blockIdx.x / ranks;
  const int first = rank * a.stages_per_rank;
  const int n_stages = max(0, min(a.stages_per_rank, a.stages - first));

  if (warp == kWarps) {
    if (lane < a.depth) {
      ptx::mbar_init(&ctl.full[lane], 1);
      ptx::mbar_init(&ctl.empty[lane], kWarps);
    }
    ptx::fence_barrier_init();
    __syncwarp();
  }
  chain_release();
  // The ranks meet here before they write to one another, and it costs nothing to arrive early.
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");

  bool ok = true;
  const int share = kOut / ranks, width = kTileM / ranks;   // outputs and weight rows of one rank
  if (warp == kWarps) {
    const bool leader = ptx::elect_one();
    auto load_w = [&](int i) {
      const int slot = i % a.depth, k = first + i;
      uint8_t* dst = smem + slot * kStage;
      uint64_t* bar = &ctl.full[slot];
      ptx::mbar_arrive_expect_tx(bar, kStage);
      if (kW4) {
        ptx::bulk_g2s(dst, a.wq + ((size_t)m_tile * a.stages + k) * kWBytes, kWBytes, bar);
      } else if (kGated) {
        ptx::tma_load_2d(dst, &map_w, k * kK, m_tile * 64, bar);
        ptx::tma_load_2d(dst + kWBytes / 2, &map_w, k * kK, a.up_row + m_tile * 64, bar);
      } else {
        ptx::tma_load_2d(dst, &map_w, k * kK, m_tile * kTileM, bar);
      }
    };
    auto load_x = [&](int i) {
      const int slot = i % a.depth, k = first + i;
      uint8_t* dst = smem + slot * kStage + kWBytes;
      ptx::tma_load_2d(dst, &map_x, k * kK, 0, &ctl.full[slot]);
      if (kW4) ptx::tma_load_2d(dst + kNT * 1024, &map_x, k * kK + 64, 0, &ctl.full[slot]);
    };
    // Ahead of the wait for the kernel before, which might have written the weights, they are only drawn
    // into L2: a copy into shared memory would keep what it read too early.
    const int head = min(n_stages, a.depth);
    if (leader) {
      for (int i = 0; i < head; ++i) {
        if (kW4) {
          prefetch_bulk(a.wq + ((size_t)m_tile * a.stages + first + i) * kWBytes, kWBytes);
        } else {
          prefetch_tile(&map_w, (first + i) * kK, m_tile * kOut);
          if (kGated) prefetch_tile(&map_w, (first + i) * kK, a.up_row + m_tile * 64);
        }
      }
      chain_wait();
      for (int i = 0; i < head; ++i) {
        load_w(i);
        load_x(i);
      }
    }
    __syncwarp();
    __syncthreads();      // the barriers are initialised: the consumers may wait on them
    if (leader)
      for (int i = head; i < n_stages; ++i) {
        if (!ptx::mbar_wait(&ctl.empty[i % a.depth], ((i / a.depth) & 1) ^ 1)) {
          ok = false;
          break;
        }
        load_w(i);
        load_x(i);
      }
    __syncwarp();
  } else {
    // A warp takes 16 rows. Two token groups: 32 rows and half of the stage's k, which halves
    // the reads of x per row (13 x 2048 x 7168: 11.9 to 9.5 us; with four groups the registers cost more).
    constexpr int kMT = kNT == 2 ? 2 : 1;
    constexpr int kSets = kNT == 1 ? 2 : 1;   // neighbouring MMAs should not wait for each other
    float acc[kSets][kMT][kNT][4];
#pragma unroll
    for (int h = 0; h < kSets; ++h)
#pragma unroll
      for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[h][m][n][i] = 0.f;
    chain_wait();   // x comes after it, and the bounded waits below do not count the kernel before
    __syncthreads();

    const int g = lane >> 2, t = lane & 3;
    const int r0 = (kMT == 1 ? warp * 16 : (warp & 3) * 32) + g, kh = kMT == 1 ? 0 : warp >> 2;
    int slot = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n_stages; ++i) {
      // after an expired wait the warp runs on, together, over what is there
      if (ok && !ptx::mbar_wait(&ctl.full[slot], phase)) ok = false;
      __syncwarp();
      const uint8_t* w = smem + slot * kStage;
      const uint8_t* xb = w + kWBytes;
      if (kW4) {
        // lane t's codes are k = 32 t .. 32 t + 31 in four words; a scale covers two of them
        constexpr int kWords = 4 / kMT;
        uint32_t word[2 * kMT][kWords], scale[2 * kMT][2];
#pragma unroll
        for (int h = 0; h < 2 * kMT; ++h) {
          const int r = r0 + 8 * h;
          const uint8_t* c = w + r * kRowCodeBytes + 16 * code_slot(r, t);
          const uint8_t* sc = w + kTileCodeBytes + r * kRowScaleBytes + 2 * t;
          if constexpr (kMT == 1) {
            const uint4 v = lds16(c);
            word[h][0] = v.x, word[h][1] = v.y, word[h][2] = v.z, word[h][3] = v.w;
            expand_scales<kHalf>(*reinterpret_cast<const uint16_t*>(sc), scale[h][0], scale[h][1]);
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(c + 8 * kh);
            word[h][0] = v.x, word[h][1] = v.y;
            if (h & 1)   // two rows' scales at a time
              expand_scales<kHalf>(sc[kh - 8 * kRowScaleBytes] | (uint32_t)sc[kh] << 8, scale[h - 1][0], scale[h][0]);
          }
        }
#pragma unroll
        for (int j = 0; j < kWords; ++j) {
          uint4 b[kNT];
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            b[n] = box_piece(xb + (t >> 1) * kNT * 1024, 8 * n + g, (t & 1) * 4 + kWords * kh + j);
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            uint32_t lo[4], hi[4];
            dequant_word<kHalf>(word[2 * m][j], scale[2 * m][kMT == 1 ? j >> 1 : 0], a.m16, a.m64, lo);
            dequant_word<kHalf>(word[2 * m + 1][j], scale[2 * m + 1][kMT == 1 ? j >> 1 : 0], a.m16, a.m64, hi);
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
              mma16816<kHalf>(acc[0][m][n], lo[0], hi[0], lo[1], hi[1], b[n].x, b[n].y);
              mma16816<kHalf>(acc[kSets - 1][m][n], lo[2], hi[2], lo[3], hi[3], b[n].z, b[n].w);
            }
          }
        }
      } else {
        // lane t's pieces are k = 16 t .. 16 t + 15, two of eight
#pragma unroll
        for (int jj = 0; jj < 2 / kMT; ++jj) {
          const int j = kMT == 1 ? jj : kh;
          uint4 b[kNT];
#pragma unroll
          for (int n = 0; n < kNT; ++n) b[n] = box_piece(xb, 8 * n + g, 2 * t + j);
#pragma unroll
          for (int m = 0; m < kMT; ++m) {
            const uint4 lo = box_piece(w, r0 + 16 * m, 2 * t + j), hi = box_piece(w, r0 + 16 * m + 8, 2 * t + j);
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
              mma16816<kHalf>(acc[0][m][n], lo.x, hi.x, lo.y, hi.y, b[n].x, b[n].y);
              mma16816<kHalf>(acc[kSets - 1][m][n], lo.z, hi.z, lo.w, hi.w, b[n].z, b[n].w);
            }
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
    auto each_sum = [&](auto&& f) {
#pragma unroll
      for (int h = 0; h < 2 * kMT; ++h) {
        const int row = r0 + 8 * h;
        // output of the row, and whether it is the up half of a gated one
        const int o = !kGated ? row : kW4 ? (row >> 5) * 16 + (row & 15) : row & 63;
        const int up = !kGated ? 0 : kW4 ? (row >> 4) & 1 : row >> 6;
        const int owner = o / share, at = owner * width + up * share + o - owner * share;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int tok = 8 * n + 2 * t + i;
            const float v = acc[0][h >> 1][n][2 * (h & 1) + i];
            if (tok < toks) f(sums[tok * kPitch + at], kSets > 1 ? v + acc[kSets - 1][h >> 1][n][2 * (h & 1) + i] : v);
          }
      }
    };
    if (kh == 0) each_sum([](float& s, float v) { s = v; });
    if (kMT > 1) {   // the second half of k, once the first is there
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
      if (kh == 1) each_sum([](float& s, float v) { s += v; });
    }
  }
  if (!ok) give_up(a.error_flag);
  __syncwarp();
  chain_wait();   // add is read and the outputs are written below
  __syncthreads();
  const float scale = kW4 ? load_scale<kHalf>(a.gs) : 1.f;
  if (ranks > 1) {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    const uint32_t mine = ptx::smem_u32(recv) + rank * toks * width * 4;
    for (int i = threadIdx.x; i < toks * (kTileM / 4); i += kThreads) {
      const int tok = i / (kTileM / 4), at = i % (kTileM / 4) * 4, owner = at / width;
      const float4 v = *reinterpret_cast<const float4*>(sums + tok * kPitch + at);
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(mine), "r"(owner));
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + (tok * width + at - owner * width) * 4),
                   "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
                   : "memory");
    }
    cluster_sync();
  }

  const float* from = ranks > 1 ? recv : sums;
  const int tok_pitch = ranks > 1 ? width : kPitch;
  for (int i = threadIdx.x; i < share * toks; i += kThreads) {
    const int tok = i / share, o = i - tok * share;
    const int col = m_tile * kOut + rank * share + o;
    if (col >= a.n_out) continue;
    float add = 0.f;
    if (a.add) add = load16(dtype, a.add + (size_t)tok * a.ld_add + col);
    const float* p = from + tok * tok_pitch + o;
    float v = 0.f, up = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < ranks) {
        v += p[k * toks * width];
        if (kGated) up += p[k * toks * width + share];
      }
    v *= scale;
    if (kGated) {
      up *= scale;
      if (!kW4 && a.ab) {
        a.ab[(size_t)tok * 2 * a.n_out + col] = v;
        a.ab[(size_t)tok * 2 * a.n_out + a.n_out + col] = up;
      }
      v = silu_f(v) * up;
    }
    a.out[(size_t)tok * a.ldo + col] = round16(dtype, v + add);
  }
}

// Shared memory beside the ring: the sums twice, the barriers and alignment.
size_t rest_bytes(int tokens) { return 1024 + (size_t)4 * (kTileM + kPitch) * tokens + sizeof(Ctl); }

// CTAs to aim for: about two on every SM keep enough copies in flight.
constexpr int kTargetCtas = 2 * 148;
constexpr size_t kCtaBytes = 112 * 1024;   // shared memory of one: two on an SM

template <bool kW4, int kNT, bool kHalf, bool kGated>
int launch(FewArgs a, int m_tiles, const CUtensorMap& mx, const CUtensorMap& mw, cudaStream_t st) {
  constexpr int kStage = kStageBytes<kW4, kNT>;
  a.ranks = 1;
  while (a.ranks < 8 && m_tiles * a.ranks * 2 <= kTargetCtas && a.stages >= 4 * a.ranks) a.ranks *= 2;
  a.stages_per_rank = (a.stages + a.ranks - 1) / a.ranks;
  a.depth = (int)((kCtaBytes - rest_bytes(a.tokens)) / kStage);
  if (a.depth > kMaxDepth) a.depth = kMaxDepth;
  if (a.depth > a.stages_per_rank) a.depth = a.stages_per_rank;
  const size_t smem = rest_bytes(a.tokens) + (size_t)a.depth * kStage;
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
  const int rows = gated ? 64 : kTileM;
  CUtensorMap mx, mw;
  int rc = make_operand_map(&mx, g.a, g.m, g.k, g.dtype, box_tokens(g.m));
  if (!rc) rc = make_operand_map(&mw, g.b, g.n, g.k, g.dtype, rows);
  if (rc) return rc;
  return launch_sized<false>(a, g.dtype, gated, (a.n_out + rows - 1) / rows, mx, mw, st);
}

}  // namespace muse
