// y = x . W^T with the weight rows on the MMA's M side ("swap-AB"), on tcgen05: the product
// of a prepared NVFP4 weight with more than a few tokens, and the feed-forward block's forward
// products of 16-bit weights where that beats tokens on the M side (dense_gemm.cu).
//
// 128 weight rows of a CTA are M and up to 256 tokens N, in steps of 32, so a batch of any size wastes
// little. From a certain size a pair of CTAs works on one tile of 256 rows (cta_group::2: B is read
// once for both); below, single CTAs issue their MMAs in half the time (an MMA of a pair takes its
// issuer ~75 to 100 clocks however small N is, one of a CTA ~44). B is x by TMA. A is
//   16-bit weights: by TMA. Gated: a view of w13 as [I / 8][gate, up][8] rows puts eight gate rows
//   and the eight matching up rows next to one another, in one box.
//   NVFP4: per 128-code chunk a CTA copies its 128 rows' codes and scales (one bulk copy of 9 KiB)
//   into an eight-deep ring; sixteen warps turn them into exact 16-bit weights in registers (thread =
//   weight row) and store them to tensor memory, from where the MMAs read A. Through shared memory,
//   which carries B, the codes and its own 16 KiB twice, a stage took ~450 clocks at 64 tokens and
//   ~630 at 256.
// Where a group has several tiles its accumulators are double buffered in tensor memory, so that the
// epilogue overlaps the next tile's MMAs; it reads them as matrix fragments
// and turns them over (rows are weight rows, y's rows are tokens) with transposed matrix stores
// into shared memory, so that global stores run along y's rows. Gated tiles hold gate and up rows
// of an output in one thread's fragments.
// With fewer tiles than groups K is split over the groups (CTAs or pairs) of a cluster of up to eight
// CTAs. Each group owns every splits-th 32-token chunk of the tile's outputs and receives the others'
// accumulators of it, as fragments, through distributed shared memory (the rings are done by then): the
// owner adds them to its own, in split order, and finishes the chunk. One launch, no scratch memory.
// Tens of tokens are bound by set-up, exchange and the stages' hand-over more than by weight bytes (64 x
// 4096 x 8192 gated: 14.5 us, 1.4 TB/s, tensor pipe 19 % active). With NVFP4 weights hundreds and
// thousands are bound by a stage's dequantisation and hand-over, longer than its MMAs (4096 x 4096 x 4096:
// tensor pipe 75 % active, issue slots 48 %; 106 us at full clock, 119 in a loop under the power limit;
// 1000 x 4096 x 4096: 28 and 32 us; 2000 x 7168 x 4096 gated: 88 and 103 us).
#undef MUSE_TRACE  // these kernels record no stamps
#include "kernels.cuh"
#include "pair.cuh"
#include "w4.cuh"

namespace muse {
namespace {

constexpr int kMaxStages = 12;
constexpr int kABytes = kTileM * 128;
constexpr int kCodes = 8;                    // code ring: 128-code chunks of 9 KiB
constexpr int kCodeBytes = kLinearTileBytes;
// 64-k stages in shared memory: B (128 bytes a token; half the tokens in a pair) and, 16-bit weights,
// A (16 KiB). NVFP4's A takes 32 columns of tensor memory.
template <bool kW4> constexpr int kRingBytes = kW4 ? 8 * kABytes : 13 * kABytes;
template <bool kW4> constexpr int kStageA = kW4 ? 0 : kABytes;
constexpr int kTmemCols = 512;
constexpr int kPatch = 32 * 64;              // an epilogue warp's outputs of 32 tokens, 64 bytes each
constexpr int kDeqWarp0 = 4;                 // warps 0-2: codes, MMA, TMA; then dequantisers; then the epilogue
template <bool kW4> constexpr int kEpiWarp0 = kW4 ? 20 : 4;
template <bool kW4> constexpr int kThreads = 32 * (kEpiWarp0<kW4> + 4);

struct Ctl {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t code_full[kCodes], code_empty[kCodes];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem;
};
template <bool kW4>
constexpr size_t kSmem = 1024 + (size_t)kRingBytes<kW4> + (kW4 ? kCodes * kCodeBytes : 0) + 4 * kPatch + sizeof(Ctl);
static_assert(kSmem<true> <= 232448 && kSmem<false> <= 232448, "shared memory of one CTA");

struct GemmPlan {
  int ctas, bn, accs, stages, tiles_m, tiles_n, splits, units, units_per_split;  // units of K: 128 codes or 64 columns
};

struct Args {
  LinearArgs l;
  GemmPlan p;
  uint32_t idesc;
  uint32_t b_bytes;    // one CTA's B bytes per stage
  int out_vec, add_vec;  // rows of out / add are 16-byte aligned
  int* error_flag;
};

struct Tile {
  int m_tile, tok0, c0, c1;
};
// Tile `idx` (eight row tiles per token tile) as CTA `rank` of group `split` sees it.
template <int kCtas>
__device__ __forceinline__ Tile tile_of(const GemmPlan& p, int idx, uint32_t rank, int split) {
  constexpr int kGroup = 8;
  Tile t;
  const int group = idx / (kGroup * p.tiles_n);
  const int first = group * kGroup;
  const int rows = min(kGroup, p.tiles_m - first);
  const int r = idx - group * kGroup * p.tiles_n;
  t.m_tile = kCtas * (first + r % rows) + (int)rank;
  t.tok0 = r / rows * p.bn;
  t.c0 = split * p.units_per_split;
  t.c1 = min(p.units, t.c0 + p.units_per_split);
  return t;
}

// Position in a ring.
struct Pos {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int size) {
    if (++slot == size) {
      slot = 0;
      phase ^= 1;
    }
  }
  __device__ __forceinline__ void skip(int n, int size) {   // n <= size
    slot += n;
    if (slot >= size) {
      slot -= size;
      phase ^= 1;
    }
  }
};

// 128 weight rows x 64 k of tile m_tile (16-bit weights) into shared memory, or into L2. Gated: eight
// groups of eight gate and eight up rows.
template <int kCtas, bool kGated>
__device__ __forceinline__ void load_weights(uint32_t dst, const CUtensorMap* map, int k, int m_tile, uint32_t bar) {
  if (kGated)
    Group<kCtas>::tma_4d(dst, map, k, m_tile * 8, bar);
  else
    Group<kCtas>::tma_2d(dst, map, k, m_tile * kTileM, bar);
}
template <bool kGated>
__device__ __forceinline__ void prefetch_weights(const CUtensorMap* map, int k, int m_tile) {
  if (kGated)
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %2, %3}];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(k), "r"(0), "r"(m_tile * 8)
                 : "memory");
  else
    prefetch_tile(map, k, m_tile * kTileM);
}

// 16-byte piece `p` of token row `tok` of a patch; pieces are swizzled so that eight token rows of
// one piece, and the four pieces of two rows, lie in different banks.
__device__ __forceinline__ uint32_t patch_row(const uint8_t* patch, int tok, int p) {
  return ptx::smem_u32(patch) + tok * 64 + ((p ^ ((tok >> 1) & 3)) << 4);
}
// A patch of up to 32 tokens x outs 16-bit values: lane pieces (token, piece) of it.
template <int kOut>
struct PatchIo {
  static constexpr int kPieces = kOut / 8;
  // from rows tok0.. of a matrix into registers (all loads in flight together)
  static __device__ __forceinline__ void load(uint4 (&v)[kPieces], int lane, const uint16_t* base, long long ld, int tok0,
                                              int toks, int outs, int vec) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int tok = i * (32 / kPieces) + lane / kPieces, p = lane % kPieces;
      v[i] = make_uint4(0, 0, 0, 0);
      if (tok >= toks) continue;
      const uint16_t* g = base + (size_t)(tok0 + tok) * ld + 8 * p;
      if (vec && 8 * p + 8 <= outs) {
        v[i] = __ldcg(reinterpret_cast<const uint4*>(g));
      } else {
        uint32_t e[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = 8 * p + j < outs ? __ldcg(g + j) : 0;
        v[i] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
      }
    }
  }
  static __device__ __forceinline__ void put(uint8_t* patch, int lane, const uint4 (&v)[kPieces]) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int tok = i * (32 / kPieces) + lane / kPieces, p = lane % kPieces;
      *reinterpret_cast<uint4*>(patch + tok * 64 + ((p ^ ((tok >> 1) & 3)) << 4)) = v[i];
    }
  }
  // from the patch to rows tok0.. of a matrix
  static __device__ __forceinline__ void store(const uint8_t* patch, int lane, uint16_t* base, long long ld, int tok0,
                                               int toks, int outs, int vec) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int tok = i * (32 / kPieces) + lane / kPieces, p = lane % kPieces;
      if (tok >= toks) continue;
      const uint4 v = *reinterpret_cast<const uint4*>(patch + tok * 64 + ((p ^ ((tok >> 1) & 3)) << 4));
      uint16_t* g = base + (size_t)(tok0 + tok) * ld + 8 * p;
      if (vec && 8 * p + 8 <= outs) {
        *reinterpret_cast<uint4*>(g) = v;
      } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (8 * p + j < outs) g[j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
      }
    }
  }
};

template <int kCtas, bool kW4, bool kHalf, bool kGated>
__global__ void __launch_bounds__(kThreads<kW4>, 1)
swap_gemm(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Args a) {
  using G = Group<kCtas>;
  constexpr int kUnit = kW4 ? 2 : 1;   // stages of a unit
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* codes = smem + kRingBytes<kW4>;
  const int n_stages = a.p.stages, stage_bytes = kStageA<kW4> + a.b_bytes;
  uint8_t* patches = codes + (kW4 ? kCodes * kCodeBytes : 0);
  Ctl& ctl = *reinterpret_cast<Ctl*>(patches + 4 * kPatch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a cluster is the `splits` groups of one tile at a time; `team` counts clusters
  const int splits = a.p.splits;
  const uint32_t cta = cluster_rank(), rank = cta % kCtas, leader = cta - rank, mask = 3u << leader;
  const int split = (int)(cta / kCtas);
  const int team = blockIdx.x / (kCtas * splits), teams = gridDim.x / (kCtas * splits);
  const int total = a.p.tiles_m * a.p.tiles_n;

  // Barriers, one lane each.
  if (warp == 0) {
    if (kW4 && lane < kCodes) {
      ptx::mbar_init(&ctl.code_full[lane], 1);
      ptx::mbar_init(&ctl.code_empty[lane], 4);
    }
    ptx::fence_barrier_init();
  } else if (warp == 1) {
    G::alloc(&ctl.tmem, kTmemCols);
  } else if (warp == 2) {
    if (lane < n_stages) {
      ptx::mbar_init(&ctl.full[lane], kW4 ? 1 + kCtas * 4 : 1);  // bytes announced by the leader; NVFP4's A by four warps of each CTA
      ptx::mbar_init(&ctl.empty[lane], 1);
    } else if (lane < n_stages + 2) {
      ptx::mbar_init(&ctl.acc_full[lane - n_stages], 1);
      ptx::mbar_init(&ctl.acc_empty[lane - n_stages], kCtas * 4);
    }
    ptx::fence_barrier_init();
    if (lane == 0) ptx::prefetch_tensormap(&map_x);
  }
  ptx::tc_fence_before();
  __syncthreads();
  // A pair's CTAs use each other's barriers from the start, which the codes' warp does not: it goes on.
  // Groups meet when they exchange sums.
  if (kCtas > 1) {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    if (warp > 0) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  }
  ptx::tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  // tensor memory: one accumulator (two where a group has several tiles), then NVFP4's A stages
  const uint32_t a_cols = tmem + a.p.accs * a.p.bn;
  chain_release();

  bool ok = true;
  // ---- epilogue of a tile: this group's chunks of 32 tokens (all of them unless K is split)
  constexpr int dtype = kHalf ? kFp16 : kBf16;
  constexpr int kOut = kGated ? 16 : 32;                  // outputs of an epilogue warp
  using Io = PatchIo<kOut>;
  const int quarter = warp & 3, epi = warp - kEpiWarp0<kW4>, step = 32 * splits;
  const int chunks = (a.p.bn / 32 + splits - 1) / splits; // most chunks of one owner
  // fragments of this group's chunk `i` from another group (`from` counts the others)
  auto received = [&](uint8_t* base, int from, int i) { return base + (((from * chunks + i) * 4 + epi) << 12) + lane * 16; };
  uint4 ahead[Io::kPieces];                               // the next patch's addend
  auto first_addend = [&](const Tile& t) {
    const int o0 = kGated ? t.m_tile * 64 + quarter * 16 : t.m_tile * kTileM + quarter * 32;
    const int outs = min(kOut, a.l.n_out - o0), n_tok = min(a.p.bn, a.l.tokens - t.tok0);
    if (!a.l.add || outs <= 0) return;
    // the warp's rows of this tile's addend start for L2 together, while the sums are still being taken
    for (int tok = 32 * split + lane; tok < n_tok; tok += step)
      prefetch_l2(a.l.add + (size_t)(t.tok0 + tok) * a.l.ld_add + o0);
    if (32 * split < n_tok)
      Io::load(ahead, lane, a.l.add + o0, a.l.ld_add, t.tok0 + 32 * split, min(32, n_tok - 32 * split), outs, a.add_vec);
  };
  auto tile_epilogue = [&](const Tile& t, int buf) {
    const uint32_t acc = tmem + ((uint32_t)quarter << 21) + buf * a.p.bn;
    const float gs = kW4 ? load_scale<kHalf>(a.l.gs) : 1.f;
    uint8_t* patch = patches + epi * kPatch;
    const int o0 = kGated ? t.m_tile * 64 + quarter * 16 : t.m_tile * kTileM + quarter * 32;
    const int outs = min(kOut, a.l.n_out - o0);
    const int n_tok = min(a.p.bn, a.l.tokens - t.tok0);
    const bool adds = a.l.add && outs > 0;
    for (int c = 32 * split; c < n_tok && t.m_tile * kTileM < a.l.padded_rows; c += step) {
      // fragments of rows 0-15 and 16-31 of the warp's quarter (gated: gate and up of the same
      // outputs), through a transposed patch [token][output] so that stores run along outputs
      float lo[16], hi[16];
      tmem_ld_frag(acc + c, lo);
      tmem_ld_frag(acc + c + (16u << 16), hi);
      ptx::tmem_wait_ld();
      for (int from = 0; from < splits - 1; ++from) {
        const uint8_t* v = received(smem, from, c / step);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 x = *reinterpret_cast<const float4*>(v + i * 512), y = *reinterpret_cast<const float4*>(v + (i + 4) * 512);
          lo[4 * i] += x.x, lo[4 * i + 1] += x.y, lo[4 * i + 2] += x.z, lo[4 * i + 3] += x.w;
          hi[4 * i] += y.x, hi[4 * i + 1] += y.y, hi[4 * i + 2] += y.z, hi[4 * i + 3] += y.w;
        }
      }
      const int tok0 = t.tok0 + c, toks = min(32, n_tok - c);
      if (!kW4 && kGated && a.l.ab && outs > 0) {   // keep the pre-activations: eight outputs of a token at a time
        const int g = lane >> 2;
        float* to = a.l.ab + (size_t)tok0 * 2 * a.l.n_out + o0 + g;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int tok = 8 * (j >> 2) + 2 * (lane & 3) + (j & 1), up = j & 2 ? a.l.n_out : 0;
          if (tok >= toks) continue;
          if (g < outs) to[(size_t)tok * 2 * a.l.n_out + up] = lo[j];
          if (g + 8 < outs) to[(size_t)tok * 2 * a.l.n_out + up + 8] = hi[j];
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = 4 * b + i;
          if (!kGated) {
            lo[j] *= gs;
            hi[j] *= gs;
          } else if (kW4) {          // rows 0-15 gate, 16-31 up
            lo[j] = silu_f(lo[j] * gs) * (hi[j] * gs);
          } else if (i < 2) {        // rows 0-7 gate, 8-15 up; 16-23 gate, 24-31 up
            lo[j] = silu_f(lo[j]) * lo[j + 2];
            lo[j + 2] = silu_f(hi[j]) * hi[j + 2];
          }
        }
      __syncwarp();                                       // the patch's last readers are done
      if (adds) {
        Io::put(patch, lane, ahead);
        if (c + step < n_tok)
          Io::load(ahead, lane, a.l.add + o0, a.l.ld_add, tok0 + step, min(32, n_tok - c - step), outs, a.add_vec);
        __syncwarp();
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          uint32_t f[kGated ? 2 : 4];
          ldmatrix2_t(patch_row(patch, 8 * b + (lane & 7), (lane >> 3) & 1), f[0], f[1]);
          if (!kGated) ldmatrix2_t(patch_row(patch, 8 * b + (lane & 7), 2 + ((lane >> 3) & 1)), f[2], f[3]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 u = unpack16(dtype, f[i]);
            lo[4 * b + 2 * i] += u.x;
            lo[4 * b + 2 * i + 1] += u.y;
            if (!kGated) {
              const float2 w2 = unpack16(dtype, f[2 + i]);
              hi[4 * b + 2 * i] += w2.x;
              hi[4 * b + 2 * i + 1] += w2.y;
            }
          }
        }
        __syncwarp();
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        stmatrix2_t(patch_row(patch, 8 * b + (lane & 7), (lane >> 3) & 1), pack16(dtype, lo[4 * b], lo[4 * b + 1]),
                    pack16(dtype, lo[4 * b + 2], lo[4 * b + 3]));
        if (!kGated)
          stmatrix2_t(patch_row(patch, 8 * b + (lane & 7), 2 + ((lane >> 3) & 1)),
                      pack16(dtype, hi[4 * b], hi[4 * b + 1]), pack16(dtype, hi[4 * b + 2], hi[4 * b + 3]));
      }
      __syncwarp();
      if (outs > 0) Io::store(patch, lane, a.l.out + o0, a.l.ldo, tok0, toks, outs, a.out_vec);
    }
  };

  if (warp == 0) {
    if (kW4 && lane == 0) {
      // The kernel before might have written the weight: ahead of it the first codes are only drawn into L2.
      auto tile_codes = [&](int m_tile) {
        // a pair's second tile may lie past the last: it multiplies the last tile and stores nothing
        return a.l.wq + (size_t)min(m_tile, a.l.padded_rows / kTileM - 1) * a.p.units * kLinearTileBytes;
      };
      if (team < total) {
        const Tile t = tile_of<kCtas>(a.p, team, rank, split);
        for (int c = t.c0; c < min(t.c1, t.c0 + kCodes); ++c)
          prefetch_bulk(tile_codes(t.m_tile) + (size_t)c * kLinearTileBytes, kLinearTileBytes);
      }
      chain_wait();
      Pos q;
      for (int w = team; w < total && ok; w += teams) {
        const Tile t = tile_of<kCtas>(a.p, w, rank, split);
        const uint8_t* src = tile_codes(t.m_tile);
        for (int c = t.c0; c < t.c1; ++c, q.next(kCodes)) {
          if (!ptx::mbar_wait_sleep(&ctl.code_empty[q.slot], q.phase ^ 1)) {
            ok = false;
            break;
          }
          ptx::mbar_arrive_expect_tx(&ctl.code_full[q.slot], kCodeBytes);
          ptx::bulk_g2s(codes + q.slot * kCodeBytes, src + (size_t)c * kLinearTileBytes, kCodeBytes, &ctl.code_full[q.slot]);
        }
      }
    }
    __syncwarp();
    if (kCtas > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      chain_wait();   // B comes after it: the bounded waits do not count the kernel before
      Pos s;
      int it = 0;
      for (int w = team; w < total && ok; w += teams, ++it) {
        const Tile t = tile_of<kCtas>(a.p, w, rank, split);
        const int buf = it & 1;
        if (!ptx::mbar_wait(&ctl.acc_empty[buf], ((it >> 1) & 1) ^ 1)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t d = tmem + buf * a.p.bn;
        for (int n = kUnit * t.c0; n < kUnit * t.c1; ++n) {
          if (!ptx::mbar_wait(&ctl.full[s.slot], s.phase)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t sa = ptx::smem_u32(smem + s.slot * stage_bytes);
          const uint64_t da = operand_desc<false>(sa), db = operand_desc<false>(sa + kStageA<kW4>);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t more = n > kUnit * t.c0 || j > 0;
            if (kW4)
              G::mma_ts(d, a_cols + 32 * s.slot + 8 * j, db + j * kStepDesc<false>, a.idesc, more);
            else
              G::mma(d, da + j * kStepDesc<false>, db + j * kStepDesc<false>, a.idesc, more);
          }
          G::commit(&ctl.empty[s.slot], mask);
          s.next(n_stages);
        }
        G::commit(&ctl.acc_full[buf], mask);
      }
    }
  } else if (warp == 2) {
    if (ptx::elect_one()) {
      if (!kW4 && team < total) {
        // 16-bit weights might have been written by the kernel before: only drawn into L2 ahead of it
        const Tile t = tile_of<kCtas>(a.p, team, rank, split);
        for (int n = t.c0; n < min(t.c1, t.c0 + n_stages); ++n) prefetch_weights<kGated>(&map_w, n * 64, t.m_tile);
      }
      chain_wait();
      Pos s;
      for (int w = team; w < total && ok; w += teams) {
        const Tile t = tile_of<kCtas>(a.p, w, rank, split);
        const int row = t.tok0 + (int)rank * (a.p.bn / kCtas);
        for (int n = kUnit * t.c0; n < kUnit * t.c1; ++n) {
          if (!ptx::mbar_wait(&ctl.empty[s.slot], s.phase ^ 1)) {
            ok = false;
            break;
          }
          if (rank == 0) ptx::mbar_arrive_expect_tx(&ctl.full[s.slot], kCtas * stage_bytes);
          const uint32_t dst = ptx::smem_u32(smem + s.slot * stage_bytes), bar = G::shared_bar(&ctl.full[s.slot], leader);
          if (!kW4) load_weights<kCtas, kGated>(dst, &map_w, n * 64, t.m_tile, bar);
          G::tma_2d(dst + kStageA<kW4>, &map_x, n * 64, row, bar);
          s.next(n_stages);
        }
      }
      // the commits that free the last stages arrive here too: see them land before leaving
      for (int i = 0; i < n_stages && ok; ++i) {
        if (!ptx::mbar_wait(&ctl.empty[s.slot], s.phase ^ 1)) ok = false;
        s.next(n_stages);
      }
    }
  } else if (kW4 && warp >= kDeqWarp0 && warp < kEpiWarp0<kW4>) {
    chain_wait();
    // Up to four groups of four warps take the chunks (of all tiles, one sequence here) in turn, thread =
    // weight row. A group may only wait for a stage whose use before last is known to be over, as
    // the phases of a barrier are told apart by parity alone: two stages a group fit the ring.
    const int groups = min(4, n_stages / 2), group = (warp - kDeqWarp0) >> 2;
    const int r = (warp & 3) * 32 + lane;
    const Tile any = tile_of<kCtas>(a.p, team, rank, split);
    const int n = team < total && group < groups ? ((total - team + teams - 1) / teams) * (any.c1 - any.c0) : 0;
    Pos q, s;
    q.skip(group, kCodes);
    s.skip(2 * group, n_stages);
    uint4 code[4];
    uint2 sc;
    auto fetch = [&] {   // this group's next codes and scales into registers
      if (!warp_wait(&ctl.code_full[q.slot], q.phase)) ok = false;
      const uint8_t* src = codes + q.slot * kCodeBytes;
#pragma unroll
      for (int k = 0; k < 4; ++k) code[k] = *reinterpret_cast<const uint4*>(src + r * kRowCodeBytes + 16 * code_slot(r, k));
      sc = *reinterpret_cast<const uint2*>(src + kTileCodeBytes + r * kRowScaleBytes);
    };
    if (group < n) fetch();
    for (int i = group; i < n && ok; i += groups) {
      Pos at = s;
      int slots[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {   // a stage is half of the chunk
        const uint32_t sch = h ? sc.y : sc.x;
        uint32_t scale[4], v[32];
        expand_scales<kHalf>(sch & 0xFFFF, scale[0], scale[1]);
        expand_scales<kHalf>(sch >> 16, scale[2], scale[3]);
        if (!warp_wait(&ctl.empty[at.slot], at.phase ^ 1)) ok = false;   // (then it runs on over what is there)
        ptx::tc_fence_after();   // the MMAs that read this stage before
        const uint32_t word[8] = {code[2 * h].x,     code[2 * h].y,     code[2 * h].z,     code[2 * h].w,
                                  code[2 * h + 1].x, code[2 * h + 1].y, code[2 * h + 1].z, code[2 * h + 1].w};
#pragma unroll
        for (int k = 0; k < 8; ++k)
          dequant_word<kHalf>(word[k], scale[k >> 1], a.l.m16, a.l.m64, *reinterpret_cast<uint32_t(*)[4]>(v + 4 * k));
        tmem_st32(a_cols + ((uint32_t)(warp & 3) << 21) + 32 * at.slot, v);
        slots[h] = at.slot;
        at.next(n_stages);
      }
      // The slot is given back only here, where the stores have taken what was made of the loaded values.
      // An arrival does not wait for loads before it: with the epilogue's accesses to a large output
      // in the queue ahead of them (2^20 tokens) the next copy overtook them.
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&ctl.code_empty[q.slot]);
      q.skip(groups, kCodes);
      if (i + groups < n) fetch();  // while the stores are on their way
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane < 2) G::arrive(&ctl.full[lane ? slots[1] : slots[0]], leader);
      s.skip(2 * groups, n_stages);
    }
  } else if (warp >= kEpiWarp0<kW4>) {
    chain_wait();
    if (splits == 1) {
      int it = 0;
      for (int w = team; w < total && ok; w += teams, ++it) {
        const Tile t = tile_of<kCtas>(a.p, w, rank, split);
        first_addend(t);
        if (!warp_wait_sleep(&ctl.acc_full[it & 1], (it >> 1) & 1)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        tile_epilogue(t, it & 1);
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) G::arrive(&ctl.acc_empty[it & 1], leader);
      }
    } else {
      first_addend(tile_of<kCtas>(a.p, team, rank, split));
      if (!warp_wait_sleep(&ctl.acc_full[0], 0)) ok = false;
      ptx::tc_fence_after();
    }
  }
  if (!ok) give_up(a.error_flag);
  __syncwarp();
  if (splits > 1) {
    const Tile t = tile_of<kCtas>(a.p, team, rank, split);
    cluster_sync();   // every group's MMAs are done, and with them the reads of the rings
    if (warp >= kEpiWarp0<kW4>) {
      const uint32_t acc = tmem + ((uint32_t)quarter << 21);
      const int n_tok = min(a.p.bn, a.l.tokens - t.tok0);
      for (int c = 0; c < n_tok; c += 32) {
        const int owner = c / 32 % splits;
        if (owner == split) continue;
        float lo[16], hi[16];
        tmem_ld_frag(acc + c, lo);
        tmem_ld_frag(acc + c + (16u << 16), hi);
        ptx::tmem_wait_ld();
        const uint32_t to = map_rank(received(smem, split - (split > owner), c / step), kCtas * owner + rank);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float* v = i < 4 ? lo + 4 * i : hi + 4 * (i - 4);
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to + i * 512), "f"(v[0]), "f"(v[1]),
                       "f"(v[2]), "f"(v[3])
                       : "memory");
        }
      }
    }
    cluster_sync();
    if (warp >= kEpiWarp0<kW4>) tile_epilogue(t, 0);
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  // a pair's MMAs read both CTAs' shared memory, commits write both CTAs' barriers
  if (kCtas > 1) cluster_sync_relaxed();
  ptx::tc_fence_after();
  if (warp == 1) G::dealloc(tmem, kTmemCols);
}

constexpr int kSms = 148;

// Clusters of this many CTAs that are resident together (SMs come in groups of 16 to 20).
constexpr int clusters_of(int ctas) {
  return ctas == 1 ? kSms : ctas == 2 ? kSms / 2 : ctas == 4 ? 33 : ctas == 6 ? 22 : ctas == 8 ? 15 : 0;
}

// Groups of one CTA or two, token tile and split of K from the sizes alone: the least estimated time in
// SM clocks. A 64-k stage costs its MMAs (2 bn) or more: NVFP4 what dequantisation and MMAs together
// measured (400 + 1.2 bn for a CTA, 380 + 0.86 bn for a pair, whose B is shared) or the ring's latency
// over its depth (~2400 from a freed stage over dequantisation, arrival, MMA and commit to the next
// free one); 16 bits its loads (~60 B per clock and SM from L2) and its MMAs' issue (~200, a pair's
// ~295). A tile's start and epilogue take 2000 + 8 per token, a split's exchange with two cluster
// barriers, which wait for the slowest group, 4500 + 8 per token.
template <bool kW4>
GemmPlan make_plan(int tokens, int padded_rows, int units, double* cost_out = nullptr) {
  constexpr int kUnit = kW4 ? 2 : 1;
  GemmPlan best{};
  double best_cost = 0;
  for (int ctas = 1; ctas <= 2; ++ctas)
    for (int bn = 32; bn <= 128 * ctas; bn += 32) {
      GemmPlan p;
      p.ctas = ctas;
      p.bn = bn;
      p.tiles_m = (padded_rows + kTileM * ctas - 1) / (kTileM * ctas);
      p.tiles_n = (tokens + bn - 1) / bn;
      p.units = units;
      const long long tiles = (long long)p.tiles_m * p.tiles_n;
      for (int s = 1; s * ctas <= 8; ++s) {
        const int room = clusters_of(s * ctas);
        if (room == 0 || (s > 1 && (tiles > room || kUnit * units / s < 4))) continue;
        p.units_per_split = (units + s - 1) / s;
        if ((units + p.units_per_split - 1) / p.units_per_split != s) continue;   // a group would have nothing to do
        p.splits = s;
        const int stage_bytes = kStageA<kW4> + bn / ctas * 128;
        p.stages = kRingBytes<kW4> / stage_bytes;
        if (p.stages > kMaxStages) p.stages = kMaxStages;
        p.accs = tiles <= room || s > 1 ? 1 : 2;
        if (kW4) {
          const int cols = (kTmemCols - p.accs * bn) / 32;
          if (cols < 4) continue;   // two dequantising groups
          if (p.stages > cols) p.stages = cols;
        }
        double stage = kW4 ? (ctas == 1 ? 400 + 1.2 * bn : 380 + 0.86 * bn) : stage_bytes / 60.0;
        if (kW4 && 2400.0 / p.stages > stage) stage = 2400.0 / p.stages;
        if (!kW4 && stage < (ctas == 1 ? 200 : 295)) stage = ctas == 1 ? 200 : 295;
        if (2.0 * bn > stage) stage = 2.0 * bn;
        const double waves = (double)((tiles + room - 1) / room);
        double cost = waves * (kUnit * p.units_per_split * stage) + 2000 + 8.0 * bn;
        if (s > 1) cost += 4500 + 8.0 * bn;
        if (best.bn == 0 || cost < best_cost) {
          best = p;
          best_cost = cost;
        }
      }
    }
  if (cost_out) *cost_out = best_cost;
  return best;
}

template <int kCtas, bool kW4, bool kHalf, bool kGated>
int launch(const CUtensorMap& mx, const CUtensorMap& mw, const Args& a, cudaStream_t st) {
  static bool set[64] = {};  // per device: the attribute belongs to its context
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const auto kernel = swap_gemm<kCtas, kW4, kHalf, kGated>;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem<kW4>);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  const int tiles = a.p.tiles_m * a.p.tiles_n;
  const int teams = a.p.splits > 1 || tiles < kSms / kCtas ? tiles : kSms / kCtas;
  return launch_chained(kernel, dim3(kCtas * a.p.splits * teams), dim3(kThreads<kW4>), kSmem<kW4>, st,
                        kCtas * a.p.splits, mx, mw, a);
}

template <int kCtas, bool kW4>
int launch_typed(const CUtensorMap& mx, const CUtensorMap& mw, const Args& a, int dtype, bool gated, cudaStream_t st) {
  if (dtype == kFp16)
    return gated ? launch<kCtas, kW4, true, true>(mx, mw, a, st) : launch<kCtas, kW4, true, false>(mx, mw, a, st);
  return gated ? launch<kCtas, kW4, false, true>(mx, mw, a, st) : launch<kCtas, kW4, false, false>(mx, mw, a, st);
}

template <bool kW4>
int launch_any(const LinearArgs& l, const GemmPlan& p, const CUtensorMap& mw, int dtype, bool gated, int* error_flag,
               cudaStream_t st) {
  Args a{};
  a.l = l;
  a.p = p;
  if ((long long)p.tiles_m * p.tiles_n > (1 << 28)) return MUSE_ERR_UNSUPPORTED_SHAPE;
  const uint32_t type = dtype == kBf16 ? 1u : 0u;  // operand format: 0 f16, 1 bf16
  a.idesc = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(p.bn >> 3) << 17) |
            ((uint32_t)(kTileM * p.ctas >> 4) << 24);
  a.b_bytes = (uint32_t)p.bn / p.ctas * 128;
  auto vec = [](const void* q, long long ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 8 == 0; };
  a.out_vec = vec(l.out, l.ldo);
  a.add_vec = vec(l.add, l.ld_add);
  a.error_flag = error_flag;
  CUtensorMap mx;
  const int rc = make_operand_map(&mx, DenseOperand{l.x, l.ldx, true}, l.tokens, l.cols, dtype, p.bn / p.ctas);
  if (rc) return rc;
  return p.ctas == 2 ? launch_typed<2, kW4>(mx, mw, a, dtype, gated, st) : launch_typed<1, kW4>(mx, mw, a, dtype, gated, st);
}

PlanInfo info(const GemmPlan& p) {
  const long long tiles = (long long)p.tiles_m * p.tiles_n, groups = kSms / p.ctas;
  return {1, p.bn, tiles, p.splits > 1 ? 0 : tiles, p.splits, p.splits > 1 ? 1 : (tiles + groups - 1) / groups};
}

int padded_rows_of(const DenseGemm& g) { return (g.n + kTileM - 1) / kTileM * kTileM; }

}  // namespace

int launch_linear_gemm(const LinearArgs& l, int dtype, bool gated, int* error_flag, cudaStream_t st) {
  return launch_any<true>(l, make_plan<true>(l.tokens, l.padded_rows, l.k_chunks), CUtensorMap{}, dtype, gated, error_flag, st);
}

PlanInfo linear_gemm_plan(int tokens, int padded_rows, int k_chunks) {
  return info(make_plan<true>(tokens, padded_rows, k_chunks));
}

PlanInfo swap_dense_plan(int m, int n, int k) {
  return info(make_plan<false>(m, (n + kTileM - 1) / kTileM * kTileM, (k + 63) / 64));
}

double swap_dense_cost(int m, int n, int k) {
  double cost;
  make_plan<false>(m, (n + kTileM - 1) / kTileM * kTileM, (k + 63) / 64, &cost);
  return cost;
}

int launch_swap_dense(const DenseGemm& g, cudaStream_t st) {
  const bool gated = g.mode == kGate;
  LinearArgs l{};
  l.x = static_cast<const uint16_t*>(g.a.ptr);
  l.ldx = g.a.ld;
  l.add = static_cast<const uint16_t*>(g.add);
  l.ld_add = g.ld_add;
  l.out = static_cast<uint16_t*>(g.out);
  l.ldo = g.ldo;
  l.tokens = g.m;
  l.cols = g.k;
  l.n_out = gated ? g.n / 2 : g.n;
  l.ab = gated ? g.ab : nullptr;
  l.padded_rows = padded_rows_of(g);
  CUtensorMap mw;
  const int rc = gated ? make_gated_map(&mw, g.b, l.n_out, g.k, g.dtype)
                       : make_operand_map(&mw, g.b, g.n, g.k, g.dtype, kTileM);
  if (rc) return rc;
  return launch_any<false>(l, make_plan<false>(g.m, l.padded_rows, (g.k + 63) / 64), mw, g.dtype, gated, g.error_flag, st);
}

}  // namespace muse
