// Dense 16-bit matrix products on the 5th-generation tensor cores (tcgen05, sm_100a), for the
// gated feed-forward block: D[m, n] = sum_k A[m, k] B[n, k], fp32 accumulators in tensor memory.
//
//   forward   ab = x . W13^T (A, B along k)      epilogue h = silu(a) * b, ab kept in fp32 to train
//             y  = h . W2^T                      epilogue + add
//   backward  dh = dy . W2 (B along n)           epilogue da, db, h from ab
//             dx = [da db] . W13 (B along n);  dW13 = [da db]^T x, dW2 = dy^T h (A along m, B along n)
//
// A CTA pair (cluster of two, cta_group::2) computes a 256 x bn tile (bn <= 256): each CTA loads
// its own 128 rows of A and half of B's columns, one thread of the leader issues M = 256 MMAs that
// read both halves, so an SM fetches 32 KB for 2 * 128 * 256 * 64 operations and the two operands'
// shared-memory reads stay below the port's rate. Operands that run along m or n are fetched as
// they lie (64-wide boxes, "MN-major" descriptors): no transposed copy is made.
// Six ring stages of 64 k; two accumulators of 256 columns, so a tile's epilogue (eight warps)
// overlaps the next tile's MMAs. Pairs are persistent and walk a static tile list, eight row tiles
// to a group, so that the tiles in flight share their operands in L2. Tiles that do not
// fill a wave of the pairs are split along K and their fp32 partials summed, in split order, by a
// second kernel: results do not depend on timing.
// In the gate product the leader's half of B is gate rows and its peer's half the matching up
// rows, so one thread holds a and b of the same element.
// Bound by the tensor pipe, which is 88 to 94 % busy in the products of a 4096-token step (dy . W2: 74 %,
// its 128 tiles are 1.7 waves and its epilogue the longest), and in a loop by the card's power: the
// step's six products take 862 us, 1.26 PFLOP/s, the library's six without the epilogues 896 us.
#undef MUSE_TRACE  // these kernels record no stamps
#include "dense.cuh"

#include <cudaTypedefs.h>

#include "kernels.cuh"
#include "pair.cuh"

namespace muse {
namespace {

constexpr int kBm = 128;                  // rows of A per CTA (256 per pair)
constexpr int kBk = 64;                   // k per stage: one 128-byte swizzle row
constexpr int kMaxBn = 256;
constexpr int kStages = 6;
constexpr int kABytes = kBm * kBk * 2;    // 16 KiB
constexpr int kBBytes = kMaxBn / 2 * kBk * 2;
constexpr int kStageBytes = kABytes + kBBytes;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 32 * (2 + kEpiWarps);
constexpr int kPatch = 32 * 32 * 4;       // one epilogue warp's 32 x 32 fp32 staging patch
constexpr int kGroupM = 8;                // row tiles per raster group

struct Ctl {
  uint64_t full[kStages], empty[kStages];
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem;
};
constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kEpiWarps * kPatch + sizeof(Ctl);
static_assert(kSmem <= 232448, "shared memory of one CTA");

struct Args {
  int m, n, inter;                    // inter: I of the gate modes (0 otherwise)
  int bn, tiles_m, tiles_n, kb_total;
  int whole, splits, kb_per_split;    // tiles done whole; the others (the tail) in `splits` items each
  int dtype;
  uint32_t idesc;
  uint32_t tx_bytes;                  // both CTAs' bytes per stage
  void* out;
  long long ldo;
  const void* add;
  long long ld_add;
  float* ab;
  void* h_out;
  float* partials;
  int* error_flag;
};

struct Tile {
  int m0, n0, kb0, kb1;
  float* partial;  // an item of the tail: its 256 x bn block of partial sums (else null)
};
// Tile `idx` of the raster: kGroupM row tiles per column tile. n0 is the column tile's index.
__device__ __forceinline__ void raster(const Args& a, int idx, int& m0, int& n0) {
  const int group = idx / (kGroupM * a.tiles_n);
  const int first = group * kGroupM;
  const int rows = min(kGroupM, a.tiles_m - first);
  const int r = idx - group * kGroupM * a.tiles_n;
  m0 = (first + r % rows) * 2 * kBm;
  n0 = r / rows;
}
// Work items: the whole tiles, then the tail's, splits innermost.
__device__ __forceinline__ Tile tile_of(const Args& a, int w) {
  Tile t;
  int idx = w;
  t.kb0 = 0;
  t.kb1 = a.kb_total;
  t.partial = nullptr;
  if (w >= a.whole && a.splits > 1) {
    const int item = w - a.whole, split = item % a.splits;
    idx = a.whole + item / a.splits;
    t.kb0 = split * a.kb_per_split;
    t.kb1 = min(a.kb_total, t.kb0 + a.kb_per_split);
    t.partial = a.partials + (size_t)item * 2 * kBm * a.bn;
  }
  raster(a, idx, t.m0, t.n0);
  return t;
}

__device__ __forceinline__ void store4(int dtype, void* base, long long ld, int row, int col, float4 v) {
  uint2 p;
  p.x = pack16(dtype, v.x, v.y);
  p.y = pack16(dtype, v.z, v.w);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(base) + (size_t)row * ld + col) = p;
}
__device__ __forceinline__ uint2 load4(const void* base, long long ld, int row, int col) {
  return __ldcg(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(base) + (size_t)row * ld + col));
}
__device__ __forceinline__ float4 add4(int dtype, uint2 p, float4 v) {
  const float2 lo = unpack16(dtype, p.x), hi = unpack16(dtype, p.y);
  return make_float4(v.x + lo.x, v.y + lo.y, v.z + hi.x, v.w + hi.y);
}
// da, db and h of four elements from dh, a, b:  s = 1 / (1 + exp(-a)),
// da = dh * b * s * (1 + a * (1 - s)), db = dh * a * s, h = a * s * b.
__device__ __forceinline__ void dgate1(float dh, float a, float b, float& da, float& db, float& h) {
  const float s = sigmoid_f(a);
  const float as = a * s;
  da = dh * b * (s + as * (1.f - s));
  db = dh * as;
  h = as * b;
}
__device__ __forceinline__ void dgate4(const Args& p, int row, int col, float4 dh, float4 a, float4 b) {
  float4 da, db, h;
  dgate1(dh.x, a.x, b.x, da.x, db.x, h.x);
  dgate1(dh.y, a.y, b.y, da.y, db.y, h.y);
  dgate1(dh.z, a.z, b.z, da.z, db.z, h.z);
  dgate1(dh.w, a.w, b.w, da.w, db.w, h.w);
  store4(p.dtype, p.out, p.ldo, row, col, da);
  store4(p.dtype, p.out, p.ldo, row, p.inter + col, db);
  store4(p.dtype, p.h_out, p.inter, row, col, h);
}

// What a patch is combined with, one 4-column piece for each of a lane's eight rows: the addend, or a
// and b.
template <int kMode> struct SideInput {
  uint2 add[8];
  // every second 128-byte line of a row (the quarter's other warp takes the others)
  static __device__ __forceinline__ void prefetch(const Args& p, int row, int col, int end) {
    if (p.add)
      for (; col < end; col += 128) prefetch_l2(static_cast<const uint16_t*>(p.add) + (size_t)row * p.ld_add + col);
  }
  __device__ __forceinline__ void load(const Args& p, int i, int row, int col, bool more) {
    if (p.add && more && row < p.m && col < p.n) add[i] = load4(p.add, p.ld_add, row, col);
  }
};
template <> struct SideInput<kDGate> {
  float4 a[8], b[8];
  static __device__ __forceinline__ void prefetch(const Args& p, int row, int col, int end) {
    for (; col < end; col += 128)
      for (int i = 0; i < 64 && col + i < end; i += 32) {
        prefetch_l2(p.ab + (size_t)row * 2 * p.inter + col + i);
        prefetch_l2(p.ab + (size_t)row * 2 * p.inter + p.inter + col + i);
      }
  }
  __device__ __forceinline__ void load(const Args& p, int i, int row, int col, bool more) {
    if (more && row < p.m && col < p.n) {
      const float* at = p.ab + (size_t)row * 2 * p.inter + col;
      a[i] = __ldcg(reinterpret_cast<const float4*>(at));
      b[i] = __ldcg(reinterpret_cast<const float4*>(at + p.inter));
    }
  }
};
template <> struct SideInput<kGate> {
  static __device__ __forceinline__ void prefetch(const Args&, int, int, int) {}
  __device__ __forceinline__ void load(const Args&, int, int, int, bool) {}
};

// 32 x 32 fp32 patch of one warp: thread = row writes its 32 columns, then lane l reads columns
// 4 (l % 8) .. + 3 of row 4 i + l / 8. 16-byte pieces are swizzled by the row: no bank conflicts.
__device__ __forceinline__ void patch_put(uint8_t* patch, int lane, const float (&v)[32]) {
#pragma unroll
  for (int p = 0; p < 8; ++p)
    *reinterpret_cast<float4*>(patch + lane * 128 + ((p ^ (lane & 7)) << 4)) =
        make_float4(v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]);
}
__device__ __forceinline__ float4 patch_get(const uint8_t* patch, int lane, int i) {
  const int row = 4 * i + (lane >> 3), p = lane & 7;
  return *reinterpret_cast<const float4*>(patch + row * 128 + ((p ^ (row & 7)) << 4));
}

template <bool kAMn, bool kBMn, int kMode>
__global__ void __launch_bounds__(kThreads, 1)
dense_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* patches = smem + kStages * kStageBytes;
  Ctl& ctl = *reinterpret_cast<Ctl*>(patches + kEpiWarps * kPatch);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int total = a.whole + (a.tiles_m * a.tiles_n - a.whole) * a.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      ptx::mbar_init(&ctl.full[s], 1);
      ptx::mbar_init(&ctl.empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      ptx::mbar_init(&ctl.acc_full[b], 1);
      ptx::mbar_init(&ctl.acc_empty[b], 2 * kEpiWarps);
    }
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&map_a);
    ptx::prefetch_tensormap(&map_b);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(ptx::smem_u32(&ctl.tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  ptx::tc_fence_before();
  __syncthreads();
  cluster_sync();
  ptx::tc_fence_after();
  const uint32_t tmem = ctl.tmem;
  chain_release();
  chain_wait();

  bool ok = true;
  if (warp == 0) {
    if (ptx::elect_one()) {
      int slot = 0;
      uint32_t phase = 0;
      for (int w = pair; w < total && ok; w += pairs) {
        const Tile t = tile_of(a, w);
        const int row = t.m0 + rank * kBm;
        const int half = a.bn >> 1;
        int col;
        if (kMode == kGate) col = rank * a.inter + t.n0 * half;
        else col = t.n0 * a.bn + rank * half;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ptx::mbar_wait(&ctl.empty[slot], phase ^ 1)) {
            ok = false;
            break;
          }
          const uint32_t sa = ptx::smem_u32(smem + slot * kStageBytes), sb = sa + kABytes;
          const uint32_t bar = map_rank(&ctl.full[slot], 0);
          if (rank == 0) ptx::mbar_arrive_expect_tx(&ctl.full[slot], a.tx_bytes);
          if (kAMn) {
            tma_pair(sa, &map_a, row, kb * kBk, bar);
            tma_pair(sa + 8192, &map_a, row + 64, kb * kBk, bar);
          } else {
            tma_pair(sa, &map_a, kb * kBk, row, bar);
          }
          if (kBMn) {
            tma_pair(sb, &map_b, col, kb * kBk, bar);
            if (half > 64) tma_pair(sb + 8192, &map_b, col + 64, kb * kBk, bar);
          } else {
            tma_pair(sb, &map_b, kb * kBk, col, bar);
          }
          if (++slot == kStages) {
            slot = 0;
            phase ^= 1;
          }
        }
      }
      // the commits that free the last stages arrive here too: see them land before leaving
      for (int s = 0; s < kStages && ok; ++s) {
        if (!ptx::mbar_wait(&ctl.empty[slot], phase ^ 1)) ok = false;
        if (++slot == kStages) {
          slot = 0;
          phase ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      int slot = 0, it = 0;
      uint32_t phase = 0;
      for (int w = pair; w < total && ok; w += pairs, ++it) {
        const Tile t = tile_of(a, w);
        const int buf = it & 1;
        if (!ptx::mbar_wait(&ctl.acc_empty[buf], ((it >> 1) & 1) ^ 1)) {
          ok = false;
          break;
        }
        ptx::tc_fence_after();
        const uint32_t d = tmem + buf * kMaxBn;
        for (int kb = t.kb0; kb < t.kb1; ++kb) {
          if (!ptx::mbar_wait(&ctl.full[slot], phase)) {
            ok = false;
            break;
          }
          ptx::tc_fence_after();
          const uint32_t sa = ptx::smem_u32(smem + slot * kStageBytes);
          const uint64_t da = operand_desc<kAMn>(sa), db = operand_desc<kBMn>(sa + kABytes);
#pragma unroll
          for (int j = 0; j < kBk / 16; ++j)
            mma_pair(d, da + j * kStepDesc<kAMn>, db + j * kStepDesc<kBMn>, a.idesc, kb > t.kb0 || j > 0);
          commit_pair(&ctl.empty[slot]);
          if (++slot == kStages) {
            slot = 0;
            phase ^= 1;
          }
        }
        commit_pair(&ctl.acc_full[buf]);
      }
    }
  } else {
    const int e = warp - 2, quarter = warp & 3, half = e >> 2;
    uint8_t* patch = patches + e * kPatch;
    const uint32_t lane_base = tmem + ((uint32_t)quarter << 21);
    const int rr = lane >> 3, cc = (lane & 7) * 4;
    int it = 0;
    for (int w = pair; w < total; w += pairs, ++it) {
      const Tile t = tile_of(a, w);
      const int buf = it & 1;
      // what the tile is combined with starts for L2, and for the first patch for registers, while the
      // sums are still being taken
      SideInput<kMode> side;
      if (!t.partial) {
        const int row = t.m0 + rank * kBm + quarter * 32 + lane;
        if (row < a.m) SideInput<kMode>::prefetch(a, row, t.n0 * a.bn + half * 64, min(a.n, (t.n0 + 1) * a.bn));
#pragma unroll
        for (int i = 0; i < 8; ++i)
          side.load(a, i, t.m0 + rank * kBm + quarter * 32 + 4 * i + rr, t.n0 * a.bn + 32 * half + cc, true);
      }
      if (!warp_wait_sleep(&ctl.acc_full[buf], (it >> 1) & 1)) {
        ok = false;
        break;
      }
      ptx::tc_fence_after();
      const uint32_t acc = lane_base + buf * kMaxBn;
      const int row0 = t.m0 + rank * kBm + quarter * 32;
      const bool rows = row0 < a.m;        // a warp whose rows all lie past the end stores nothing
      // rows 4 i + rr of the patch, columns cc .. cc + 3, for every i whose row exists
      auto each = [&](const float (&v)[32], auto&& f) {
        __syncwarp();
        patch_put(patch, lane, v);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (row0 + 4 * i + rr < a.m) f(row0 + 4 * i + rr, patch_get(patch, lane, i));
      };
      if (rows && kMode == kGate) {
        const int pairs_cols = a.bn >> 1;  // gate columns of the tile; the up columns follow
        for (int c = 32 * half; c < pairs_cols; c += 64) {
          const int col = t.n0 * pairs_cols + c + cc;
          if (t.n0 * pairs_cols + c >= a.inter) break;
          float g[32], u[32];
          tmem_ld32(acc + c, g);
          tmem_ld32(acc + pairs_cols + c, u);
          ptx::tmem_wait_ld();
          const bool in = col < a.inter;
          if (t.partial) {
            float* to = t.partial + (size_t)(rank * kBm + quarter * 32) * a.bn + c + cc;
            each(g, [&](int r, float4 v) { *reinterpret_cast<float4*>(to + (size_t)(r - row0) * a.bn) = v; });
            each(u, [&](int r, float4 v) { *reinterpret_cast<float4*>(to + (size_t)(r - row0) * a.bn + pairs_cols) = v; });
            continue;
          }
          if (a.ab) {
            each(g, [&](int r, float4 v) {
              if (in) *reinterpret_cast<float4*>(a.ab + (size_t)r * a.n + col) = v;
            });
            each(u, [&](int r, float4 v) {
              if (in) *reinterpret_cast<float4*>(a.ab + (size_t)r * a.n + a.inter + col) = v;
            });
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = silu_f(g[j]) * u[j];
          each(g, [&](int r, float4 v) {
            if (in) store4(a.dtype, a.out, a.ldo, r, col, v);
          });
        }
      } else if (rows) {
        for (int c = 32 * half; c < a.bn; c += 64) {
          const int col = t.n0 * a.bn + c + cc;
          if (t.n0 * a.bn + c >= a.n) break;
          const bool in = col < a.n;
          float v[32];
          tmem_ld32(acc + c, v);
          ptx::tmem_wait_ld();
          __syncwarp();
          patch_put(patch, lane, v);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = row0 + 4 * i + rr;
            float4 x = patch_get(patch, lane, i);
            if (t.partial) {
              if (r < a.m && in)
                *reinterpret_cast<float4*>(t.partial + (size_t)(r - t.m0) * a.bn + c + cc) = x;
              continue;
            }
            if (r < a.m && in) {
              if constexpr (kMode == kDGate) {
                dgate4(a, r, col, x, side.a[i], side.b[i]);
              } else if constexpr (kMode == kStore) {
                if (a.add) x = add4(a.dtype, side.add[i], x);
                store4(a.dtype, a.out, a.ldo, r, col, x);
              }
            }
          }
          // the next patch's, all after the last use: loads and uses in turn would wait for one another
          if (!t.partial) {
#pragma unroll
            for (int i = 0; i < 8; ++i) side.load(a, i, row0 + 4 * i + rr, col + 64, c + 64 < a.bn);
          }
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(map_rank(&ctl.acc_empty[buf], 0));
    }
  }
  if (!ok) give_up(a.error_flag);
  __syncwarp();
  ptx::tc_fence_before();
  __syncthreads();
  cluster_sync_relaxed();  // the pair's MMAs read both CTAs' shared memory, commits write both CTAs' barriers
  ptx::tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Sums of the tail's partials, in split order, with the mode's epilogue: a block takes eight rows of
// a tile, a thread four columns at a time. The partials were just written and are read from L2.
constexpr int kReduceRows = 8;

template <int kMode>
__global__ void __launch_bounds__(256) dense_reduce(const Args a) {
  chain_release();
  chain_wait();
  int m0, n0;
  raster(a, a.whole + blockIdx.x, m0, n0);
  const int width = kMode == kGate ? a.bn >> 1 : a.bn;
  const int q = width >> 2;
  const size_t plane = (size_t)2 * kBm * a.bn;
  const float* tile = a.partials + (size_t)blockIdx.x * a.splits * plane;
  const int last = kMode == kGate ? a.inter : a.n;
  for (int i = threadIdx.x; i < kReduceRows * q; i += 256) {
    const int r = blockIdx.y * kReduceRows + i / q, c = i % q * 4;
    const int row = m0 + r, col = n0 * width + c;
    if (row >= a.m || col >= last) continue;
    auto sum = [&](int at) {
      const float* p = tile + (size_t)r * a.bn + at;
      float4 s = __ldcg(reinterpret_cast<const float4*>(p));
#pragma unroll 4
      for (int k = 1; k < a.splits; ++k) {
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p + k * plane));
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      return s;
    };
    float4 x = sum(c);
    if (kMode == kGate) {
      const float4 u = sum(width + c);
      if (a.ab) {
        float* at = a.ab + (size_t)row * a.n + col;
        *reinterpret_cast<float4*>(at) = x;
        *reinterpret_cast<float4*>(at + a.inter) = u;
      }
      x = make_float4(silu_f(x.x) * u.x, silu_f(x.y) * u.y, silu_f(x.z) * u.z, silu_f(x.w) * u.w);
      store4(a.dtype, a.out, a.ldo, row, col, x);
    } else if (kMode == kDGate) {
      const float* at = a.ab + (size_t)row * 2 * a.inter + col;
      dgate4(a, row, col, x, __ldcg(reinterpret_cast<const float4*>(at)),
             __ldcg(reinterpret_cast<const float4*>(at + a.inter)));
    } else {
      if (a.add) x = add4(a.dtype, load4(a.add, a.ld_add, row, col), x);
      store4(a.dtype, a.out, a.ldo, row, col, x);
    }
  }
}

constexpr int kPairs = 74;  // 148 SMs, two to a pair

struct Plan {
  int bn, tiles_m, tiles_n, kb_total, whole, splits, kb_per_split;
  int tail() const { return splits > 1 ? (int)((long long)tiles_m * tiles_n - whole) : 0; }
};

// Tile width, and the split of K for the tail: the tiles that do not fill a wave of all pairs are cut
// along K into one item per pair (448 tiles, as a 4096-token step has, would else pay a seventh wave
// for its last four). Chosen from the sizes alone, by the least estimated time in SM clocks. A stage
// of a pair costs the larger of its MMA time (2 bn clocks for 64 k) and its loads ((128 + bn / 2)
// rows of 128 B at ~60 B per clock and SM from L2); a tile's start and last epilogue ~2500; a split
// adds the reduction's launch and its partials' way through L2 (~2 KB per clock over the chip).
Plan make_plan(int m, int n, int k, int mode, bool b_k_major, double* cost_out = nullptr) {
  Plan best{};
  double best_cost = 0;
  const int kb = (k + kBk - 1) / kBk;
  for (int bn = 256; bn >= 64; bn -= 32) {
    if (!b_k_major && bn != 256 && bn != 128) continue;
    if (mode == kGate && bn % 64) continue;
    Plan p;
    p.bn = bn;
    p.tiles_m = (m + 2 * kBm - 1) / (2 * kBm);
    p.tiles_n = (n + bn - 1) / bn;
    if (mode == kGate) p.tiles_n = (n / 2 + bn / 2 - 1) / (bn / 2);
    p.kb_total = kb;
    const long long tiles = (long long)p.tiles_m * p.tiles_n, tail = tiles % kPairs;
    const double stage = 2.0 * bn > (128 + bn / 2) * 128 / 60.0 ? 2.0 * bn : (128 + bn / 2) * 128 / 60.0;
    for (int s = 1; s <= 16 && (s == 1 || (tail * s <= kPairs && kb / s >= 4 && tail > 0)); ++s) {
      p.kb_per_split = (kb + s - 1) / s;
      p.splits = (kb + p.kb_per_split - 1) / p.kb_per_split;
      p.whole = (int)(p.splits > 1 ? tiles - tail : tiles);
      double cost = (double)(tiles / kPairs) * kb * stage + 2500;
      if (tail) cost += p.kb_per_split * stage;
      if (p.splits > 1) cost += 4000 + 8.0 * 256 * bn * tail * p.splits / 2000;
      if (best.bn == 0 || cost < best_cost) {
        best = p;
        best_cost = cost;
      }
    }
  }
  if (cost_out) *cost_out = best_cost;
  return best;
}

template <bool kAMn, bool kBMn, int kMode>
int launch(const CUtensorMap& ma, const CUtensorMap& mb, const Args& a, cudaStream_t st) {
  // once per device and kernel: the attribute belongs to the device's context
  static bool set[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !set[dev]) {
    e = cudaFuncSetAttribute(dense_gemm<kAMn, kBMn, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) set[dev] = true;
  }
  const int tail = a.splits > 1 ? a.tiles_m * a.tiles_n - a.whole : 0;
  const int total = a.whole + tail * a.splits;
  const int pairs = total < kPairs ? total : kPairs;
  int rc = launch_chained(dense_gemm<kAMn, kBMn, kMode>, dim3(2 * pairs), dim3(kThreads), kSmem, st, 2, ma, mb, a);
  if (rc || !tail) return rc;
  return launch_chained(dense_reduce<kMode>, dim3(tail, 2 * kBm / kReduceRows), dim3(256), 0, st, 1, a);
}

}  // namespace

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// Map of an operand with `extent` m (or n) and k: boxes of 64 k x box rows (K-major) or of
// 64 m x 64 k.
int make_operand_map(CUtensorMap* map, const DenseOperand& o, int extent, int k, int dtype, int box) {
  const auto encode = encode_fn();
  if (!encode) return MUSE_ERR_NO_DEVICE;
  cuuint64_t dims[2] = {(cuuint64_t)(o.k_major ? k : extent), (cuuint64_t)(o.k_major ? extent : k)};
  cuuint64_t strides[1] = {(cuuint64_t)o.ld * 2};
  cuuint32_t boxes[2] = {64, (cuuint32_t)(o.k_major ? box : 64)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r =
      encode(map, dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
             const_cast<void*>(o.ptr), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MUSE_OK : MUSE_ERR_INVALID_ARGUMENT;
}

int make_gated_map(CUtensorMap* map, const DenseOperand& o, int inter, int k, int dtype) {
  const auto encode = encode_fn();
  if (!encode) return MUSE_ERR_NO_DEVICE;
  const cuuint64_t row = (cuuint64_t)o.ld * 2;
  cuuint64_t dims[4] = {(cuuint64_t)k, 8, 2, (cuuint64_t)inter / 8};
  cuuint64_t strides[3] = {row, row * inter, row * 8};
  cuuint32_t boxes[4] = {64, 8, 2, 8};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r =
      encode(map, dtype == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(o.ptr), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MUSE_OK : MUSE_ERR_INVALID_ARGUMENT;
}

double dense_cost(int m, int n, int k, int mode, bool b_k_major) {
  double cost;
  make_plan(m, n, k, mode, b_k_major, &cost);
  return cost;
}

PlanInfo dense_plan(int m, int n, int k, int mode, bool b_k_major) {
  const Plan p = make_plan(m, n, k, mode, b_k_major);
  const long long tiles = (long long)p.tiles_m * p.tiles_n, items = p.whole + (long long)p.tail() * p.splits;
  return {2, p.bn, tiles, tiles - p.tail(), p.splits, (items + kPairs - 1) / kPairs};
}

size_t dense_scratch_bytes(int m, int n, int k, int mode, bool b_k_major) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const Plan p = make_plan(m, n, k, mode, b_k_major);
  return (size_t)4 * p.tail() * p.splits * 2 * kBm * p.bn;
}

int launch_dense_gemm(const DenseGemm& g, cudaStream_t stream) {
  const Plan p = make_plan(g.m, g.n, g.k, g.mode, g.b.k_major);
  if ((long long)p.tiles_m * p.tiles_n > (1 << 30)) return MUSE_ERR_UNSUPPORTED_SHAPE;
  Args a{};
  a.m = g.m;
  a.n = g.n;
  a.inter = g.mode == kGate ? g.n / 2 : g.mode == kDGate ? g.n : 0;
  a.bn = p.bn;
  a.tiles_m = p.tiles_m;
  a.tiles_n = p.tiles_n;
  a.kb_total = p.kb_total;
  a.whole = p.whole;
  a.splits = p.splits;
  a.kb_per_split = p.kb_per_split;
  a.dtype = g.dtype;
  const uint32_t type = g.dtype == kBf16 ? 1u : 0u;  // operand format: 0 f16, 1 bf16
  a.idesc = (1u << 4) | (type << 7) | (type << 10) | ((g.a.k_major ? 0u : 1u) << 15) |
            ((g.b.k_major ? 0u : 1u) << 16) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(2 * kBm >> 4) << 24);
  a.tx_bytes = 2 * (kABytes + (uint32_t)p.bn / 2 * kBk * 2);
  a.out = g.out;
  a.ldo = g.ldo;
  a.add = g.add;
  a.ld_add = g.ld_add;
  a.ab = g.ab;
  a.h_out = g.h_out;
  a.partials = g.partials;
  a.error_flag = g.error_flag;
  if (p.tail() && !g.partials) return MUSE_ERR_WORKSPACE_TOO_SMALL;
  CUtensorMap ma, mb;
  int rc = make_operand_map(&ma, g.a, g.m, g.k, g.dtype, kBm);
  if (!rc) rc = make_operand_map(&mb, g.b, g.n, g.k, g.dtype, p.bn / 2);
  if (rc) return rc;
  if (g.a.k_major && g.b.k_major) {
    if (g.mode == kGate) return launch<false, false, kGate>(ma, mb, a, stream);
    if (g.mode == kStore) return launch<false, false, kStore>(ma, mb, a, stream);
  } else if (g.a.k_major) {
    if (g.mode == kDGate) return launch<false, true, kDGate>(ma, mb, a, stream);
    if (g.mode == kStore) return launch<false, true, kStore>(ma, mb, a, stream);
  } else if (!g.b.k_major && g.mode == kStore) {
    return launch<true, true, kStore>(ma, mb, a, stream);
  }
  return MUSE_ERR_INVALID_ARGUMENT;
}

}  // namespace muse
