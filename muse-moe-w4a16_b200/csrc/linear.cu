// y = x . W^T with an NVFP4 weight (E2M1 codes, an e4m3 scale per 16 of them along K, one fp32
// scale): the dense projections and the 4-bit shared expert beside the routed experts.
//
//   y[t, n] = gs * sum_k x[t, k] * e2m1[n, k] * e4m3[n, k / 16]     (+ add[t, n])
//   gated:  y[t, i] = silu(a) * b,  a, b = the products with gate row i and up row i
//
// The weight is kept in the routed experts' tile order (layout.cuh: 128 rows x 128 codes, permuted
// so that a code pair drops into a bf16x2 with one logic op), rows and K padded with zero codes, and
// each tile's scales behind its codes: a tile is one copy, and the tiles of one row range follow
// one another along K.
#undef MUSE_TRACE  // these kernels record no stamps
#include "few_tokens.cuh"
#include "kernels.cuh"

namespace muse {
namespace {

// ---------------------------------------------------------------------------- repack

// One CTA per (128-row tile, 128-code chunk), chunks innermost, thread = tile row. Rows and codes past the
// matrix are zero codes with zero scales. gate_up > 0: rows of gate and up interleave by 16 as
// in a w13 tile; `gate_up` is I, padded to 64 rows per half on its own.
__global__ void __launch_bounds__(kTileM)
prepare_linear_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int rows, int cols,
                      int gate_up, int k_chunks, uint8_t* __restrict__ out) {
  const int m = blockIdx.x / k_chunks, kc = blockIdx.x % k_chunks, r = threadIdx.x;
  int src = m * kTileM + r;
  bool row_ok = src < rows;
  if (gate_up > 0) {
    const int j = 64 * m + 16 * (r >> 5) + (r & 15);  // output column
    row_ok = j < gate_up;
    src = (r & 16) ? gate_up + j : j;
  }
  const size_t tile = blockIdx.x;
  uint8_t* dst = out + tile * kLinearTileBytes + r * kRowCodeBytes;
  uint8_t* sdst = out + tile * kLinearTileBytes + kTileCodeBytes + r * kRowScaleBytes;
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

int padded(int v, int to) { return (v + to - 1) / to * to; }
int padded_rows_of(int rows, int gated) { return gated ? 2 * padded(rows / 2, 64) : padded(rows, kTileM); }
long long tiles_of(int rows, int cols, int gated) {
  return (long long)(padded_rows_of(rows, gated) / kTileM) * (padded(cols, kChunkK) / kChunkK);
}

int check_linear(int rows, int cols, int gated) {
  if (rows <= 0 || cols <= 0 || (gated != 0 && gated != 1) || (gated && rows % 2)) return MUSE_ERR_INVALID_ARGUMENT;
  if (cols % kBlock || rows > (1 << 24) || cols > (1 << 24)) return MUSE_ERR_UNSUPPORTED_SHAPE;
  if (tiles_of(rows, cols, gated) > 0x7FFFFFFF) return MUSE_ERR_UNSUPPORTED_SHAPE;   // a grid's x
  return MUSE_OK;
}

bool misaligned(const void* p, unsigned to) { return reinterpret_cast<uintptr_t>(p) % to != 0; }

}  // namespace
}  // namespace muse

using namespace muse;

extern "C" int muse_moe_linear_prepared_size(int rows, int cols, int gated, size_t* bytes) {
  if (!bytes) return MUSE_ERR_INVALID_ARGUMENT;
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  *bytes = (size_t)tiles_of(rows, cols, gated) * kLinearTileBytes;
  return MUSE_OK;
}

extern "C" int muse_moe_linear_plan(int tokens, int rows, int cols, int gated, int* plan) {
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  if (!plan || tokens <= 0) return MUSE_ERR_INVALID_ARGUMENT;
  if (tokens > kMaxRows) return MUSE_ERR_UNSUPPORTED_SHAPE;
  return put_plan(streams_w4(tokens, rows, cols)
                      ? PlanInfo{}
                      : linear_gemm_plan(tokens, padded_rows_of(rows, gated), padded(cols, kChunkK) / kChunkK),
                  plan);
}

extern "C" int muse_moe_prepare_linear(const uint8_t* w, const uint8_t* w_sf, int rows, int cols, int gated,
                                       uint8_t* out, muse_stream_t stream) {
  const int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  if (!w || !w_sf || !out || misaligned(w, 8) || misaligned(out, 16)) return MUSE_ERR_INVALID_ARGUMENT;
  prepare_linear_kernel<<<(unsigned)tiles_of(rows, cols, gated), kTileM, 0, (cudaStream_t)stream>>>(
      w, w_sf, rows, cols, gated ? rows / 2 : 0, padded(cols, kChunkK) / kChunkK, out);
  return last_launch_status();
}

extern "C" int muse_moe_linear_w4(const void* x, long long ldx, int dtype, int tokens, int rows, int cols, int gated,
                                  const uint8_t* wp, const float* w_gs, const void* add,
                                  long long ld_add, void* out, long long ldo, muse_stream_t stream) {
  int rc = check_linear(rows, cols, gated);
  if (rc) return rc;
  const int n_out = gated ? rows / 2 : rows;
  if (tokens < 0 || (dtype != kBf16 && dtype != kFp16)) return MUSE_ERR_INVALID_ARGUMENT;
  if (tokens == 0) return MUSE_OK;
  if (tokens > kMaxRows) return MUSE_ERR_UNSUPPORTED_SHAPE;
  if (!x || !wp || !w_gs || !out || misaligned(x, 16) || ldx % 8 || misaligned(wp, 16) ||
      misaligned(w_gs, 4) || misaligned(add, 2) || misaligned(out, 2) ||
      (tokens > 1 && (ldx < cols || ldo < n_out || (add && ld_add < n_out))))
    return MUSE_ERR_INVALID_ARGUMENT;
  LinearArgs a{};
  a.wq = wp;
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
  int* flag = nullptr;
  if ((rc = device_status_ptr(&flag))) return rc;
  if (streams_w4(tokens, rows, cols)) return launch_few_w4(a, dtype, gated, flag, st);
  return launch_linear_gemm(a, dtype, gated, flag, st);
}
