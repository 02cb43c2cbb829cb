// Entry points of the encoder product on 8-bit rows (kernels: encode_fp8.h).
#include "encode_fp8.h"

namespace sff8 {
namespace {

using namespace sfenc;

// Up to 32 tokens: the pass over W bounds it; two waves of 32 features, five stages in flight.
typedef SlimTile<1, 1, 1, 2, 8, 6> F8x32;
// Middling sizes: 128 x 128, three stages.
typedef SlimTile<2, 2, 2, 2, 8, 3> F8x128;
// Large: 256 x 256, 8 waves of 128 x 64.
typedef SlimTile<4, 2, 2, 4, 8, 2> F8x256;

template <typename TL, int AUX>
hipError_t launch_tile(F8Args& a, hipStream_t s) {
  a.tiles_m = (int)((a.M + TL::TM - 1) / TL::TM);
  a.tiles_n = (int)((a.N + TL::TN - 1) / TL::TN);
  a.group_n = std::min(a.group_n, a.tiles_n);
  const dim3 grid(a.tiles_m * a.tiles_n), block(TL::NT);
  if (a.out_dt == SF_F32) hipLaunchKernelGGL((gemm_f8_kernel<TL, EPI_DENSE, AUX, true>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_f8_kernel<TL, EPI_DENSE, AUX, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

// 256x256 tiles of 16-bit results: the persistent form, one workgroup per CU (at most one per
// tile, whole XCD groups of eight). ctr: TILE_CTR_BYTES of the caller's workspace.
hipError_t launch_persist(F8Args& a, void* ctr, hipStream_t s) {
  a.tiles_m = (int)((a.M + BM - 1) / BM);
  a.tiles_n = (int)((a.N + BN - 1) / BN);
  a.group_n = std::min(a.group_n, a.tiles_n);
  a.tile_ctr = (int32_t*)ctr;
  const int cus = device_cus();
  if (cus <= 0) return hipErrorInvalidDevice;
  const int total = a.tiles_m * a.tiles_n;
  const dim3 grid((unsigned)std::max(8, std::min(cus / 8 * 8, (total + 7) / 8 * 8))), block(256);
  hipLaunchKernelGGL(clear_counters_kernel, dim3(1), dim3(64), 0, s, a.tile_ctr);
  const bool plain = a.act != SF_ACT_JUMPRELU && !a.row_nnz;
  if (a.out_dt == SF_F16) {
    if (plain) hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_F16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_F16, false>), grid, block, 0, s, a);
  } else {
    if (plain) hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_BF16, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_BF16, false>), grid, block, 0, s, a);
  }
  return hipGetLastError();
}

bool aligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_rows(const char* fn, const char* what, const void* q, int64_t sq, const void* scale, int64_t ss, int64_t K) {
  SF_REQUIRE(q && scale, "%s: %s: codes and scales must not be NULL", fn, what);
  SF_REQUIRE(aligned(q, 16) && sq % 16 == 0, "%s: %s: rows of codes must be 16-B aligned", fn, what);
  SF_REQUIRE(aligned(scale, 4) && ss % 4 == 0, "%s: %s: rows of scales must be 4-B aligned", fn, what);
  SF_REQUIRE(sq >= code_bytes(K) && sq <= (1 << 22), "%s: %s: rows of codes %lld bytes apart, %lld to 4194304 wanted",
             fn, what, (long long)sq, (long long)code_bytes(K));
  SF_REQUIRE(ss >= scale_bytes(K) && ss <= (1 << 22), "%s: %s: rows of scales %lld bytes apart, %lld to 4194304 wanted", fn, what,
             (long long)ss, (long long)scale_bytes(K));
  return SF_OK;
}

int check_call(const char* fn, const void* b_enc, int benc_dt, const void* thr, int thr_dt, const void* out,
               int64_t som, int out_dt, int64_t M, int64_t N, int64_t K, int act) {
  SF_REQUIRE(sf_valid_dtype(out_dt) && (!b_enc || sf_valid_dtype(benc_dt)), "%s: bad dtype code", fn);
  SF_REQUIRE(act == SF_ACT_RELU || act == SF_ACT_JUMPRELU || act == SF_ACT_NONE, "%s: bad activation %d", fn, act);
  SF_REQUIRE(M >= 0 && N >= 0 && K >= 1, "%s: bad size (M=%lld N=%lld K=%lld)", fn, (long long)M, (long long)N,
             (long long)K);
  SF_REQUIRE(M <= INT32_MAX && N <= INT32_MAX && K <= (1 << 22), "%s: size too large (M=%lld N=%lld K=%lld)", fn,
             (long long)M, (long long)N, (long long)K);
  if (M == 0 || N == 0) return SF_OK;
  SF_REQUIRE(act != SF_ACT_JUMPRELU || (thr && sf_valid_dtype(thr_dt)), "%s: jumprelu needs a threshold", fn);
  SF_REQUIRE(out, "%s: out must not be NULL", fn);
  SF_REQUIRE(som >= N || M == 1, "%s: rows of the result overlap", fn);
  return SF_OK;
}

int product(const char* fn, const void* xq, int64_t sxq, const void* xs, int64_t sxs, const void* wq, int64_t swq,
            const void* ws, int64_t sws, const void* b_enc, int benc_dt, const void* thr, int thr_dt, void* out,
            int64_t som, int out_dt, int32_t* row_nnz, int64_t M, int64_t N, int64_t K, int act, void* ctr, hipStream_t s) {
  F8Args a = {};
  a.xw = (const char*)xq; a.Kp = sxq; a.xs = (const uint8_t*)xs; a.sxs = sxs;
  a.w = (const char*)wq; a.swn = swq; a.swk = 1; a.ws = (const uint8_t*)ws; a.sws = sws;
  a.b_enc = b_enc; a.benc_dt = benc_dt; a.thr = thr; a.thr_dt = thr_dt;
  a.out = out; a.som = som; a.son = 1; a.out_dt = out_dt;
  a.row_nnz = row_nnz; a.M = M; a.N = N; a.K = K; a.act = act;
  a.group_m = 1;
  a.group_n = 8;
  a.ksteps = (int)blocks_of(K);
  a.vec_store = som * sf_dtype_size(out_dt) % 16 == 0 && aligned(out, 16);
  const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256);
  SF_REQUIRE(((M + 31) / 32) * ((N + 63) / 64) < (1ll << 24) || M > 32, "%s: too many tiles", fn);
  SF_REQUIRE(tiles < (1ll << 22), "%s: too many tiles", fn);
  hipError_t e;
  if (M <= 32) e = launch_tile<F8x32, AUX_NT>(a, s);
  else if (tiles >= 256 && out_dt != SF_F32) e = launch_persist(a, ctr, s);
  else if (tiles < 512) e = launch_tile<F8x128, 0>(a, s);
  else e = launch_tile<F8x256, 0>(a, s);
  if (e != hipSuccess) return sf_fail(SF_EHIP, "%s: kernel launch failed: %s", fn, hipGetErrorString(e));
  return SF_OK;
}

}  // namespace
}  // namespace sff8

extern "C" int sf_encode_fp8_rows(const void* xq, int64_t sxq, const void* xs, int64_t sxs, const void* wq, int64_t swq,
                                  const void* ws, int64_t sws, const void* b_enc, int benc_dt, const void* thr,
                                  int thr_dt, void* out, int64_t som, int out_dt, int32_t* row_nnz, int64_t M, int64_t N,
                                  int64_t K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace sff8;
  static const char* fn = "sf_encode_fp8_rows";
  sf_clear_error();
  if (const int rc = check_call(fn, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, M, N, K, act)) return rc;
  if (M == 0 || N == 0) return SF_OK;
  SF_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= TILE_CTR_BYTES,
             "%s: needs a 16-B aligned workspace of %lld bytes", fn, (long long)TILE_CTR_BYTES);
  if (const int rc = check_rows(fn, "x", xq, sxq, xs, sxs, K)) return rc;
  if (const int rc = check_rows(fn, "w", wq, swq, ws, sws, K)) return rc;
  return product(fn, xq, sxq, xs, sxs, wq, swq, ws, sws, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M, N, K,
                 act, workspace, (hipStream_t)stream);
}

extern "C" int sf_encode_fp8_workspace_size(int64_t M, int64_t K, int64_t* bytes) {
  using namespace sff8;
  sf_clear_error();
  SF_REQUIRE(bytes, "sf_encode_fp8_workspace_size: bytes must not be NULL");
  SF_REQUIRE(M >= 0 && M <= INT32_MAX && K >= 1 && K <= (1 << 22), "sf_encode_fp8_workspace_size: bad size (M=%lld K=%lld)",
             (long long)M, (long long)K);
  *bytes = (M * (code_bytes(K) + scale_bytes(K)) + 63) / 64 * 64 + TILE_CTR_BYTES;
  return SF_OK;
}

extern "C" int sf_encode_fp8(const void* x, int64_t sxm, int64_t sxk, int x_dt, const void* b_dec, int bdec_dt,
                             const void* wq, int64_t swq, const void* ws, int64_t sws, const void* b_enc, int benc_dt,
                             const void* thr, int thr_dt, void* out, int64_t som, int out_dt, int32_t* row_nnz,
                             int64_t M, int64_t N, int64_t K, int act, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace sff8;
  static const char* fn = "sf_encode_fp8";
  sf_clear_error();
  SF_REQUIRE(sf_valid_dtype(x_dt) && (!b_dec || sf_valid_dtype(bdec_dt)), "%s: bad dtype code", fn);
  if (const int rc = check_call(fn, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, M, N, K, act)) return rc;
  if (M == 0 || N == 0) return SF_OK;
  SF_REQUIRE(x, "%s: x must not be NULL", fn);
  const int64_t sq = code_bytes(K), ss = scale_bytes(K);
  const int64_t ctr = (M * (sq + ss) + 63) / 64 * 64;
  SF_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= ctr + TILE_CTR_BYTES,
             "%s: needs a 16-B aligned workspace of %lld bytes", fn, (long long)(ctr + TILE_CTR_BYTES));
  if (const int rc = check_rows(fn, "w", wq, swq, ws, sws, K)) return rc;
  char* xs = (char*)workspace + M * sq;
  if (const int rc = launch_quantize(x, sxm, sxk, x_dt, b_dec, bdec_dt, M, K, workspace, sq, xs, ss, 0, M,
                                     (hipStream_t)stream))
    return rc;
  return product(fn, workspace, sq, xs, ss, wq, swq, ws, sws, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M,
                 N, K, act, (char*)workspace + ctr, (hipStream_t)stream);
}
