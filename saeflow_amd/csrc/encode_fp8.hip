// Entry points of the encoder product on 8-bit rows (kernels: encode_fp8.h).
#include <math.h>

#include "encode_fp8.h"

namespace sff8 {
namespace {

using namespace sfenc;

// The tiles, tokens x features, with the stages that leave room for two workgroups a CU: narrow ones for few
// tokens, where the pass over W bounds the product, wider ones where the matrix cores do. Eight waves each from
// 64 tokens on: 128x128 tiles with waves of 32x64 5.5% faster than four waves of 64x64 over 148 shapes
// (128 tokens and more, 16-bit results; -18 to +4%), 64x128 with waves of 32x32 2.3% faster than four of 64x32.
// fp32 results alike on average.
typedef SlimTile<1, 1, 1, 4, 8, 3> F8x32;    // 32 x 128
typedef SlimTile<1, 1, 2, 4, 8, 3> F8x64;    // 64 x 128
typedef SlimTile<1, 2, 4, 2, 8, 2> F8x128;   // 128 x 128
typedef SlimTile<2, 1, 2, 4, 8, 4> F8x128one;  // 128 x 128, a CU to itself
typedef SlimTile<1, 1, 1, 2, 8, 6> F8few;    // 32 x 64, tokens quantised in the kernel

template <typename TL, bool FUSED = false, bool F32 = true>  // F32: fp32 results are asked of it
hipError_t launch_tile(F8Args& a, hipStream_t s) {
  a.tiles_m = (int)((a.M + TL::TM - 1) / TL::TM);
  a.tiles_n = (int)((a.N + TL::TN - 1) / TL::TN);
  a.group_n = std::min(a.group_n, a.tiles_n);
  const dim3 grid(a.tiles_m * a.tiles_n), block(TL::NT);
  const bool plain = a.act != SF_ACT_JUMPRELU && !a.row_nnz;
  if (a.out_dt == SF_F32) {
    if constexpr (F32) {
      if (plain) hipLaunchKernelGGL((gemm_f8_kernel<TL, true, true, FUSED>), grid, block, 0, s, a);
      else hipLaunchKernelGGL((gemm_f8_kernel<TL, true, false, FUSED>), grid, block, 0, s, a);
    } else {
      return hipErrorInvalidValue;
    }
  } else {
    if (plain) hipLaunchKernelGGL((gemm_f8_kernel<TL, false, true, FUSED>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((gemm_f8_kernel<TL, false, false, FUSED>), grid, block, 0, s, a);
  }
  return hipGetLastError();
}

// 256x256 tiles: the persistent form, one workgroup per CU (at most one per
// tile, whole XCD groups of eight). ctr: TILE_CTR_BYTES of the caller's workspace, `cleared` already or not.
hipError_t launch_persist(F8Args& a, void* ctr, bool cleared, hipStream_t s) {
  a.tiles_m = (int)((a.M + BM - 1) / BM);
  a.tiles_n = (int)((a.N + BN - 1) / BN);
  a.group_n = std::min(a.group_n, a.tiles_n);
  const int cus = device_cus();
  if (cus <= 0) return hipErrorInvalidDevice;
  const int total = a.tiles_m * a.tiles_n;
  const dim3 grid((unsigned)std::max(8, std::min(cus / 8 * 8, (total + 7) / 8 * 8))), block(256);
  // (with a workgroup for every tile nothing is claimed)
  a.tile_ctr = total > (int)grid.x ? (int32_t*)ctr : nullptr;
  if (a.tile_ctr && !cleared) hipLaunchKernelGGL(clear_counters_kernel, dim3(1), dim3(64), 0, s, a.tile_ctr);
  const bool plain = a.act != SF_ACT_JUMPRELU && !a.row_nnz;
  if (a.out_dt == SF_F32) {
    if (plain) hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_F32, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((gemm_f8_persist_kernel<SF_F32, false>), grid, block, 0, s, a);
  } else if (a.out_dt == SF_F16) {
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
               int64_t som, int out_dt, const int32_t* row_nnz, int64_t M, int64_t N, int64_t K, int act) {
  SF_REQUIRE(sf_valid_dtype(out_dt) && (!b_enc || sf_valid_dtype(benc_dt)), "%s: bad dtype code", fn);
  SF_REQUIRE(act == SF_ACT_RELU || act == SF_ACT_JUMPRELU || act == SF_ACT_NONE, "%s: bad activation %d", fn, act);
  SF_REQUIRE(act != SF_ACT_NONE || !row_nnz, "%s: row counts need relu or jumprelu", fn);
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

// Tokens are quantised by each workgroup of the product for itself where their blocks are one round of
// loads for it and there are at most two workgroups a CU: one token of d_in 2304 over 16384 features 10.6 us a
// call against 13.1 with a quantisation of its own, over 65536 (four a CU) 27.5 against 26.5.
constexpr int64_t FUSED_FEATURES = 32768;
struct Tokens {
  const void* x;
  int64_t sxm, sxk;
  int x_dt;
  const void* shift;
  int shift_dt;
};

// Estimated time of a product in us with tiles of tm x tn: a fixed part, and for each round of tiles over
// the CUs a part per block of K (`alone` times that with one workgroup a CU) and one per tile; at least
// the bytes at the rate that the shape streams them. Fitted to 220 shapes of 1 to 4096 tokens, d_in 256 to
// 4096, 4096 to 131072 features, in both result sizes, before results went through L2 where lines are shared. Over 715
// other shapes with the stores as they are (1 to 8192 tokens, d_in 120 to 4096, two of three with rows off 16 B) the pick is
// 1.6% (fp32 0.6%) slower than the best in the mean, 30% at most (2175 tokens of d_in 256 over 58624 features: 256x256
// 85 us, 128x128 67). Where each of the first four wins at d_in 2304, d_sae 65536, bf16 (us in
// order): 32 tokens 24 25 25 32 (d_sae 16384: 11 11 16 26), 128 tokens 42 30 26 33, 256 tokens 79 53 42 37, 4096
// tokens 1133 803 626 494; fp32 results of 128 tokens 59 46 40 60, of 256 109 87 73 66, of 4096 1714 1394 1104
// 962.
struct Shape {
  int tm, tn;
  float fixed, step, alone, tile, tail, tbs;
};
constexpr Shape SHAPES[2][5] = {
    // 16-bit results
    {{32, 128, 2.27f, 0.215f, 1.61f, 0.94f, 0.40f, 6.66f}, {64, 128, 1.81f, 0.300f, 1.38f, 1.29f, 0.38f, 6.90f},
     {128, 128, 1.16f, 0.472f, 1.47f, 1.77f, 0.30f, 5.50f}, {256, 256, 4.42f, 1.655f, 0.61f, 3.43f, 0.24f, 6.65f},
     {128, 128, 1.20f, 0.487f, 0.84f, 2.78f, 0.14f, 6.72f}},
    // fp32 results
    {{32, 128, 2.30f, 0.319f, 1.37f, 1.22f, 0.27f, 6.91f}, {64, 128, 2.02f, 0.534f, 1.06f, 1.70f, 0.14f, 6.53f},
     {128, 128, 1.87f, 0.840f, 0.96f, 2.40f, 0.39f, 5.01f}, {256, 256, 0.f, 2.815f, 0.69f, 11.99f, 0.20f, 3.90f}, {}}};
// The fifth, 128 x 128 with eight waves and four stages, has a CU to itself: for one round of 16-bit
// results only (d_in 4096, d_sae 12288, 256 tokens 18 us against 21 with 64 x 128; from two rounds on two
// workgroups a CU win).
constexpr int ONE_ROUND = 4;
// What result rows off 16 B cost a 256x256 tile (bf16: 4096 tokens of d_in 768 over 16391 features 92 us, 128x128 tiles
// 73). Over 326 such shapes the pick is 1.3% slower than the best with 4 us, 2.0% with 3, 1.9% with 5, 4.2% with none (169
// of fp32: 0.6, 0.5, 0.6, 1.7%).
constexpr float UNALIGNED_TILE = 4.f;

// Whether 256x256 tiles store 16-bit result rows off whole lines past the caches too. Time past the caches over time
// through L2 (geometric means over 290 such shapes, d_in 64 to 4096, bf16):
//   MB of results     250-448  448-530  530-600  600-750  750-1300
//   d_in up to 128      1.42     1.39     1.40     1.35     1.24    (one K-step a tile)
//   d_in 192 to 768     1.08     1.07     1.01     0.95     0.90
//   d_in 1024 to 4096   1.02     0.99     0.93     0.91     0.85
// The rule costs 1.2% over the better of both in the mean.
bool stream_shared(int64_t M, int64_t N, int64_t K) {
  const double bytes = (double)M * N * 2;
  return K > BLOCK && bytes > (K < 1024 ? 600e6 : 448e6);
}

int pick_shape(int64_t M, int64_t N, int64_t K, int out_dt, bool unaligned) {
  const int nb = (int)blocks_of(K), wide = out_dt == SF_F32;
  const double bytes = (double)N * K + (double)M * K + (double)M * N * sf_dtype_size(out_dt);
  int best = -1;
  double least = 0;
  for (int i = 0; i < (wide ? 4 : 5); ++i) {
    const Shape& h = SHAPES[wide][i];
    const double x = (double)((M + h.tm - 1) / h.tm) * (double)((N + h.tn - 1) / h.tn) / 256;
    if (i == ONE_ROUND && x > 1) continue;
    const double rounds = x <= 1 ? 1 : (x < 3 ? ceil(x) : x + h.tail);
    const double tile = h.tile + (i == 3 && unaligned ? UNALIGNED_TILE : 0.f);
    const double t = std::max(h.fixed + (nb * h.step * (x <= 1 ? h.alone : 1) + tile) * rounds,
                              h.fixed + tile + bytes / h.tbs * 1e-6);
    if (best < 0 || t < least) {
      best = i;
      least = t;
    }
  }
  return best;
}

int product(const char* fn, const Tokens* tokens, const void* xq, int64_t sxq, const void* xs, int64_t sxs,
            const void* wq, int64_t swq, const void* ws, int64_t sws, const void* b_enc, int benc_dt, const void* thr,
            int thr_dt, void* out, int64_t som, int out_dt, int32_t* row_nnz, int64_t M, int64_t N, int64_t K, int act,
            void* ctr, bool cleared, hipStream_t s) {
  F8Args a = {};
  a.xw = (const char*)xq; a.Kp = sxq; a.xs = (const uint8_t*)xs; a.sxs = sxs;
  a.w = (const char*)wq; a.swn = swq; a.swk = 1; a.ws = (const uint8_t*)ws; a.sws = sws;
  a.b_enc = b_enc; a.benc_dt = benc_dt; a.thr = thr; a.thr_dt = thr_dt;
  a.out = out; a.som = som; a.son = 1; a.out_dt = out_dt;
  a.row_nnz = row_nnz; a.M = M; a.N = N; a.K = K; a.act = act;
  a.group_m = 1;
  a.group_n = 8;
  a.ksteps = (int)blocks_of(K);
  a.stream = aligned(out, 128) && som * sf_dtype_size(out_dt) % 128 == 0;
  hipError_t e;
  if (tokens) {
    a.x = tokens->x; a.sxm = tokens->sxm; a.sxk = tokens->sxk; a.x_dt = tokens->x_dt;
    a.x_rows = a.sxk == 1 && aligned(a.x, 16) && a.sxm * sf_dtype_size(a.x_dt) % 16 == 0;
    a.shift = tokens->shift; a.shift_dt = tokens->shift_dt;
    a.shift_vec = a.shift && a.shift_dt == a.x_dt && aligned(a.shift, 16);
    e = launch_tile<F8few, true>(a, s);
  } else {
    const int shape = pick_shape(M, N, K, out_dt, som * sf_dtype_size(out_dt) % 16 != 0 || !aligned(out, 16));
    const Shape& h = SHAPES[out_dt == SF_F32][shape];
    if (shape == 3 && out_dt != SF_F32 && stream_shared(M, N, K)) a.stream = 1;
    SF_REQUIRE(((M + h.tm - 1) / h.tm) * ((N + h.tn - 1) / h.tn) < (1ll << 23), "%s: too many tiles", fn);
    switch (shape) {
      case 0: e = launch_tile<F8x32>(a, s); break;
      case 1: e = launch_tile<F8x64>(a, s); break;
      case 2: e = launch_tile<F8x128>(a, s); break;
      case ONE_ROUND: e = launch_tile<F8x128one, false, false>(a, s); break;
      default: e = launch_persist(a, ctr, cleared, s); break;
    }
  }
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
  if (const int rc = check_call(fn, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M, N, K, act)) return rc;
  if (M == 0 || N == 0) return SF_OK;
  SF_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= TILE_CTR_BYTES,
             "%s: needs a 16-B aligned workspace of %lld bytes", fn, (long long)TILE_CTR_BYTES);
  if (const int rc = check_rows(fn, "x", xq, sxq, xs, sxs, K)) return rc;
  if (const int rc = check_rows(fn, "w", wq, swq, ws, sws, K)) return rc;
  return product(fn, nullptr, xq, sxq, xs, sxs, wq, swq, ws, sws, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M, N, K,
                 act, workspace, false, (hipStream_t)stream);
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
  if (const int rc = check_call(fn, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M, N, K, act)) return rc;
  if (M == 0 || N == 0) return SF_OK;
  SF_REQUIRE(x, "%s: x must not be NULL", fn);
  const int64_t sq = code_bytes(K), ss = scale_bytes(K);
  const int64_t ctr = (M * (sq + ss) + 63) / 64 * 64;
  SF_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= ctr + TILE_CTR_BYTES,
             "%s: needs a 16-B aligned workspace of %lld bytes", fn, (long long)(ctr + TILE_CTR_BYTES));
  if (const int rc = check_rows(fn, "w", wq, swq, ws, sws, K)) return rc;
  if (M * blocks_of(K) <= FUSED_BLOCKS && N <= FUSED_FEATURES) {
    const Tokens tokens = {x, sxm, sxk, x_dt, b_dec, bdec_dt};
    return product(fn, &tokens, nullptr, 0, nullptr, 0, wq, swq, ws, sws, b_enc, benc_dt, thr, thr_dt, out, som, out_dt,
                   row_nnz, M, N, K, act, nullptr, false, (hipStream_t)stream);
  }
  char* xs = (char*)workspace + M * sq;
  int32_t* counters = (int32_t*)((char*)workspace + ctr);
  if (const int rc = launch_quantize(x, sxm, sxk, x_dt, b_dec, bdec_dt, M, K, workspace, sq, xs, ss, 0, M,
                                     counters, (hipStream_t)stream))
    return rc;
  return product(fn, nullptr, workspace, sq, xs, ss, wq, swq, ws, sws, b_enc, benc_dt, thr, thr_dt, out, som, out_dt, row_nnz, M,
                 N, K, act, counters, true, (hipStream_t)stream);
}
