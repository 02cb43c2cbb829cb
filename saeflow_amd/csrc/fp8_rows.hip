// 8-bit rows written and read back (format: fp8.h). Both are one pass over the data, bound by HBM.
#include <algorithm>
#include <type_traits>

#include "fp8.h"

namespace sff8 {

// Sixteen lanes take one block of 128, eight elements each: the maximum is four rotations within a
// DPP row, each lane's eight codes are one 8-B store and the sixteen of a block one cache line.
// Blocks are numbered row by row over [0, total), total < 2^31, so the row is a 32-bit division. Bound by
// memory: 16384 rows of 2304 take 28 us in bf16 and 34 us in fp32 where x was just written (4.0 and 5.6 TB/s),
// 42 and 64 us out of HBM with dirty lines to evict; loads past the caches 30 and 36, 35 and 47; two blocks a
// lane under way change nothing. Rows off 16 B are read element by element (SRC_ANY): 16384 rows of 2303 take 49 us in bf16
// and 67 in fp32 where rows of 2304 take 21 and 27, every second element of rows of 4608 78 us.
template <int DT, int SRC>
__global__ __launch_bounds__(256) void quantize_kernel(const void* x, int64_t sxm, int64_t sxk, const void* shift,
                                                       int shift_dt, int shift_vec, int64_t K, uint32_t nb,
                                                       uint32_t total, uint8_t* q, int64_t sq, uint8_t* scale,
                                                       int64_t ss, int64_t row0, int64_t R, int pad, int32_t* ctr) {
  if (ctr && blockIdx.x == 0 && threadIdx.x < 8) ctr[threadIdx.x * 16] = 0;
  const uint32_t lane16 = threadIdx.x & 15;
  for (uint32_t b = blockIdx.x * 16 + (threadIdx.x >> 4); b < total; b += gridDim.x * 16) {
    const uint32_t m = b / nb, kb = b - m * nb;
    const int64_t k0 = (int64_t)kb * BLOCK + lane16 * 8;
    float v[8];
    load_shifted<DT, SRC>(x, sxm, sxk, shift, shift_dt, shift_vec, K, m, k0, v);
    uint32_t byte;
    const u32x2 codes = quantize8(v, byte);
    int64_t r = row0 + m;
    if (r >= R) r -= R;
    *(u32x2*)(q + r * sq + k0) = codes;
    if (lane16 == 0) scale[r * ss + kb] = (uint8_t)byte;
    if (lane16 > 0 && lane16 <= (uint32_t)pad && kb + 1 == nb) scale[r * ss + kb + lane16] = 0;
  }
}

// Columns contiguous (x[m, k] at m + k * sxk, a dictionary's W_enc^T): a workgroup takes CROWS rows x one
// block of 128, read as 128 pieces of CROWS elements (512 B) into LDS, and every four lanes write one
// row's 128 codes, a whole cache line. LDS piece k lies at k * CROWS E + (k / 32) * 16 E: the four lanes of
// a row read pieces 32 apart, 16 rows at once, which fills the 64 banks exactly. Bound by HBM, and by how
// much of a row of x one workgroup takes: 65536 columns of 2304 bf16 elements 97 us out of HBM (4.7 TB/s)
// with 512-B pieces, 101 with 256 B, 103 with 128 B.
template <int DT>
constexpr int CROWS = DT == SF_F32 ? 128 : 256;
template <int DT>
__global__ __launch_bounds__(4 * CROWS<DT>) void quantize_columns_kernel(const void* x, int64_t sxk, int vec, const void* shift,
                                                               int shift_dt, int64_t M, int64_t K, int64_t nb,
                                                               uint8_t* q, int64_t sq, uint8_t* scale, int64_t ss,
                                                               int64_t row0, int64_t R, int pad, int32_t* ctr) {
  if (ctr && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 8) ctr[threadIdx.x * 16] = 0;
  constexpr int CROWS = sff8::CROWS<DT>, E = DT == SF_F32 ? 4 : 2, EPC = 16 / E, CPR = CROWS / EPC, NT = 4 * CROWS, PER = 128 * CPR / NT;
  __shared__ __attribute__((aligned(16))) char st[128 * CROWS * E + 4 * 16 * E];
  const int t = threadIdx.x;
  const int64_t m0 = (int64_t)blockIdx.x * CROWS, kb = blockIdx.y, k0 = kb * BLOCK;
  if (vec && m0 + CROWS <= M) {
    u32x4 v[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = (i * NT + t) / CPR, c = t % CPR;
      v[i] = u32x4{0, 0, 0, 0};
      if (k0 + k < K) v[i] = __builtin_nontemporal_load((const u32x4*)((const char*)x + ((k0 + k) * sxk + m0) * E + c * 16));
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = (i * NT + t) / CPR, c = t % CPR;
      *(u32x4*)(st + k * CROWS * E + (k >> 5) * 16 * E + c * 16) = v[i];
    }
  } else {
    for (int i = t; i < 128 * CROWS; i += NT) {
      const int k = i / CROWS, m = i % CROWS;
      const uint32_t bits = k0 + k < K && m0 + m < M ? load_bits(x, DT, (k0 + k) * sxk + m0 + m) : 0u;
      char* dst = st + k * CROWS * E + (k >> 5) * 16 * E + m * E;
      if constexpr (E == 4) *(uint32_t*)dst = bits;
      else *(u16*)dst = (u16)bits;
    }
  }
  __syncthreads();
  const int m = t >> 2, kq = t & 3;
  float v[32];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int k = kq * 32 + i;
    v[i] = load_as_f32(st + k * CROWS * E + kq * 16 * E, DT, m);
    if (shift && k0 + k < K) v[i] -= load_as_f32(shift, shift_dt, k0 + k);
    top = max(top, finite_bits(v[i]));
  }
  const uint32_t byte = scale_byte(max4(top));
  const float inv = inverse_of(byte);
  if (m0 + m >= M) return;
  int64_t r = row0 + m0 + m;
  if (r >= R) r -= R;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    w[i] = pack4(scaled(v[4 * i], inv), scaled(v[4 * i + 1], inv), scaled(v[4 * i + 2], inv), scaled(v[4 * i + 3], inv));
  char* dst = (char*)q + r * sq + k0 + kq * 32;
  *(u32x4*)dst = u32x4{w[0], w[1], w[2], w[3]};
  *(u32x4*)(dst + 16) = u32x4{w[4], w[5], w[6], w[7]};
  if (kq == 0) scale[r * ss + kb] = (uint8_t)byte;
  if (kq > 0 && kq <= pad && kb + 1 == nb) scale[r * ss + kb + kq] = 0;
}

// Eight codes a lane, sixteen lanes a block, U blocks a lane under way, as quantize_kernel. Row m of the
// result is row (row0 + m) % R of the store, or rows[m]; an id outside [0, R) gives zeros. Bound by memory:
// 16384 rows of 2304 to bf16 take 20 us with two blocks a lane under way (5.7 TB/s), 22 with one; to fp32
// (whose lanes write twice as much) 50 with one, 57 with two. Stores go past the caches: 65536 rows 92 us
// against 96, 177 against 183 with a pass over the result behind it (16384: 46 against 44). Result rows off 16 B
// are stored element by element: 16384 rows of 2303 take 49 us in bf16 and 91 in fp32, of 2304 18 and 52.
template <int ODT, int U>
__global__ __launch_bounds__(256) void dequantize_kernel(const uint8_t* q, int64_t sq, const uint8_t* scale, int64_t ss,
                                                         int64_t R, const int64_t* rows, int64_t row0,
                                                         const void* shift, int shift_dt, int shift_vec, int64_t K,
                                                         uint32_t nb, uint32_t total, void* out, int64_t som, int vec) {
  const uint32_t lane16 = threadIdx.x & 15, stride = gridDim.x * 16;
  for (uint32_t b0 = blockIdx.x * 16 + (threadIdx.x >> 4); b0 < total; b0 += U * stride) {
    u32x2 c[U];
    uint32_t byte[U], m[U], kb[U];
    bool in[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t b = min(b0 + u * stride, total - 1);
      m[u] = b / nb;
      kb[u] = b - m[u] * nb;
      int64_t r;
      if (rows) {
        r = rows[m[u]];
      } else {
        r = row0 + m[u];
        if (r >= R) r -= R;
      }
      in[u] = r >= 0 && r < R;
      if (!in[u]) r = 0;
      c[u] = *(const u32x2*)(q + r * sq + (int64_t)kb[u] * BLOCK + lane16 * 8);  // (rows are padded to whole blocks)
      byte[u] = scale[r * ss + kb[u]];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t k0 = (int64_t)kb[u] * BLOCK + lane16 * 8;
      if (k0 >= K || (U > 1 && b0 + u * stride >= total)) continue;
      float v[8];
      const float f = scale_of(byte[u]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[u][i], false);
        const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[u][i], true);
        v[4 * i] = lo[0] * f;
        v[4 * i + 1] = lo[1] * f;
        v[4 * i + 2] = hi[0] * f;
        v[4 * i + 3] = hi[1] * f;
      }
      if (shift_vec && k0 + 8 <= K) {
        float s[8];
        load8<ODT>(shift, k0, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += s[e];
      } else if (shift) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + e < K) v[e] += load_as_f32(shift, shift_dt, k0 + e);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = in[u] ? v[e] : 0.f;
      if (vec && k0 + 8 <= K) {
        if constexpr (ODT == SF_F32) {
          u32x4* dst = (u32x4*)((float*)out + m[u] * som + k0);
#pragma unroll
          for (int i = 0; i < 2; ++i)
            __builtin_nontemporal_store(u32x4{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                              __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])}, dst + i);
        } else {
          u32x4 o;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = f32_to_bits(v[2 * e], ODT) | f32_to_bits(v[2 * e + 1], ODT) << 16;
          __builtin_nontemporal_store(o, (u32x4*)((u16*)out + m[u] * som + k0));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k0 + e < K) {
            if constexpr (ODT == SF_F32) ((float*)out)[m[u] * som + k0 + e] = v[e];
            else ((u16*)out)[m[u] * som + k0 + e] = (u16)f32_to_bits(v[e], ODT);
          }
      }
    }
  }
}

namespace {

constexpr int64_t MOST_BLOCKS = 1ll << 30;  // of one launch (32-bit block numbers)

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Blocks under way in a lane: one where there are few, so that they spread over the chip.
constexpr int64_t UNROLL_FROM = 65536;
// Workgroups of 16 blocks (times those under way): enough to fill the chip several times over, then a
// grid stride.
unsigned grid_of(int64_t total, int unroll) {
  return (unsigned)std::min<int64_t>((total + 16 * unroll - 1) / (16 * unroll), 1 << 16);
}

int check_store(const void* q, int64_t sq, const void* scale, int64_t ss, int64_t R, int64_t K) {
  SF_REQUIRE(q && scale, "codes and scales must not be NULL");
  SF_REQUIRE(aligned16(q) && sq % 16 == 0, "rows of codes must be 16-B aligned");
  SF_REQUIRE(((uintptr_t)scale & 3) == 0 && ss % 4 == 0, "rows of scales must be 4-B aligned");
  SF_REQUIRE(sq >= code_bytes(K), "rows of codes hold %lld bytes, %lld are needed for %lld elements", (long long)sq,
             (long long)code_bytes(K), (long long)K);
  SF_REQUIRE(ss >= scale_bytes(K), "rows of scales hold %lld bytes, %lld are needed for %lld elements", (long long)ss,
             (long long)scale_bytes(K), (long long)K);
  SF_REQUIRE(R >= 0, "negative number of rows");
  return SF_OK;
}

template <int DT>
int quantize_typed(const void* x, int64_t sxm, int64_t sxk, const void* shift, int shift_dt, int64_t M, int64_t K,
                   void* q, int64_t sq, void* scale, int64_t ss, int64_t row0, int64_t R, int32_t* ctr, hipStream_t s) {
  constexpr int E = DT == SF_F32 ? 4 : 2, CR = CROWS<DT>;
  const int64_t nb = blocks_of(K);
  const int pad = (int)(scale_bytes(K) - nb);
  if (sxm == 1 && sxk != 1 && M >= 16 && nb < 65536) {
    // 65536 * CR rows a launch at most
    const int vec = aligned16(x) && sxk * E % 16 == 0;
    for (int64_t m = 0; m < M; m += (int64_t)CR << 16) {
      const int64_t n = std::min<int64_t>(M - m, (int64_t)CR << 16);
      const int64_t at = (row0 + m) % R;
      hipLaunchKernelGGL((quantize_columns_kernel<DT>), dim3((unsigned)((n + CR - 1) / CR), (unsigned)nb), dim3(4 * CR), 0, s,
                         (const char*)x + m * E, sxk, vec, shift, shift_dt, n, K, nb, (uint8_t*)q, sq, (uint8_t*)scale,
                         ss, at, R, pad, ctr);
      SF_LAUNCH_CHECK("quantize_columns");
    }
    return SF_OK;
  }
  const bool rows = sxk == 1 && aligned16(x) && sxm * E % 16 == 0;
  const int svec = shift && shift_dt == DT && aligned16(shift);
  const int64_t step = std::max<int64_t>(1, MOST_BLOCKS / nb);
  for (int64_t m = 0; m < M; m += step) {
    const int64_t n = std::min(M - m, step);
    const int64_t at = (row0 + m) % R;
    const char* xm = (const char*)x + m * sxm * E;
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(grid_of(n * nb, 1)), dim3(256), 0, s, xm, sxm, sxk, shift, shift_dt, svec, K,
                         (uint32_t)nb, (uint32_t)(n * nb), (uint8_t*)q, sq, (uint8_t*)scale, ss, at, R, pad, ctr);
    };
    if (rows) go(quantize_kernel<DT, SRC_ROWS>);
    else go(quantize_kernel<DT, SRC_ANY>);
    SF_LAUNCH_CHECK("quantize");
  }
  return SF_OK;
}

}  // namespace

int launch_quantize(const void* x, int64_t sxm, int64_t sxk, int x_dt, const void* shift, int shift_dt, int64_t M,
                    int64_t K, void* q, int64_t sq, void* scale, int64_t ss, int64_t row0, int64_t R, int32_t* ctr,
                    hipStream_t s) {
  switch (x_dt) {
    case SF_F32: return quantize_typed<SF_F32>(x, sxm, sxk, shift, shift_dt, M, K, q, sq, scale, ss, row0, R, ctr, s);
    case SF_BF16: return quantize_typed<SF_BF16>(x, sxm, sxk, shift, shift_dt, M, K, q, sq, scale, ss, row0, R, ctr, s);
    default: return quantize_typed<SF_F16>(x, sxm, sxk, shift, shift_dt, M, K, q, sq, scale, ss, row0, R, ctr, s);
  }
}

}  // namespace sff8

extern "C" int sf_quantize_rows(const void* x, int64_t sxm, int64_t sxk, int x_dt, const void* shift, int shift_dt,
                                int64_t M, int64_t K, void* q, int64_t sq, void* scale, int64_t ss, int64_t row0,
                                int64_t R, void* stream) {
  using namespace sff8;
  sf_clear_error();
  SF_REQUIRE(sf_valid_dtype(x_dt) && (!shift || sf_valid_dtype(shift_dt)), "unsupported dtype code");
  SF_REQUIRE(M >= 0 && K >= 1 && K <= (1 << 24), "bad shape [%lld, %lld]", (long long)M, (long long)K);
  if (M == 0) return SF_OK;
  SF_REQUIRE(x, "x must not be NULL");
  if (const int rc = check_store(q, sq, scale, ss, R, K)) return rc;
  SF_REQUIRE(M <= R, "%lld rows do not fit %lld", (long long)M, (long long)R);
  SF_REQUIRE(row0 >= 0 && row0 < R, "first row %lld outside [0, %lld)", (long long)row0, (long long)R);
  return launch_quantize(x, sxm, sxk, x_dt, shift, shift_dt, M, K, q, sq, scale, ss, row0, R, nullptr, (hipStream_t)stream);
}

extern "C" int sf_dequantize_rows(const void* q, int64_t sq, const void* scale, int64_t ss, int64_t R,
                                  const int64_t* rows, int64_t row0, const void* shift, int shift_dt, int64_t M,
                                  int64_t K, void* out, int64_t som, int out_dt, void* stream) {
  using namespace sff8;
  sf_clear_error();
  SF_REQUIRE(sf_valid_dtype(out_dt) && (!shift || sf_valid_dtype(shift_dt)), "unsupported dtype code");
  SF_REQUIRE(M >= 0 && K >= 1 && K <= (1 << 24), "bad shape [%lld, %lld]", (long long)M, (long long)K);
  if (M == 0) return SF_OK;
  if (const int rc = check_store(q, sq, scale, ss, R, K)) return rc;
  SF_REQUIRE(R >= 1, "a store of no rows has none to read");
  SF_REQUIRE(out, "out must not be NULL");
  SF_REQUIRE(som >= K || M == 1, "rows of the result overlap");
  if (!rows) {
    SF_REQUIRE(M <= R, "%lld rows asked for of %lld", (long long)M, (long long)R);
    SF_REQUIRE(row0 >= 0 && row0 < R, "first row %lld outside [0, %lld)", (long long)row0, (long long)R);
  }
  const int64_t nb = blocks_of(K), step = std::max<int64_t>(1, MOST_BLOCKS / nb);
  const int E = sf_dtype_size(out_dt);
  const int vec = aligned16(out) && som * E % 16 == 0;
  const int svec = shift && shift_dt == out_dt && aligned16(shift);
  for (int64_t m = 0; m < M; m += step) {
    const int64_t n = std::min(M - m, step);
    const int64_t at = rows ? 0 : (row0 + m) % R;
    const int64_t* ids = rows ? rows + m : nullptr;
    void* o = (char*)out + m * som * E;
    auto go = [&](auto kernel, int unroll) {
      hipLaunchKernelGGL(kernel, dim3(grid_of(n * nb, unroll)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)q, sq,
                         (const uint8_t*)scale, ss, R, ids, at, shift, shift_dt, svec, K, (uint32_t)nb, (uint32_t)(n * nb),
                         o, som, vec);
    };
    auto typed = [&](auto dt_tag) {
      constexpr int DT = decltype(dt_tag)::value;
      if (DT == SF_F32 || n * nb < UNROLL_FROM) go(dequantize_kernel<DT, 1>, 1);
      else go(dequantize_kernel<DT, 2>, 2);
    };
    if (out_dt == SF_F32) typed(std::integral_constant<int, SF_F32>{});
    else if (out_dt == SF_BF16) typed(std::integral_constant<int, SF_BF16>{});
    else typed(std::integral_constant<int, SF_F16>{});
    SF_LAUNCH_CHECK("dequantize");
  }
  return SF_OK;
}
