// Layer norm on gfx950: the forward pass (optionally leaving x - mean in 8 bits for the backward pass), the
// backward pass with the reductions of weight's and bias's gradients, and the norm undone.
//
// Row x of D elements: mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), xh = (x - mean) rstd,
// y = xh w + b. Given g = dL/dy, with q = g w:
//   dx = rstd (q - c1 - xh c2),  c1 = sum q / D,  c2 = sum q xh / D;  dw = sum_m g xh,  db = sum_m g.
// Gradients gm and gr of mean and rstd themselves add gm / D - gr rstd^2 xh / D to dx.
//
// All of it is bound by HBM: a row is read once and held in registers between the sums and the result. Measured for
// 16384 rows of 2304 in bf16 (75.5 MB; a large copy reads and writes 4.9 TB/s on this card), calls one after the other, the
// data partly in the last-level cache: forward 26.2 us (5.8 TB/s), with 8-bit rows 32.9 (5.7; 38 where x was not just read),
// backward with its parameters' sums 43 (5.2), from 8-bit rows 40 (4.7), undone 24.4 (6.2), its backward pass 35 (6.4; 38
// behind other kernels). In fp32 62, 71, 92, 71, 65 and 90 us (4.6 to 5.3 TB/s). Rows of 2303 begin anywhere and take 3 to
// 18% longer.
#include <algorithm>
#include <type_traits>

#include "fp8.h"
#include "wave.h"

namespace {

using sff8::u32x2;
using sff8::u32x4;
// 16 B at any element's address: rows of odd widths begin anywhere, and the hardware takes it
typedef u32x4 u32x4_any __attribute__((aligned(2)));

constexpr int X_FP8 = 3;  // the source of a backward pass: 8-bit rows of x - mean (beside SF_F32, SF_BF16, SF_F16)

// ------------------------------------------------------------------ eight consecutive elements of a row
// Raw registers of elements k0 .. k0 + 7 of 2-byte (N = 4) or 4-byte (N = 8) type; zeros past D.
template <int ES>
struct Raw {
  uint32_t r[2 * ES];
};
template <int ES>
__device__ __forceinline__ Raw<ES> load_raw(const char* row, int64_t k0, int64_t D) {
  Raw<ES> v;
  if (k0 + 8 <= D) {
#pragma unroll
    for (int i = 0; i < ES / 2; ++i) {
      const u32x4 c = *(const u32x4_any*)(row + k0 * ES + i * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) v.r[4 * i + j] = c[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2 * ES; ++i) v.r[i] = 0;
    if (k0 >= D) return v;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < D) {
        if constexpr (ES == 4) v.r[e] = ((const uint32_t*)row)[k0 + e];
        else v.r[e >> 1] |= (uint32_t)((const u16*)row)[k0 + e] << ((e & 1) * 16);
      }
  }
  return v;
}
// The same in two steps, for rows of at least eight elements, so that loads stay in flight without a branch: a
// lane whose chunk runs past D loads the row's last eight elements, and shifts by `off` = k0 - (D - 8) elements
// (zeros come in; eight or more: all zeros) once they are there.
template <int ES>
__device__ __forceinline__ Raw<ES> load_at(const char* row, uint32_t at) {  // (a uniform row, a lane's own offset)
  Raw<ES> v;
#pragma unroll
  for (int i = 0; i < ES / 2; ++i) {
    const u32x4 c = *(const u32x4_any*)(row + at + i * 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) v.r[4 * i + j] = c[j];
  }
  return v;
}
template <int ES>
__device__ __forceinline__ Raw<ES> load_back(const char* row, int64_t k0, int64_t D) {
  return load_at<ES>(row, (uint32_t)min(k0, D - 8) * ES);
}
template <int ES>
__device__ __forceinline__ void shift_back(Raw<ES>& v, int off) {
  constexpr int N = 2 * ES;
  if constexpr (ES == 2) {  // an odd element first
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t next = i + 1 < N ? v.r[i + 1] : 0;
      v.r[i] = off & 1 ? (v.r[i] >> 16) | (next << 16) : v.r[i];
    }
  }
#pragma unroll
  for (int by = 1; by < N; by <<= 1) {  // then whole registers
    const bool go = off & (ES == 2 ? 2 * by : by);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t from = i + by < N ? v.r[i + by] : 0;
      v.r[i] = go ? from : v.r[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v.r[i] = off >= 8 ? 0 : v.r[i];
}
template <int ES>
__device__ __forceinline__ float raw_elem(const Raw<ES>& v, int e, bool bf16) {
  if constexpr (ES == 4) {
    return __uint_as_float(v.r[e]);
  } else {
    const uint32_t h = (v.r[e >> 1] >> ((e & 1) * 16)) & 0xffffu;
    return bf16 ? bf16_to_f32(h) : f16_to_f32(h);
  }
}
// the same of a buffer whose type is known at run time (a parameter vector)
__device__ __forceinline__ void load8_any(const void* p, int dt, int64_t k0, int64_t D, float (&v)[8]) {
  if (dt == SF_F32) {
    const Raw<4> r = load_raw<4>((const char*)p, k0, D);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = raw_elem(r, e, false);
  } else {
    const Raw<2> r = load_raw<2>((const char*)p, k0, D);
    if (dt == SF_BF16) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = raw_elem(r, e, true);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = raw_elem(r, e, false);
    }
  }
}
// eight results, rounded once to dt; elements past D are not written
__device__ __forceinline__ void store8_any(char* row, int dt, int64_t k0, int64_t D, const float (&v)[8]) {
  if (k0 + 8 <= D) {
    if (dt == SF_F32) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *(u32x4_any*)(row + k0 * 4 + i * 16) = u32x4{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                                     __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])};
    } else {
      u32x4 o;
      if (dt == SF_BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = f32_to_bf16(v[2 * i]) | f32_to_bf16(v[2 * i + 1]) << 16;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = f32_to_f16(v[2 * i]) | f32_to_f16(v[2 * i + 1]) << 16;
      }
      *(u32x4_any*)(row + k0 * 2) = o;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < D) {
        if (dt == SF_F32) ((float*)row)[k0 + e] = v[e];
        else ((u16*)row)[k0 + e] = (u16)f32_to_bits(v[e], dt);
      }
  }
}

// the same through a buffer resource over a row, which drops what lies past its bounds (the row may begin anywhere)
template <int DT>
__device__ __forceinline__ void put8_rsrc(__amdgpu_buffer_rsrc_t rs, int k0, const float (&v)[8]) {
  if constexpr (DT == SF_F32) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                                   __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])},
                                             rs, k0 * 4 + 16 * i, 0, 0);
  } else {
    u32x4 q;
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = f32_to_bits(v[2 * i], DT) | f32_to_bits(v[2 * i + 1], DT) << 16;
    __builtin_amdgcn_raw_buffer_store_b128(q, rs, k0 * 2, 0, 0);
  }
}

// Sum of v over the wave in 64 bits, in every lane (wave_sum's moves on both halves).
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_add_f64(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROW_MASK, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROW_MASK, 0xF, false);
  return v + __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v = dpp_add_f64<0xB1, 0xF>(v);
  v = dpp_add_f64<0x4E, 0xF>(v);
  v = dpp_add_f64<0x141, 0xF>(v);
  v = dpp_add_f64<0x140, 0xF>(v);
  v = dpp_add_f64<0x142, 0xA>(v);
  v = dpp_add_f64<0x143, 0xC>(v);
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, 63);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// sum / D to the last bit, per_d the rounded 1 / D: the product's remainder is exact in an fma, and the product corrected by it is
// the quotient (of 64-bit numbers; an infinite sum has no remainder). The product alone moves some means that lie halfway
// between two fp32 numbers; a division would take 1 to 3% of the kernels' time (70000 x 128 bf16 27.8 -> 28.5 us).
__device__ __forceinline__ double over_d(double sum, int64_t D, double per_d) {
  const double q = sum * per_d, rest = fma(-q, (double)D, sum);
  return fabs(rest) < __builtin_inf() ? fma(rest, per_d, q) : q;
}
__device__ __forceinline__ float inverse_std(float sum_sq, float D, float eps) { return 1.0f / sqrtf(sum_sq / D + eps); }
// Whether 32 bits did not hold a row's sum of squares: deviations of about 1e19 overflow it (NaN and infinities in the row come
// out here too), and squares under 2^-126 lose their bits, which matters to sums under 1e-30 where eps is as small. Such a
// row's squares are summed again, of deviations times 2^-80 or 2^80, which hold all that counts of either sum. The look at the
// sum costs 1 to 2% (16384 x 2304 bf16 25.8 -> 26.2 us, 4096 x 5120 21.4 -> 22.2); squares in 64 bits from the start cost 2 to
// 9, and lost rows done again behind all others 1 to 7, by registers.
__device__ __forceinline__ bool squares_lost(float sum_sq, float eps) {
  return !(sum_sq < __builtin_inff()) || (sum_sq < 1e-30f && eps < 1e-30f);
}
__device__ __forceinline__ float squares_scale(float sum_sq) { return sum_sq < 1e-30f ? 0x1p80f : 0x1p-80f; }
__device__ __forceinline__ float inverse_std_scaled(float sum_sq, float D, float eps, float c) {
  // (infinite: a deviation itself is, or an element; NaN, as zero would leave the row's other elements at the bias)
  return sum_sq < __builtin_inff() ? c * (1.0f / sqrtf(sum_sq / D + eps * c * c)) : __builtin_nanf("");
}

// ------------------------------------------------------------------ forward
struct FwdArgs {
  const char* x;
  int64_t sxm;  // row strides in bytes here and below
  const void* w;
  const void* b;
  int w_dt, b_dt;
  float eps;
  double per_d;  // 1 / D
  int64_t M, D;
  char* y;
  int64_t sym;
  int y_dt;
  float *mean, *rstd;  // or NULL
  uint8_t* q;          // 8-bit rows of x - mean
  int64_t sq;
  uint8_t* scale;
  int64_t ss;
  int64_t kp;  // D rounded up to whole blocks
  int pad;     // scale bytes behind the last block's
};

// Results of the elements k0 .. k0 + 7 of row m, d = x - mean there.
__device__ __forceinline__ void put_y(const FwdArgs& a, int64_t m, int64_t k0, const float (&d)[8], float rstd) {
  float y[8], p[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = d[e] * rstd;
  if (a.w && a.b) {
    float c[8];
    load8_any(a.w, a.w_dt, k0, a.D, p);
    load8_any(a.b, a.b_dt, k0, a.D, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], p[e], c[e]);
  } else if (a.w) {
    load8_any(a.w, a.w_dt, k0, a.D, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= p[e];
  } else if (a.b) {
    load8_any(a.b, a.b_dt, k0, a.D, p);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] += p[e];
  }
  store8_any(a.y + m * a.sym, a.y_dt, k0, a.D, y);
}

// sff8::quantize8 of finite elements: no look at each for NaN and infinity.
__device__ __forceinline__ u32x2 quantize8_finite(float (&v)[8], uint32_t& byte) {
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
  byte = sff8::scale_byte(sff8::max16(__float_as_uint(top)));
  const float inv = sff8::inverse_of(byte);
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] *= inv;
  return u32x2{sff8::pack4(v[0], v[1], v[2], v[3]), sff8::pack4(v[4], v[5], v[6], v[7])};
}

// The same elements as codes: sixteen lanes hold a block, and all of a wave's lanes come here.
__device__ __forceinline__ void put_codes(const FwdArgs& a, int64_t m, int64_t k0, const float (&d)[8]) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = d[e];
  uint32_t byte;
  const u32x2 codes = sff8::quantize8(v, byte);
  if (k0 < a.kp) {
    *(u32x2*)(a.q + m * a.sq + k0) = codes;
    const int lane16 = threadIdx.x & 15;
    const int64_t kb = k0 / sff8::BLOCK;
    if (lane16 == 0) a.scale[m * a.ss + kb] = (uint8_t)byte;
    if (lane16 > 0 && lane16 <= a.pad && (kb + 1) * sff8::BLOCK == a.kp) a.scale[m * a.ss + kb + lane16] = 0;
  }
}

// A wave a row, U = ceil(D / 512) chunks of eight elements a lane; y is of x's type. The mean's sum and quotient are held in
// 64 bits: the mean, and with it every code of x - mean, is the definition's in every form of this kernel, but where a
// sum that 64 bits do not hold exactly lies within their rounding, 1e-16 of sum |x|, of a border between two fp32 means.
// The wave's next row is under way while this one is worked on: rows leave by buffer stores, whose
// bounds drop the lanes past the last whole chunk without a branch, and weight and bias are kept in LDS as fp32, so
// that no wait for a row's loads waits for anything else. In LDS the lower four elements of all chunks lie before the
// upper four: lanes read 16 B side by side. (16384 x 2304 bf16: 33 us with a row a wave and parameters from L1 -> 25.5; 49
// -> 42 with 8-bit rows, 38 once finite rows, which the sum of squares tells, are not searched for NaN and infinity.)
// A token alone takes 3.6 us, 5.2 before.
// W: waves of a row, one up to 4096 elements and a block's four up to 8192, which then exchange their sums through LDS
// (4096 rows of 5120 in bf16: 22.5 us, 52 by norm_any_kernel; of 8192 31 and 58).
// Up to seven chunks of 16-bit types (five of fp32) without codes keep 128 registers, for the four waves a SIMD that the grid
// gives (8192 x 3500 fp16 20.2 us, 23.2 at 132 registers).
template <int DT, int U, bool HOLD, int W>
__global__ __launch_bounds__(256, W == 1 && !HOLD && U <= (DT == SF_F32 ? 5 : 7) ? 4 : 1) void norm_kernel(FwdArgs a) {
  constexpr int ES = DT == SF_F32 ? 4 : 2, CH = W * U * 64, ROWS = 4 / W;
  constexpr bool bf = DT == SF_BF16;
  __shared__ u32x4 s_par[4 * CH];  // weight's lower and upper halves, then bias's
  __shared__ double s_sum[W > 1 ? 2 : 1][4];
  __shared__ float s_sq[W > 1 ? 2 : 1][4];
  const int lane = threadIdx.x & 63, D = (int)a.D, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c0 = W > 1 ? wave * U : 0;  // the wave's first chunk of 64 lanes
  const bool affine = a.w || a.b;
  auto at = [&](int i) { return ((c0 + i) * 64 + lane) * 8; };
  // only a wave's last chunk, or any of a row's last wave, can run past the row's end
  auto past = [&](int i) { return (W > 1 || i + 1 == U) && (c0 + i + 1) * 512 > D; };
  int64_t m = (int64_t)blockIdx.x * ROWS + (W > 1 ? 0 : wave);
  const int64_t step = (int64_t)gridDim.x * ROWS;
  Raw<ES> raw[U];
  auto load = [&](int64_t row) {
    const char* p = a.x + min(row, a.M - 1) * a.sxm;  // (a wave past the last row loads that again)
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i] = load_at<ES>(p, (uint32_t)(W > 1 || i + 1 == U ? min(at(i), D - 8) : at(i)) * ES);
  };
  load(m);
  if (affine) {
    for (int c = threadIdx.x; c < CH; c += 256) {
      float w[8], b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = 1.f;
        b[e] = 0.f;
      }
      if (a.w) load8_any(a.w, a.w_dt, c * 8, D, w);
      if (a.b) load8_any(a.b, a.b_dt, c * 8, D, b);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s_par[h * CH + c] = u32x4{__float_as_uint(w[4 * h]), __float_as_uint(w[4 * h + 1]), __float_as_uint(w[4 * h + 2]), __float_as_uint(w[4 * h + 3])};
        s_par[(2 + h) * CH + c] = u32x4{__float_as_uint(b[4 * h]), __float_as_uint(b[4 * h + 1]), __float_as_uint(b[4 * h + 2]), __float_as_uint(b[4 * h + 3])};
      }
    }
    __syncthreads();
  }
  int buf = 0;
  for (; m < a.M; m += step, buf ^= 1) {
    float v[U][8];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (past(i)) shift_back(raw[i], max(0, at(i) - (D - 8)));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] = raw_elem(raw[i], e, bf);
        sum += (double)v[i][e];
      }
    }
    load(m + step);
    sum = wave_sum_f64(sum);
    if constexpr (W > 1) {
      if (lane == 0) s_sum[buf][wave] = sum;
      __syncthreads();
      sum = (s_sum[buf][0] + s_sum[buf][1]) + (s_sum[buf][2] + s_sum[buf][3]);
    }
    const float mean = (float)over_d(sum, D, a.per_d);
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < U; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[i][e] -= mean;
        if (W > 1 || i + 1 == U) v[i][e] = at(i) + e < D ? v[i][e] : 0.f;
        sq = fmaf(v[i][e], v[i][e], sq);
      }
    sq = wave_sum(sq);
    if constexpr (W > 1) {
      if (lane == 0) s_sq[buf][wave] = sq;
      __syncthreads();
      sq = (s_sq[buf][0] + s_sq[buf][1]) + (s_sq[buf][2] + s_sq[buf][3]);
    }
    float rstd = inverse_std(sq, (float)D, a.eps);
    if (__builtin_expect(squares_lost(sq, a.eps), 0)) {  // wave-uniform, and with W > 1 the same in the whole block
      const float c = squares_scale(sq);
      sq = 0.f;
#pragma unroll
      for (int i = 0; i < U; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(v[i][e] * c, v[i][e] * c, sq);
      sq = wave_sum(sq);
      if constexpr (W > 1) {
        if (lane == 0) s_sum[buf][wave] = (double)sq;  // (all have read the row's sum: they have met since)
        __syncthreads();
        sq = (float)((s_sum[buf][0] + s_sum[buf][1]) + (s_sum[buf][2] + s_sum[buf][3]));
      }
      rstd = inverse_std_scaled(sq, (float)D, a.eps, c);
      sq = __builtin_inff();  // (not known to be finite)
    }
    if constexpr (HOLD) {
      const bool finite = sq < __builtin_inff();  // so is every element: no NaN or infinity to look for
      const int words = (D + 511) / 512 * 4;
      const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc((void*)(a.q + m * a.sq), (short)0, (int)a.kp, (int)SF_RSRC_W3);
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(a.scale + m * a.ss), (short)0, words, (int)SF_RSRC_W3);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = v[i][e];
        uint32_t byte;
        const u32x2 codes = finite ? quantize8_finite(c, byte) : sff8::quantize8(c, byte);
        __builtin_amdgcn_raw_buffer_store_b64(codes, rq, at(i), 0, 0);
        // four blocks a chunk of 64 lanes: their bytes are one word of the row's scales (zero behind the last block)
        const uint32_t word = (uint32_t)__builtin_amdgcn_readlane((int)byte, 0) | (uint32_t)__builtin_amdgcn_readlane((int)byte, 16) << 8 |
                              (uint32_t)__builtin_amdgcn_readlane((int)byte, 32) << 16 | (uint32_t)__builtin_amdgcn_readlane((int)byte, 48) << 24;
        __builtin_amdgcn_raw_buffer_store_b32(word, rs, lane == 0 ? 4 * (c0 + i) : words, 0, 0);
      }
    }
    char* out = a.y + m * a.sym;
    const __amdgpu_buffer_rsrc_t ry = __builtin_amdgcn_make_buffer_rsrc((void*)out, (short)0, (D & ~7) * ES, (int)SF_RSRC_W3);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = v[i][e] * rstd;
      if (affine) {
        const int c = (c0 + i) * 64 + lane;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 w = s_par[h * CH + c], b = s_par[(2 + h) * CH + c];
#pragma unroll
          for (int e = 0; e < 4; ++e) y[4 * h + e] = fmaf(y[4 * h + e], __uint_as_float(w[e]), __uint_as_float(b[e]));
        }
      }
      put8_rsrc<DT>(ry, at(i), y);
      if (past(i) && (D & 7) && at(i) < D && at(i) + 8 > D) store8_any(out, DT, at(i), D, y);
    }
    if (lane == 0 && c0 == 0) {
      if (a.mean) a.mean[m] = mean;
      if (a.rstd) a.rstd[m] = rstd;
    }
  }
}

// Sum over a row's NT threads, in every one of them: a wave, or a block of 1024.
template <int NT>
__device__ __forceinline__ double row_sum(double v, double*) { return wave_sum_f64(v); }
template <int NT>
__device__ __forceinline__ float row_sum(float v, float*) { return wave_sum(v); }
template <class T>
__device__ __forceinline__ T block_sum_1024(T v, T* s_w) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  v = row_sum<64>(v, s_w);
  __syncthreads();  // the last sum has been read
  if (lane == 0) s_w[w] = v;
  __syncthreads();
  T s = s_w[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) s += s_w[i];
  return s;
}
template <>
__device__ __forceinline__ double row_sum<1024>(double v, double* s) { return block_sum_1024(v, s); }
template <>
__device__ __forceinline__ float row_sum<1024>(float v, float* s) { return block_sum_1024(v, s); }

// Everything else, in three passes over the row, the last two out of the caches: a wave a row where y is of another type
// than x or rows have less than eight elements (16384 x 2304 bf16 to fp32 57 us, 4.0 TB/s), a block of 1024 a row where no
// block holds it (2048 rows of 12288 in bf16 40 us, 2.5 TB/s of the bytes that it cannot do without, fp32 48, 4.2; 512 of
// 32768 bf16 25, 2.7): each pass waits for the row's sum before the next one's loads begin.
template <int DT, bool HOLD, int NT>
__global__ __launch_bounds__(NT == 64 ? 256 : 1024) void norm_any_kernel(FwdArgs a) {
  constexpr int ES = DT == SF_F32 ? 4 : 2, ROWS = NT == 64 ? 4 : 1;
  constexpr bool bf = DT == SF_BF16;
  __shared__ double s_d[16];
  __shared__ float s_f[16];
  const int t = threadIdx.x % NT;
  const int64_t first = (int64_t)blockIdx.x * ROWS + (NT == 64 ? (int)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
  for (int64_t m = first; m < a.M; m += (int64_t)gridDim.x * ROWS) {
    const char* row = a.x + m * a.sxm;
    double sum = 0.0;
    for (int64_t k0 = t * 8; k0 < a.D; k0 += NT * 8) {
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (double)raw_elem(r, e, bf);
    }
    const float mean = (float)over_d(row_sum<NT>(sum, s_d), a.D, a.per_d);
    float sq = 0.f;
    for (int64_t k0 = t * 8; k0 < a.D; k0 += NT * 8) {
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = k0 + e < a.D ? raw_elem(r, e, bf) - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    sq = row_sum<NT>(sq, s_f);
    float rstd = inverse_std(sq, (float)a.D, a.eps);
    if (squares_lost(sq, a.eps)) {  // the same in all of the row's threads
      const float c = squares_scale(sq);
      sq = 0.f;
      for (int64_t k0 = t * 8; k0 < a.D; k0 += NT * 8) {
        const Raw<ES> r = load_raw<ES>(row, k0, a.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float d = k0 + e < a.D ? (raw_elem(r, e, bf) - mean) * c : 0.f;
          sq = fmaf(d, d, sq);
        }
      }
      rstd = inverse_std_scaled(row_sum<NT>(sq, s_f), (float)a.D, a.eps, c);
    }
    if (t == 0) {
      if (a.mean) a.mean[m] = mean;
      if (a.rstd) a.rstd[m] = rstd;
    }
    for (int64_t k = 0; k < a.kp; k += NT * 8) {  // (whole waves: the lanes of a block of codes stay together)
      const int64_t k0 = k + t * 8;
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = k0 + e < a.D ? raw_elem(r, e, bf) - mean : 0.f;
      if (HOLD) put_codes(a, m, k0, d);
      if (k0 < a.D) put_y(a, m, k0, d, rstd);
    }
  }
}

// ------------------------------------------------------------------ backward
struct BwdArgs {
  const char* g;
  int64_t sgm;
  int g_dt;
  const char* x;  // or 8-bit rows of x - mean
  int64_t sxm;
  const uint8_t* q;
  int64_t sq;
  const uint8_t* scale;
  int64_t ss;
  const float *mean, *rstd;
  const void* w;
  int w_dt;
  const float *g_mean, *g_rstd;  // or NULL
  int64_t M, D;
  char* dx;
  int64_t sdx;
  int dx_dt;
  void *dw, *db;  // either may be NULL
  int dw_dt, db_dt;
  float* part;  // [blocks][2][D]
  int T, TB;    // waves of a row's team, teams of a block
};

// Eight elements of a row in the form they come in.
template <int XT>
struct XRaw {
  static constexpr int ES = XT == SF_F32 ? 4 : 2;
  Raw<ES> v;
  __device__ __forceinline__ void load(const BwdArgs& a, int64_t m, int64_t k0) { v = load_raw<ES>(a.x + m * a.sxm, k0, a.D); }
  __device__ __forceinline__ void load_back(const BwdArgs& a, int64_t m, int64_t k0) {
    v = ::load_back<ES>(a.x + m * a.sxm, k0, a.D);
  }
  __device__ __forceinline__ void load_at(const BwdArgs& a, int64_t m, uint32_t k) { v = ::load_at<ES>(a.x + m * a.sxm, k * ES); }
  __device__ __forceinline__ void shift_back(int off) { ::shift_back(v, off); }
  // xh
  __device__ __forceinline__ void normed(float mean, float rstd, float (&xh)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) xh[e] = (raw_elem(v, e, XT == SF_BF16) - mean) * rstd;
  }
};
template <>
struct XRaw<X_FP8> {
  u32x2 c;
  uint32_t byte;
  __device__ __forceinline__ void load(const BwdArgs& a, int64_t m, int64_t k0) {
    c = u32x2{0, 0};
    byte = 0;
    if (k0 < a.D) {  // (rows are padded to whole blocks)
      c = *(const u32x2*)(a.q + m * a.sq + k0);
      byte = a.scale[m * a.ss + k0 / sff8::BLOCK];
    }
  }
  __device__ __forceinline__ void load_at(const BwdArgs& a, int64_t m, uint32_t k) {
    c = *(const u32x2*)(a.q + m * a.sq + k);
    byte = (a.scale + m * a.ss)[k / sff8::BLOCK];
  }
  __device__ __forceinline__ void load_back(const BwdArgs& a, int64_t m, int64_t k0) {
    const int64_t k = min(k0, (a.D - 1) & ~(int64_t)7);  // a lane past the row's end loads its last chunk
    c = *(const u32x2*)(a.q + m * a.sq + k);
    byte = a.scale[m * a.ss + k / sff8::BLOCK];
  }
  __device__ __forceinline__ void shift_back(int off) {
    if (off >= 8) c = u32x2{0, 0};
  }
  __device__ __forceinline__ void normed(float, float rstd, float (&xh)[8]) const {
    const float f = sff8::scale_of(byte) * rstd;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const sff8::f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false);
      const sff8::f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
      xh[4 * i] = lo[0] * f;
      xh[4 * i + 1] = lo[1] * f;
      xh[4 * i + 2] = hi[0] * f;
      xh[4 * i + 3] = hi[1] * f;
    }
  }
};

__device__ __forceinline__ void put_param(void* p, int dt, int64_t i, float v) {
  if (dt == SF_F32) ((float*)p)[i] = v;
  else ((u16*)p)[i] = (u16)f32_to_bits(v, dt);
}

// A team's column sums: the parameters' gradients if its block is the only one, else its part of them.
__device__ __forceinline__ void put_sums(const BwdArgs& a, int64_t k0, const float (&acc_w)[8], const float (&acc_b)[8]) {
  if (gridDim.x == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < a.D) {
        if (a.dw) put_param(a.dw, a.dw_dt, k0 + e, acc_w[e]);
        if (a.db) put_param(a.db, a.db_dt, k0 + e, acc_b[e]);
      }
  } else if (k0 < a.D) {
    char* p = (char*)(a.part + (int64_t)blockIdx.x * 2 * a.D);
    store8_any(p, SF_F32, k0, a.D, acc_w);
    store8_any(p + a.D * 4, SF_F32, k0, a.D, acc_b);
  }
}

// The general form: types that mix, up to 8192 elements. R rows at a time by a team of T <= 8 waves, a lane holding the same U chunks of eight columns of every row, so
// that the columns' sums stay in its registers over all rows of the block. A row's two sums go over the team
// through LDS, those of R rows together (one barrier a batch, two buffers), while the next batch's loads are under
// way. Teams of one or two waves share a block, which adds up its teams' column sums at the end. (With the parameters'
// sums: 16384 x 2304, x in bf16 and g in fp32, 75 us, 4.0 TB/s; all bf16 4096 x 5120 43 us, 2.9 TB/s, from 8-bit rows 43, 4096 x
// 8192 51, 3.9, and 49: two chunks a lane take 173 registers, two waves a SIMD.)
constexpr int MAX_T = 8;
template <int XT, int GT, int U>
__global__ __launch_bounds__(64 * MAX_T) void norm_backward_kernel(BwdArgs a) {
  constexpr int R = 4 / U, GES = GT == SF_F32 ? 4 : 2;
  constexpr bool bf = GT == SF_BF16;
  __shared__ float s_sum[2][MAX_T][8];
  __shared__ float s_acc[U == 1 ? 3 * 64 * 16 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wave / a.T, tw = wave - team * a.T;
  int64_t k0[U];
  int off[U];
  float w[U][8], acc_w[U][8], acc_b[U][8];
  const bool past = (tw + 1) * U * 512 > a.D;  // the wave holds the row's end
#pragma unroll
  for (int u = 0; u < U; ++u) {
    k0[u] = ((tw * U + u) * 64 + lane) * 8;
    off[u] = (int)max((int64_t)0, k0[u] - (a.D - 8));
    if (a.w) {
      load8_any(a.w, a.w_dt, k0[u], a.D, w[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[u][e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) acc_w[u][e] = acc_b[u][e] = 0.f;
  }
  const int64_t batches = (a.M + R - 1) / R, step = (int64_t)gridDim.x * a.TB;
  Raw<GES> g[R][U];
  XRaw<XT> x[R][U];
  float stat_r[R], stat_m[R];
  auto load = [&](int64_t batch) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t m = min(batch * R + r, a.M - 1);  // rows past the last are loaded again and left out below
      stat_r[r] = a.rstd[m];
      stat_m[r] = XT == X_FP8 ? 0.f : a.mean[m];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        g[r][u] = load_back<GES>(a.g + m * a.sgm, k0[u], a.D);
        x[r][u].load_back(a, m, k0[u]);
      }
    }
  };
  int64_t batch = (int64_t)blockIdx.x * a.TB + team;
  load(batch);
  int buf = 0;
  for (int64_t b0 = (int64_t)blockIdx.x * a.TB; b0 < batches; b0 += step, batch += step, buf ^= 1) {
    Raw<GES> gc[R][U];
    XRaw<XT> xc[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        gc[r][u] = g[r][u];
        xc[r][u] = x[r][u];
        if (past) {
          shift_back(gc[r][u], off[u]);
          xc[r][u].shift_back(off[u]);
        }
      }
    float rstd[R], mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      rstd[r] = stat_r[r];
      mean[r] = stat_m[r];
    }
    load(batch + step);
    float s[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (batch * R + r < a.M) {  // wave-uniform
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float xh[8];
          xc[r][u].normed(mean[r], rstd[r], xh);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float ge = raw_elem(gc[r][u], e, bf), q = ge * w[u][e];
            acc_w[u][e] = fmaf(ge, xh[e], acc_w[u][e]);
            acc_b[u][e] += ge;
            s[2 * r] += q;
            s[2 * r + 1] = fmaf(q, xh[e], s[2 * r + 1]);
          }
        }
      }
    }
    if (a.dx) {
      float tot = wave_sum8(s, lane);  // lane l: s[l >> 3]
      if (a.T > 1) {
        if ((lane & 7) == 0) s_sum[buf][wave][lane >> 3] = tot;
        __syncthreads();
        tot = 0.f;
        for (int t = 0; t < a.T; ++t) tot += s_sum[buf][team * a.T + t][lane >> 3];
      }
      const float per = tot / (float)a.D;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t m = batch * R + r;
        const float c1 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(per), 16 * r));
        float c2 = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(per), 16 * r + 8));
        if (m < a.M) {
          const float c0 = a.g_mean ? a.g_mean[m] / (float)a.D : 0.f;
          if (a.g_rstd) c2 += a.g_rstd[m] * rstd[r] / (float)a.D;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            if (k0[u] >= a.D) continue;
            float xh[8], o[8];
            xc[r][u].normed(mean[r], rstd[r], xh);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float q = raw_elem(gc[r][u], e, bf) * w[u][e];
              o[e] = fmaf(rstd[r], q - c1 - xh[e] * c2, c0);
            }
            store8_any(a.dx + m * a.sdx, a.dx_dt, k0[u], a.D, o);
          }
        }
      }
    }
  }
  if (!a.dw && !a.db) return;
  if constexpr (U == 1) {
    if (a.TB > 1) {  // at most 4 waves
      if (team > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s_acc[(((team - 1) * a.T + tw) * 16 + e) * 64 + lane] = acc_w[0][e];
          s_acc[(((team - 1) * a.T + tw) * 16 + 8 + e) * 64 + lane] = acc_b[0][e];
        }
      }
      __syncthreads();
      if (team > 0) return;
      for (int t = 0; t < a.TB - 1; ++t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          acc_w[0][e] += s_acc[((t * a.T + tw) * 16 + e) * 64 + lane];
          acc_b[0][e] += s_acc[((t * a.T + tw) * 16 + 8 + e) * 64 + lane];
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) put_sums(a, k0[u], acc_w[u], acc_b[u]);
}

// The usual case of the above, straight through: x and dx of g's type (or x in 8 bits), up to 4096 elements. What
// differs is what keeps the loads going. A row's result leaves by a buffer store, whose bounds drop the lanes past
// the row's last whole chunk and rows past the last without a branch, so that waiting for the next row's loads does not
// wait for the last row's stores. Elements are unpacked once, into the registers that both halves use, and g xh is formed
// once for both sums it is in: thirteen vector instructions an element (16384 x 2304 bf16: 67 us by the general form). One row
// at a time keeps the registers at 80 (96 in fp32), for two blocks of up to ten waves a CU: 5 us less than two rows at 128
// registers, from 8-bit rows 15 less than at 96. A single block for few rows, which would save the launch
// of norm_params_kernel, was slower from 16 rows on (32 rows 21 us against 14). The row's sums are multiplied by a rounded
// 1 / D, half a unit more of error than a division's. A team of one row each makes a part for every few rows: 2048 x 768 fp32
// takes 10 us and another 5.8 to add 410 parts up, four times what its bytes need.
constexpr int FAST_WAVES = 10;
template <int XT, int GT>
__global__ __launch_bounds__(64 * FAST_WAVES, GT == SF_F32 ? 5 : 6) void norm_backward_fast_kernel(BwdArgs a) {
  constexpr int ES = GT == SF_F32 ? 4 : 2;
  constexpr bool bf = GT == SF_BF16;
  __shared__ float s_sum[2][FAST_WAVES][2];
  __shared__ float s_acc[(FAST_WAVES - 1) * 64 * 16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wave / a.T, tw = wave - team * a.T, D = (int)a.D;
  const int k0 = (tw * 64 + lane) * 8, off = max(0, k0 - (D - 8));
  const bool past = (tw + 1) * 512 > D;  // the wave holds the row's end
  const uint32_t kg = (uint32_t)min(k0, D - 8), kx = XT == X_FP8 ? (uint32_t)min(k0, (D - 1) & ~7) : kg;
  float w[8], acc_w[8], acc_b[8];
  if (a.w) {
    load8_any(a.w, a.w_dt, k0, D, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc_w[e] = acc_b[e] = 0.f;
  const int64_t step = (int64_t)gridDim.x * a.TB;
  const float per_d = 1.0f / (float)D;
  Raw<ES> g;
  XRaw<XT> x;
  float rstd_n, mean_n, gm_n, gr_n;
  const float *g_mean = a.g_mean ? a.g_mean : a.rstd, *g_rstd = a.g_rstd ? a.g_rstd : a.rstd;  // (loads without a branch)
  auto load = [&](int64_t row) {
    const int64_t m = min(row, a.M - 1);  // a team past the last row loads that again, and leaves it out below
    g = load_at<ES>(a.g + m * a.sgm, kg * ES);
    x.load_at(a, m, kx);
    rstd_n = a.rstd[m];
    mean_n = XT == X_FP8 ? 0.f : a.mean[m];
    gm_n = g_mean[m];
    gr_n = g_rstd[m];
  };
  int64_t m = (int64_t)blockIdx.x * a.TB + team;
  load(m);
  int buf = 0;
  for (int64_t m0 = (int64_t)blockIdx.x * a.TB; m0 < a.M; m0 += step, m += step, buf ^= 1) {
    const bool in = m < a.M;  // wave-uniform
    const float rstd = rstd_n, gm = a.g_mean ? gm_n : 0.f, gr = a.g_rstd ? gr_n : 0.f;
    if (past) {
      shift_back(g, off);
      x.shift_back(off);
    }
    float ge[8], xh[8], s1 = 0.f, s2 = 0.f;
    x.normed(mean_n, rstd, xh);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ge[e] = in ? raw_elem(g, e, bf) : 0.f;
      xh[e] = in ? xh[e] : 0.f;
    }
    load(m + step);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = ge[e] * xh[e];
      acc_w[e] += t;
      acc_b[e] += ge[e];
      s1 = fmaf(ge[e], w[e], s1);
      s2 = fmaf(t, w[e], s2);
    }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    if (a.T > 1) {
      if (lane == 0) {
        s_sum[buf][wave][0] = s1;
        s_sum[buf][wave][1] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
      for (int t = 0; t < a.T; ++t) {
        s1 += s_sum[buf][team * a.T + t][0];
        s2 += s_sum[buf][team * a.T + t][1];
      }
    }
    const float k1 = fmaf(gm, per_d, -rstd * (s1 * per_d)), k2 = -rstd * fmaf(gr * rstd, per_d, s2 * per_d);
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmaf(xh[e], k2, fmaf(ge[e] * w[e], rstd, k1));
    char* out = a.dx + min(m, a.M - 1) * a.sdx;
    const bool put = in && a.dx;  // without dx its bounds drop all of it: a branch would have loads wait for stores
    const __amdgpu_buffer_rsrc_t rs =
        __builtin_amdgcn_make_buffer_rsrc((void*)out, (short)0, put ? (D & ~7) * ES : 0, (int)SF_RSRC_W3);
    put8_rsrc<GT>(rs, k0, o);
    if (past && put && (D & 7) && k0 < D && k0 + 8 > D) store8_any(out, GT, k0, D, o);
  }
  if (!a.dw && !a.db) return;
  if (a.TB > 1) {
    if (team > 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s_acc[((wave - a.T) * 16 + e) * 64 + lane] = acc_w[e];
        s_acc[((wave - a.T) * 16 + 8 + e) * 64 + lane] = acc_b[e];
      }
    }
    __syncthreads();
    if (team > 0) return;
    for (int t = tw; t < (a.TB - 1) * a.T; t += a.T) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        acc_w[e] += s_acc[(t * 16 + e) * 64 + lane];
        acc_b[e] += s_acc[(t * 16 + 8 + e) * 64 + lane];
      }
    }
  }
  put_sums(a, k0, acc_w, acc_b);
}

// The parameters' gradients from the blocks' parts, in a fixed order: column c of [2][D] by 16 waves, wave i
// taking parts i, i + 16, ... (P = 0: zeros). 4.6 us for 512 parts of 2304.
__global__ __launch_bounds__(1024) void norm_params_kernel(const float* part, int64_t P, int64_t D, void* dw, int dw_dt,
                                                           void* db, int db_dt) {
  __shared__ float s_part[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * 64 + lane, cc = min(c, 2 * D - 1);
  float s = 0.f;
#pragma unroll 16
  for (int64_t p = w; p < P; p += 16) s += part[p * 2 * D + cc];
  s_part[w][lane] = s;
  __syncthreads();
  if (w != 0 || c >= 2 * D) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += s_part[i][lane];
  if (c < D) {
    if (dw) put_param(dw, dw_dt, c, s);
  } else if (db) {
    put_param(db, db_dt, c - D, s);
  }
}

// Rows longer than a team holds, or shorter than eight elements: dx by a block a row in two passes ... (With the
// parameters' sums, which read x and g a third time: 2048 x 12288 bf16 62 us, 2.4 TB/s of the bytes that it cannot do without,
// fp32 97, 3.1; 512 x 32768 bf16 48, 2.1. Rows under eight elements keep one lane of a block's 1024 busy: 65536 x 4 1.3 ms.)
template <int XT, int GT>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(BwdArgs a) {
  constexpr int GES = GT == SF_F32 ? 4 : 2;
  constexpr bool bf = GT == SF_BF16;
  __shared__ float s_w[16];
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const float rstd = a.rstd[m], mean = XT == X_FP8 ? 0.f : a.mean[m];
    float s1 = 0.f, s2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      float c0 = 0.f, c1 = 0.f, c2 = 0.f;
      if (pass == 1) {
        c1 = block_sum_1024(s1, s_w) / (float)a.D;
        c2 = block_sum_1024(s2, s_w) / (float)a.D;
        if (a.g_mean) c0 = a.g_mean[m] / (float)a.D;
        if (a.g_rstd) c2 += a.g_rstd[m] * rstd / (float)a.D;
      }
      for (int64_t k0 = threadIdx.x * 8; k0 < a.D; k0 += 8192) {
        const Raw<GES> g = load_raw<GES>(a.g + m * a.sgm, k0, a.D);
        XRaw<XT> x;
        x.load(a, m, k0);
        float w[8], xh[8], o[8];
        if (a.w) {
          load8_any(a.w, a.w_dt, k0, a.D, w);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = 1.f;
        }
        x.normed(mean, rstd, xh);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = raw_elem(g, e, bf) * w[e];
          if (pass == 0 && k0 + e < a.D) {
            s1 += q;
            s2 = fmaf(q, xh[e], s2);
          }
          o[e] = fmaf(rstd, q - c1 - xh[e] * c2, c0);
        }
        if (pass == 1) store8_any(a.dx + m * a.sdx, a.dx_dt, k0, a.D, o);
      }
    }
  }
}
// ... and the parameters' gradients by a pass over columns: block (x, y) sums 512 columns a wave over the y-th share of rows.
template <int XT, int GT>
__global__ __launch_bounds__(64) void norm_columns_kernel(BwdArgs a) {
  const int64_t k0 = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 8;
  if (k0 >= a.D) return;
  constexpr int GES = GT == SF_F32 ? 4 : 2;
  constexpr bool bf = GT == SF_BF16;
  float acc_w[8] = {}, acc_b[8] = {};
  for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y) {
    const Raw<GES> g = load_raw<GES>(a.g + m * a.sgm, k0, a.D);
    XRaw<XT> x;
    x.load(a, m, k0);
    float xh[8];
    x.normed(XT == X_FP8 ? 0.f : a.mean[m], a.rstd[m], xh);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = raw_elem(g, e, bf);
      acc_w[e] = fmaf(ge, xh[e], acc_w[e]);
      acc_b[e] += ge;
    }
  }
  char* p = (char*)(a.part + (int64_t)blockIdx.y * 2 * a.D);
  store8_any(p, SF_F32, k0, a.D, acc_w);
  store8_any(p + a.D * 4, SF_F32, k0, a.D, acc_b);
}

// ------------------------------------------------------------------ the norm undone
struct UndoArgs {
  const char* h;
  int64_t shm;
  const float *mean, *rstd;
  int64_t M, D;
  char* out;
  int64_t som;
  int out_dt;
  const char* g;
  int64_t sgm;
  float *dmean, *drstd;  // or NULL
};

// 1 / rstd to 48 bits as r + e: v / rstd is then v r + v e, off by little more than its own rounding.
__device__ __forceinline__ void inverse_pair(float rstd, float& r, float& e) {
  r = 1.0f / rstd;
  e = fmaf(-rstd, r, 1.0f) * r;
  if (!(fabsf(e) < __builtin_inff())) e = 0.f;  // rstd of zero or infinity
}
// v r + (v e + rest): v / rstd + rest. A lower part that is infinite or no number (v is, or v r is far past the largest
// number) would undo the upper one and is left out.
__device__ __forceinline__ float times_pair(float v, float r, float e, float rest) {
  const float low = fmaf(v, e, rest);
  return fmaf(v, r, fabsf(low) < __builtin_inff() ? low : rest);
}

// out = h / rstd + mean, a wave a row. Bound by memory: 24 us for 16384 x 2304 in bf16 (6.3 TB/s).
template <int HT>
__global__ __launch_bounds__(256) void undo_kernel(UndoArgs a) {
  constexpr int ES = HT == SF_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  for (int64_t m = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); m < a.M; m += (int64_t)gridDim.x * 4) {
    float r, c;
    inverse_pair(a.rstd[m], r, c);
    const float mean = a.mean[m];
    for (int64_t k0 = lane * 8; k0 < a.D; k0 += 512) {
      const Raw<ES> h = load_raw<ES>(a.h + m * a.shm, k0, a.D);
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = raw_elem(h, e, HT == SF_BF16);
        o[e] = times_pair(v, r, c, mean);
      }
      store8_any(a.out + m * a.som, a.out_dt, k0, a.D, o);
    }
  }
}

// dh = g / rstd (out), dmean = sum g, drstd = -sum g h / rstd^2, a wave a row: 35 to 39 us there.
template <int GT, int HT>
__global__ __launch_bounds__(256) void undo_backward_kernel(UndoArgs a) {
  constexpr int GES = GT == SF_F32 ? 4 : 2, HES = HT == SF_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  for (int64_t m = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); m < a.M; m += (int64_t)gridDim.x * 4) {
    float r, c, s1 = 0.f, s2 = 0.f;
    inverse_pair(a.rstd[m], r, c);
    for (int64_t k0 = lane * 8; k0 < a.D; k0 += 512) {
      const Raw<GES> g = load_raw<GES>(a.g + m * a.sgm, k0, a.D);
      if (a.drstd) {
        const Raw<HES> h = load_raw<HES>(a.h + m * a.shm, k0, a.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ge = raw_elem(g, e, GT == SF_BF16);
          s2 = fmaf(ge, raw_elem(h, e, HT == SF_BF16), s2);
        }
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ge = raw_elem(g, e, GT == SF_BF16);
        s1 += ge;
        o[e] = times_pair(ge, r, c, 0.f);
      }
      if (a.out) store8_any(a.out + m * a.som, a.out_dt, k0, a.D, o);
    }
    if (a.dmean || a.drstd) {
      s1 = wave_sum(s1);
      s2 = wave_sum(s2);
      if (lane == 0) {
        if (a.dmean) a.dmean[m] = s1;
        if (a.drstd) a.drstd[m] = -s2 * r * r;
      }
    }
  }
}

// ------------------------------------------------------------------ host
constexpr int64_t MAX_M = (1ll << 31) - 1, MAX_D = 1 << 24;
constexpr int64_t WAVE_D = 4096;          // the longest row a wave of norm_kernel holds
constexpr int64_t ROW_D = 8192;           // the longest its block holds
constexpr int64_t FWD_BLOCKS = 1024;      // of four waves: four a CU
constexpr int64_t TEAM_D = MAX_T * 1024;  // the longest row a team of norm_backward_kernel holds, two chunks a lane
constexpr int64_t FAST_D = 4096;          // the longest of norm_backward_fast_kernel
constexpr int64_t MOST_PARTS = 512;       // blocks of the backward pass: two a CU

int check_matrix(const char* what, const void* p, int64_t stride, int dt, int64_t M, int64_t D) {
  SF_REQUIRE(sf_valid_dtype(dt), "%s: unsupported dtype code", what);
  SF_REQUIRE(p, "%s must not be NULL", what);
  SF_REQUIRE((uintptr_t)p % sf_dtype_size(dt) == 0, "%s is not aligned to its elements", what);
  SF_REQUIRE(stride >= 0, "%s: negative row stride", what);
  return SF_OK;
}
int check_result(const char* what, const void* p, int64_t stride, int dt, int64_t M, int64_t D) {
  if (const int rc = check_matrix(what, p, stride, dt, M, D)) return rc;
  SF_REQUIRE(stride >= D || M == 1, "%s: rows overlap", what);
  return SF_OK;
}
int check_held(const void* q, int64_t sq, const void* scale, int64_t ss, int64_t D) {
  SF_REQUIRE(q && scale, "codes and scales must not be NULL");
  SF_REQUIRE(((uintptr_t)q & 15) == 0 && sq % 16 == 0, "rows of codes must be 16-B aligned");
  SF_REQUIRE(((uintptr_t)scale & 3) == 0 && ss % 4 == 0, "rows of scales must be 4-B aligned");
  SF_REQUIRE(sq >= sff8::code_bytes(D) && ss >= sff8::scale_bytes(D), "rows of 8 bits are too short for %lld elements",
             (long long)D);
  return SF_OK;
}
int check_shape(int64_t M, int64_t D) {
  SF_REQUIRE(M >= 0 && M <= MAX_M && D >= 1 && D <= MAX_D, "bad shape [%lld, %lld]", (long long)M, (long long)D);
  return SF_OK;
}

// Waves of a team, teams of a block and blocks of a backward pass.
struct BwdPlan {
  int T, TB, U;
  bool fast;
  int64_t blocks;
};
BwdPlan backward_plan(int64_t M, int64_t D, bool plain) {
  BwdPlan p;
  p.fast = plain && D >= 8 && D <= FAST_D;
  if (D > TEAM_D || D < 8) {
    p.T = p.TB = p.U = 0;
    p.blocks = std::min<int64_t>(M, 64);  // parts of norm_columns_kernel
    return p;
  }
  p.U = D <= MAX_T * 512 ? 1 : 2;
  p.T = (int)((D + 512 * p.U - 1) / (512 * p.U));
  p.TB = p.T == 1 ? 4 : (p.T == 2 ? 2 : 1);
  const int64_t R = p.fast ? 1 : 4 / p.U, batches = (M + R - 1) / R;
  if (p.fast) p.TB = (int)std::max<int64_t>(1, std::min<int64_t>(FAST_WAVES / p.T, batches));
  p.blocks = std::min<int64_t>(MOST_PARTS, (batches + p.TB - 1) / p.TB);
  return p;
}

// The parameters' sums go through parts unless a single block has them all.
int64_t part_bytes(const BwdPlan& p, int64_t D) { return p.T == 0 || p.blocks > 1 ? p.blocks * 2 * D * (int64_t)sizeof(float) : 0; }

template <int DT, bool HOLD>
int forward_typed(const FwdArgs& a, hipStream_t s) {
  if (a.D > ROW_D) {
    hipLaunchKernelGGL((norm_any_kernel<DT, HOLD, 1024>), dim3((unsigned)std::min<int64_t>(a.M, 1 << 16)), dim3(1024), 0, s, a);
  } else if (a.D < 8 || a.y_dt != DT) {
    hipLaunchKernelGGL((norm_any_kernel<DT, HOLD, 64>), dim3((unsigned)std::min<int64_t>((a.M + 3) / 4, 1 << 16)), dim3(256), 0, s, a);
  } else {
    const int waves = a.D <= WAVE_D ? 1 : 4;
    const dim3 grid((unsigned)std::min<int64_t>((a.M * waves + 3) / 4, FWD_BLOCKS));
#define SF_NORM(UV, WV) case 100 * WV + UV: hipLaunchKernelGGL((norm_kernel<DT, UV, HOLD, WV>), grid, dim3(256), 0, s, a); break
    switch (100 * waves + (int)((a.D + 512 * waves - 1) / (512 * waves))) {
      SF_NORM(1, 1);
      SF_NORM(2, 1);
      SF_NORM(3, 1);
      SF_NORM(4, 1);
      SF_NORM(5, 1);
      SF_NORM(6, 1);
      SF_NORM(7, 1);
      SF_NORM(8, 1);
      SF_NORM(3, 4);
      SF_NORM(4, 4);
    }
#undef SF_NORM
  }
  SF_LAUNCH_CHECK("norm_kernel");
  return SF_OK;
}
template <int DT>
int forward_of(const FwdArgs& a, hipStream_t s) {
  return a.q ? forward_typed<DT, true>(a, s) : forward_typed<DT, false>(a, s);
}

template <int XT, int GT>
int backward_typed(BwdArgs& a, const BwdPlan& p, hipStream_t s) {
  const bool pg = a.dw || a.db;
  if (p.T) {
    const dim3 grid((unsigned)p.blocks), block((unsigned)(64 * p.T * p.TB));
    if constexpr (XT == GT || XT == X_FP8) {
      if (p.fast) {
        hipLaunchKernelGGL((norm_backward_fast_kernel<XT, GT>), grid, block, 0, s, a);
        SF_LAUNCH_CHECK("norm_backward_fast_kernel");
        return SF_OK;
      }
    }
    if (p.U == 1) hipLaunchKernelGGL((norm_backward_kernel<XT, GT, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_backward_kernel<XT, GT, 2>), grid, block, 0, s, a);
    SF_LAUNCH_CHECK("norm_backward_kernel");
    return SF_OK;
  }
  if (a.dx) {
    hipLaunchKernelGGL((norm_backward_long_kernel<XT, GT>), dim3((unsigned)std::min<int64_t>(a.M, 1 << 16)), dim3(1024), 0, s, a);
    SF_LAUNCH_CHECK("norm_backward_long_kernel");
  }
  if (pg) {
    hipLaunchKernelGGL((norm_columns_kernel<XT, GT>), dim3((unsigned)((a.D + 511) / 512), (unsigned)p.blocks), dim3(64), 0, s, a);
    SF_LAUNCH_CHECK("norm_columns_kernel");
  }
  return SF_OK;
}

template <int XT>
int backward_of(BwdArgs& a, const BwdPlan& p, hipStream_t s) {
  switch (a.g_dt) {
    case SF_F32: return backward_typed<XT, SF_F32>(a, p, s);
    case SF_BF16: return backward_typed<XT, SF_BF16>(a, p, s);
    default: return backward_typed<XT, SF_F16>(a, p, s);
  }
}

}  // namespace

extern "C" int sf_layer_norm(const void* x, int64_t sxm, int x_dt, const void* w, int w_dt, const void* b, int b_dt,
                             float eps, int64_t M, int64_t D, void* y, int64_t sym, int y_dt, float* mean, float* rstd,
                             void* q, int64_t sq, void* scale, int64_t ss, void* stream) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  SF_REQUIRE(eps >= 0.f, "eps must not be negative");
  SF_REQUIRE((!w || sf_valid_dtype(w_dt)) && (!b || sf_valid_dtype(b_dt)), "unsupported dtype code");
  SF_REQUIRE(sf_valid_dtype(x_dt) && sf_valid_dtype(y_dt), "unsupported dtype code");
  if (M == 0) return SF_OK;
  if (const int rc = check_matrix("x", x, sxm, x_dt, M, D)) return rc;
  if (const int rc = check_result("y", y, sym, y_dt, M, D)) return rc;
  if (q || scale)
    if (const int rc = check_held(q, sq, scale, ss, D)) return rc;
  const int es = sf_dtype_size(x_dt);
  FwdArgs a;
  a.x = (const char*)x; a.sxm = sxm * es; a.w = w; a.b = b; a.w_dt = w_dt; a.b_dt = b_dt; a.eps = eps;
  a.per_d = 1.0 / (double)D;
  a.M = M; a.D = D; a.y = (char*)y; a.sym = sym * sf_dtype_size(y_dt); a.y_dt = y_dt; a.mean = mean; a.rstd = rstd;
  a.q = (uint8_t*)q; a.sq = sq; a.scale = (uint8_t*)scale; a.ss = ss; a.kp = sff8::code_bytes(D);
  a.pad = (int)(sff8::scale_bytes(D) - sff8::blocks_of(D));
  hipStream_t s = (hipStream_t)stream;
  switch (x_dt) {
    case SF_F32: return forward_of<SF_F32>(a, s);
    case SF_BF16: return forward_of<SF_BF16>(a, s);
    default: return forward_of<SF_F16>(a, s);
  }
}

extern "C" int sf_layer_norm_backward_workspace_size(int64_t M, int64_t D, int64_t* bytes) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  SF_REQUIRE(bytes, "sf_layer_norm_backward_workspace_size: NULL result");
  *bytes = std::max(part_bytes(backward_plan(M, D, false), D), part_bytes(backward_plan(M, D, true), D));
  return SF_OK;
}

extern "C" int sf_layer_norm_backward(const void* g, int64_t sgm, int g_dt, const void* x, int64_t sxm, int x_dt,
                                      const void* q, int64_t sq, const void* scale, int64_t ss, const float* mean,
                                      const float* rstd, const void* w, int w_dt, const float* g_mean,
                                      const float* g_rstd, int64_t M, int64_t D, void* dx, int64_t sdx, int dx_dt,
                                      void* dw, int dw_dt, void* db, int db_dt, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  SF_REQUIRE((!w || sf_valid_dtype(w_dt)) && (!dw || sf_valid_dtype(dw_dt)) && (!db || sf_valid_dtype(db_dt)),
             "unsupported dtype code");
  hipStream_t s = (hipStream_t)stream;
  const bool pg = dw || db, plain = (!dx || dx_dt == g_dt) && (!x || x_dt == g_dt);
  const BwdPlan p = backward_plan(M, D, plain);
  if (M > 0) {
    if (const int rc = check_matrix("g", g, sgm, g_dt, M, D)) return rc;
    SF_REQUIRE((x != nullptr) != (q != nullptr), "the input is given as x or in 8 bits, not both");
    if (x) {
      if (const int rc = check_matrix("x", x, sxm, x_dt, M, D)) return rc;
      SF_REQUIRE(mean, "mean must not be NULL");
    } else if (const int rc = check_held(q, sq, scale, ss, D)) {
      return rc;
    }
    SF_REQUIRE(rstd, "rstd must not be NULL");
    if (dx)
      if (const int rc = check_result("dx", dx, sdx, dx_dt, M, D)) return rc;
    const int64_t need = pg ? part_bytes(p, D) : 0;
    SF_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 4 == 0),
               "workspace of %lld bytes, need %lld", (long long)workspace_bytes, (long long)need);
    if (!dx && !pg) return SF_OK;
    BwdArgs a;
    a.g = (const char*)g; a.sgm = sgm * sf_dtype_size(g_dt); a.g_dt = g_dt;
    a.x = (const char*)x; a.sxm = x ? sxm * sf_dtype_size(x_dt) : 0;
    a.q = (const uint8_t*)q; a.sq = sq; a.scale = (const uint8_t*)scale; a.ss = ss;
    a.mean = mean; a.rstd = rstd; a.w = w; a.w_dt = w_dt; a.g_mean = g_mean; a.g_rstd = g_rstd; a.M = M; a.D = D;
    a.dx = (char*)dx; a.sdx = dx ? sdx * sf_dtype_size(dx_dt) : 0; a.dx_dt = dx_dt;
    a.dw = dw; a.db = db; a.dw_dt = dw_dt; a.db_dt = db_dt; a.part = (float*)workspace; a.T = p.T; a.TB = p.TB;
    int rc;
    switch (x ? x_dt : X_FP8) {
      case SF_F32: rc = backward_of<SF_F32>(a, p, s); break;
      case SF_BF16: rc = backward_of<SF_BF16>(a, p, s); break;
      case SF_F16: rc = backward_of<SF_F16>(a, p, s); break;
      default: rc = backward_of<X_FP8>(a, p, s);
    }
    if (rc) return rc;
  }
  if (pg && (M == 0 || p.T == 0 || p.blocks > 1)) {
    hipLaunchKernelGGL(norm_params_kernel, dim3((unsigned)((2 * D + 63) / 64)), dim3(1024), 0, s, (const float*)workspace,
                       M == 0 ? 0 : p.blocks, D, dw, dw_dt, db, db_dt);
    SF_LAUNCH_CHECK("norm_params_kernel");
  }
  return SF_OK;
}

extern "C" int sf_denormalize(const void* h, int64_t shm, int h_dt, const float* mean, const float* rstd, int64_t M,
                              int64_t D, void* out, int64_t som, int out_dt, void* stream) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  if (M == 0) return SF_OK;
  if (const int rc = check_matrix("h", h, shm, h_dt, M, D)) return rc;
  if (const int rc = check_result("out", out, som, out_dt, M, D)) return rc;
  SF_REQUIRE(mean && rstd, "mean and rstd must not be NULL");
  UndoArgs a = {};
  a.h = (const char*)h; a.shm = shm * sf_dtype_size(h_dt); a.mean = mean; a.rstd = rstd; a.M = M; a.D = D;
  a.out = (char*)out; a.som = som * sf_dtype_size(out_dt); a.out_dt = out_dt;
  const dim3 grid((unsigned)std::min<int64_t>((M + 3) / 4, 1 << 20));
  hipStream_t s = (hipStream_t)stream;
  switch (h_dt) {
    case SF_F32: hipLaunchKernelGGL(undo_kernel<SF_F32>, grid, dim3(256), 0, s, a); break;
    case SF_BF16: hipLaunchKernelGGL(undo_kernel<SF_BF16>, grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL(undo_kernel<SF_F16>, grid, dim3(256), 0, s, a);
  }
  SF_LAUNCH_CHECK("undo_kernel");
  return SF_OK;
}

extern "C" int sf_denormalize_backward(const void* g, int64_t sgm, int g_dt, const void* h, int64_t shm, int h_dt,
                                       const float* rstd, int64_t M, int64_t D, void* dh, int64_t sdh, int dh_dt,
                                       float* dmean, float* drstd, void* stream) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  if (M == 0) return SF_OK;
  if (const int rc = check_matrix("g", g, sgm, g_dt, M, D)) return rc;
  if (drstd)
    if (const int rc = check_matrix("h", h, shm, h_dt, M, D)) return rc;
  if (dh)
    if (const int rc = check_result("dh", dh, sdh, dh_dt, M, D)) return rc;
  SF_REQUIRE(rstd, "rstd must not be NULL");
  if (!dh && !dmean && !drstd) return SF_OK;
  UndoArgs a = {};
  a.g = (const char*)g; a.sgm = sgm * sf_dtype_size(g_dt); a.rstd = rstd; a.M = M; a.D = D;
  a.h = drstd ? (const char*)h : nullptr; a.shm = drstd ? shm * sf_dtype_size(h_dt) : 0;
  a.out = (char*)dh; a.som = dh ? sdh * sf_dtype_size(dh_dt) : 0; a.out_dt = dh_dt; a.dmean = dmean; a.drstd = drstd;
  const dim3 grid((unsigned)std::min<int64_t>((M + 3) / 4, 1 << 20));
  hipStream_t s = (hipStream_t)stream;
  auto typed = [&](auto g_tag) {
    constexpr int GT = decltype(g_tag)::value;
    switch (drstd ? h_dt : GT) {
      case SF_F32: hipLaunchKernelGGL((undo_backward_kernel<GT, SF_F32>), grid, dim3(256), 0, s, a); break;
      case SF_BF16: hipLaunchKernelGGL((undo_backward_kernel<GT, SF_BF16>), grid, dim3(256), 0, s, a); break;
      default: hipLaunchKernelGGL((undo_backward_kernel<GT, SF_F16>), grid, dim3(256), 0, s, a);
    }
  };
  switch (g_dt) {
    case SF_F32: typed(std::integral_constant<int, SF_F32>{}); break;
    case SF_BF16: typed(std::integral_constant<int, SF_BF16>{}); break;
    default: typed(std::integral_constant<int, SF_F16>{});
  }
  SF_LAUNCH_CHECK("undo_backward_kernel");
  return SF_OK;
}
