// Layer norm on gfx950: the forward pass (optionally leaving x - mean in 8 bits for the backward pass), the
// backward pass with the reductions of weight's and bias's gradients, and the norm undone.
//
// Row x of D elements: mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), xh = (x - mean) rstd,
// y = xh w + b. Given g = dL/dy, with q = g w:
//   dx = rstd (q - c1 - xh c2),  c1 = sum q / D,  c2 = sum q xh / D;  dw = sum_m g xh,  db = sum_m g.
// Gradients gm and gr of mean and rstd themselves add gm / D - gr rstd^2 xh / D to dx.
//
// All of it is bound by HBM: a row is read once and held in registers between the sums and the result.
#include <algorithm>

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

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
__device__ __forceinline__ float inverse_std(float sum_sq, float D, float eps) { return 1.0f / sqrtf(sum_sq / D + eps); }

// ------------------------------------------------------------------ forward
struct FwdArgs {
  const char* x;
  int64_t sxm;  // row strides in bytes here and below
  const void* w;
  const void* b;
  int w_dt, b_dt;
  float eps;
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

// A wave a row, U chunks of eight elements a lane. The mean's sum is held in 64 bits: it rounds to the same 32 bits
// in whatever order it is formed, so the codes of x - mean are the same in every form of this kernel.
template <int DT, int U, bool HOLD>
__global__ __launch_bounds__(256) void norm_kernel(FwdArgs a) {
  constexpr int ES = DT == SF_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int64_t m = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (m >= a.M) return;
  const char* row = a.x + m * a.sxm;
  Raw<ES> raw[U];
#pragma unroll
  for (int i = 0; i < U; ++i) raw[i] = load_raw<ES>(row, (i * 64 + lane) * 8, a.D);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (double)raw_elem(raw[i], e, DT == SF_BF16);
  const float mean = (float)(wave_sum_f64(sum) / (double)a.D);
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < U; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = (i * 64 + lane) * 8 + e < a.D ? raw_elem(raw[i], e, DT == SF_BF16) - mean : 0.f;
      sq = fmaf(d, d, sq);
    }
  const float rstd = inverse_std(wave_sum(sq), (float)a.D, a.eps);
  if (lane == 0) {
    if (a.mean) a.mean[m] = mean;
    if (a.rstd) a.rstd[m] = rstd;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const int64_t k0 = (i * 64 + lane) * 8;
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = k0 + e < a.D ? raw_elem(raw[i], e, DT == SF_BF16) - mean : 0.f;
    if (HOLD) put_codes(a, m, k0, d);
    if (k0 < a.D) put_y(a, m, k0, d, rstd);
  }
}

// Sum over a block of 1024 threads, in every thread.
template <class T>
__device__ __forceinline__ T block_sum_1024(T v, T* s_w) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  __syncthreads();  // the last sum has been read
  if (lane == 0) s_w[w] = v;
  __syncthreads();
  T s = s_w[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) s += s_w[i];
  return s;
}

// Rows that no wave can hold: a block a row, which is read three times (out of the caches after the first).
template <int DT, bool HOLD>
__global__ __launch_bounds__(1024) void norm_long_kernel(FwdArgs a) {
  constexpr int ES = DT == SF_F32 ? 4 : 2;
  __shared__ double s_d[16];
  __shared__ float s_f[16];
  for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
    const char* row = a.x + m * a.sxm;
    double sum = 0.0;
    for (int64_t k0 = threadIdx.x * 8; k0 < a.D; k0 += 8192) {
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (double)raw_elem(r, e, DT == SF_BF16);
    }
    const float mean = (float)(block_sum_1024(sum, s_d) / (double)a.D);
    float sq = 0.f;
    for (int64_t k0 = threadIdx.x * 8; k0 < a.D; k0 += 8192) {
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = k0 + e < a.D ? raw_elem(r, e, DT == SF_BF16) - mean : 0.f;
        sq = fmaf(d, d, sq);
      }
    }
    const float rstd = inverse_std(block_sum_1024(sq, s_f), (float)a.D, a.eps);
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[m] = mean;
      if (a.rstd) a.rstd[m] = rstd;
    }
    for (int64_t k = 0; k < a.kp; k += 8192) {  // (whole waves: the lanes of a block of codes stay together)
      const int64_t k0 = k + threadIdx.x * 8;
      const Raw<ES> r = load_raw<ES>(row, k0, a.D);
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = k0 + e < a.D ? raw_elem(r, e, DT == SF_BF16) - mean : 0.f;
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

// Eight elements of x - mean in the form they come in.
template <int XT>
struct XRaw {
  static constexpr int ES = XT == SF_F32 ? 4 : 2;
  Raw<ES> v;
  __device__ __forceinline__ void load(const BwdArgs& a, int64_t m, int64_t k0) { v = load_raw<ES>(a.x + m * a.sxm, k0, a.D); }
  __device__ __forceinline__ void centred(float mean, float (&d)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = raw_elem(v, e, XT == SF_BF16) - mean;
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
  __device__ __forceinline__ void centred(float, float (&d)[8]) const {
    const float f = sff8::scale_of(byte);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const sff8::f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], false);
      const sff8::f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[i], true);
      d[4 * i] = lo[0] * f;
      d[4 * i + 1] = lo[1] * f;
      d[4 * i + 2] = hi[0] * f;
      d[4 * i + 3] = hi[1] * f;
    }
  }
};

__device__ __forceinline__ void put_param(void* p, int dt, int64_t i, float v) {
  if (dt == SF_F32) ((float*)p)[i] = v;
  else ((u16*)p)[i] = (u16)f32_to_bits(v, dt);
}

// R rows at a time by a team of T = ceil(D / 512) waves, a lane holding the same eight columns of every row, so
// that the columns' sums stay in its registers over all rows of the block. A row's two sums go over the team
// through LDS, those of R rows together (one barrier a batch, two buffers). Teams of one or two waves share a
// block, which adds up its teams' column sums at the end.
constexpr int R = 4;
constexpr int MAX_T = 16;
template <int XT, int GES, bool DX, bool PG>
__global__ __launch_bounds__(1024) void norm_backward_kernel(BwdArgs a) {
  __shared__ float s_sum[2][MAX_T][2 * R];
  __shared__ float s_acc[PG ? 3 * 64 * 16 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int team = wave / a.T, tw = wave - team * a.T;
  const int64_t k0 = (tw * 64 + lane) * 8;
  const bool live = k0 < a.D, bf = a.g_dt == SF_BF16;
  float w[8];
  if (a.w) {
    load8_any(a.w, a.w_dt, k0, a.D, w);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  }
  float acc_w[8] = {}, acc_b[8] = {};
  const int64_t batches = (a.M + R - 1) / R, step = (int64_t)gridDim.x * a.TB;
  Raw<GES> g[R];
  XRaw<XT> x[R];
  auto load = [&](int64_t batch) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t m = min(batch * R + r, a.M - 1);  // rows past the last are loaded again and left out below
      g[r] = load_raw<GES>(a.g + m * a.sgm, k0, a.D);
      x[r].load(a, m, k0);
    }
  };
  int64_t batch = (int64_t)blockIdx.x * a.TB + team;
  load(batch);
  int buf = 0;
  for (int64_t b0 = (int64_t)blockIdx.x * a.TB; b0 < batches; b0 += step, batch += step, buf ^= 1) {
    Raw<GES> gc[R];
    XRaw<XT> xc[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      gc[r] = g[r];
      xc[r] = x[r];
    }
    float rstd[R], mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t m = min(batch * R + r, a.M - 1);
      rstd[r] = a.rstd[m];
      mean[r] = XT == X_FP8 ? 0.f : a.mean[m];
    }
    load(batch + step);
    float s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool in = batch * R + r < a.M;  // wave-uniform
      s[2 * r] = s[2 * r + 1] = 0.f;
      float d[8];
      xc[r].centred(mean[r], d);
      if (in) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ge = raw_elem(gc[r], e, bf), xh = d[e] * rstd[r], q = ge * w[e];
          if (PG) {
            acc_w[e] = fmaf(ge, xh, acc_w[e]);
            acc_b[e] += ge;
          }
          s[2 * r] += q;
          s[2 * r + 1] = fmaf(q, xh, s[2 * r + 1]);
        }
      }
      if (!live) s[2 * r] = s[2 * r + 1] = 0.f;
    }
    if constexpr (DX) {
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
        if (m < a.M && live) {
          const float c0 = a.g_mean ? a.g_mean[m] / (float)a.D : 0.f;
          if (a.g_rstd) c2 += a.g_rstd[m] * rstd[r] / (float)a.D;
          float d[8], o[8];
          xc[r].centred(mean[r], d);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float q = raw_elem(gc[r], e, bf) * w[e];
            o[e] = fmaf(rstd[r], q - c1 - d[e] * rstd[r] * c2, c0);
          }
          store8_any(a.dx + m * a.sdx, a.dx_dt, k0, a.D, o);
        }
      }
    }
  }
  if constexpr (PG) {
    if (a.TB > 1) {  // at most 4 waves
      if (team > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s_acc[(((team - 1) * a.T + tw) * 16 + e) * 64 + lane] = acc_w[e];
          s_acc[(((team - 1) * a.T + tw) * 16 + 8 + e) * 64 + lane] = acc_b[e];
        }
      }
      __syncthreads();
      if (team > 0) return;
      for (int t = 0; t < a.TB - 1; ++t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          acc_w[e] += s_acc[((t * a.T + tw) * 16 + e) * 64 + lane];
          acc_b[e] += s_acc[((t * a.T + tw) * 16 + 8 + e) * 64 + lane];
        }
      }
    }
    if (gridDim.x == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + e < a.D) {
          if (a.dw) put_param(a.dw, a.dw_dt, k0 + e, acc_w[e]);
          if (a.db) put_param(a.db, a.db_dt, k0 + e, acc_b[e]);
        }
    } else if (live) {
      char* p = (char*)(a.part + (int64_t)blockIdx.x * 2 * a.D);
      store8_any(p, SF_F32, k0, a.D, acc_w);
      store8_any(p + a.D * 4, SF_F32, k0, a.D, acc_b);
    }
  }
}

// The parameters' gradients from the blocks' parts, in a fixed order: column c of [2][D] by 16 waves, wave i
// taking parts i, i + 16, ... (P = 0: zeros).
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

// Rows longer than a team holds: dx by a block a row in two passes ...
template <int XT, int GES>
__global__ __launch_bounds__(1024) void norm_backward_long_kernel(BwdArgs a) {
  __shared__ float s_w[16];
  const bool bf = a.g_dt == SF_BF16;
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
        float w[8], d[8], o[8];
        if (a.w) {
          load8_any(a.w, a.w_dt, k0, a.D, w);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = 1.f;
        }
        x.centred(mean, d);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = raw_elem(g, e, bf) * w[e], xh = d[e] * rstd;
          if (pass == 0 && k0 + e < a.D) {
            s1 += q;
            s2 = fmaf(q, xh, s2);
          }
          o[e] = fmaf(rstd, q - c1 - xh * c2, c0);
        }
        if (pass == 1) store8_any(a.dx + m * a.sdx, a.dx_dt, k0, a.D, o);
      }
    }
  }
}
// ... and the parameters' gradients by a pass over columns: block (x, y) sums 512 columns a wave over the y-th share of rows.
template <int XT, int GES>
__global__ __launch_bounds__(64) void norm_columns_kernel(BwdArgs a) {
  const int64_t k0 = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 8;
  if (k0 >= a.D) return;
  const bool bf = a.g_dt == SF_BF16;
  float acc_w[8] = {}, acc_b[8] = {};
  for (int64_t m = blockIdx.y; m < a.M; m += gridDim.y) {
    const Raw<GES> g = load_raw<GES>(a.g + m * a.sgm, k0, a.D);
    XRaw<XT> x;
    x.load(a, m, k0);
    float d[8];
    x.centred(XT == X_FP8 ? 0.f : a.mean[m], d);
    const float rstd = a.rstd[m];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ge = raw_elem(g, e, bf);
      acc_w[e] = fmaf(ge, d[e] * rstd, acc_w[e]);
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
  if (!(fabsf(e) < 1e30f)) e = 0.f;  // rstd of zero or infinity
}

// out = h / rstd + mean, a wave a row.
template <int ES>
__global__ __launch_bounds__(256) void undo_kernel(UndoArgs a, int h_dt) {
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
        const float v = raw_elem(h, e, h_dt == SF_BF16);
        o[e] = fmaf(v, r, fmaf(v, c, mean));
      }
      store8_any(a.out + m * a.som, a.out_dt, k0, a.D, o);
    }
  }
}

// dh = g / rstd (out), dmean = sum g, drstd = -sum g h / rstd^2, a wave a row.
template <int GES, int HES>
__global__ __launch_bounds__(256) void undo_backward_kernel(UndoArgs a, int g_dt, int h_dt) {
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
          const float ge = raw_elem(g, e, g_dt == SF_BF16);
          s2 = fmaf(ge, raw_elem(h, e, h_dt == SF_BF16), s2);
        }
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float ge = raw_elem(g, e, g_dt == SF_BF16);
        s1 += ge;
        o[e] = fmaf(ge, r, ge * c);
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
constexpr int64_t TEAM_D = MAX_T * 512;   // the longest row a team of norm_backward_kernel holds
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
  int T, TB;
  int64_t blocks;
};
BwdPlan backward_plan(int64_t M, int64_t D) {
  BwdPlan p;
  if (D > TEAM_D) {
    p.T = p.TB = 0;
    p.blocks = std::min<int64_t>(M, 64);
    return p;
  }
  p.T = (int)((D + 511) / 512);
  p.TB = p.T == 1 ? 4 : (p.T == 2 ? 2 : 1);
  const int64_t batches = (M + R - 1) / R;
  p.blocks = std::min<int64_t>(MOST_PARTS, (batches + p.TB - 1) / p.TB);
  return p;
}

template <int DT, bool HOLD>
int forward_typed(const FwdArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.M + 3) / 4));
#define SF_NORM(UV) hipLaunchKernelGGL((norm_kernel<DT, UV, HOLD>), grid, dim3(256), 0, s, a)
  switch (a.D > WAVE_D ? 0 : (a.D + 511) / 512) {
    case 1: SF_NORM(1); break;
    case 2: SF_NORM(2); break;
    case 3: SF_NORM(3); break;
    case 4: SF_NORM(4); break;
    case 5: SF_NORM(5); break;
    case 6: SF_NORM(6); break;
    case 7: SF_NORM(7); break;
    case 8: SF_NORM(8); break;
    default:
      hipLaunchKernelGGL((norm_long_kernel<DT, HOLD>), dim3((unsigned)std::min<int64_t>(a.M, 1 << 16)), dim3(1024), 0, s, a);
  }
#undef SF_NORM
  SF_LAUNCH_CHECK("norm_kernel");
  return SF_OK;
}

template <int XT, int GES>
int backward_typed(BwdArgs& a, const BwdPlan& p, hipStream_t s) {
  const bool pg = a.dw || a.db;
  if (p.T) {
    const dim3 grid((unsigned)p.blocks), block((unsigned)(64 * p.T * p.TB));
    if (a.dx && pg) hipLaunchKernelGGL((norm_backward_kernel<XT, GES, true, true>), grid, block, 0, s, a);
    else if (a.dx) hipLaunchKernelGGL((norm_backward_kernel<XT, GES, true, false>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((norm_backward_kernel<XT, GES, false, true>), grid, block, 0, s, a);
    SF_LAUNCH_CHECK("norm_backward_kernel");
    return SF_OK;
  }
  if (a.dx) {
    hipLaunchKernelGGL((norm_backward_long_kernel<XT, GES>), dim3((unsigned)std::min<int64_t>(a.M, 1 << 16)), dim3(1024), 0, s, a);
    SF_LAUNCH_CHECK("norm_backward_long_kernel");
  }
  if (pg) {
    hipLaunchKernelGGL((norm_columns_kernel<XT, GES>), dim3((unsigned)((a.D + 511) / 512), (unsigned)p.blocks), dim3(64), 0, s, a);
    SF_LAUNCH_CHECK("norm_columns_kernel");
  }
  return SF_OK;
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
  a.M = M; a.D = D; a.y = (char*)y; a.sym = sym * sf_dtype_size(y_dt); a.y_dt = y_dt; a.mean = mean; a.rstd = rstd;
  a.q = (uint8_t*)q; a.sq = sq; a.scale = (uint8_t*)scale; a.ss = ss; a.kp = sff8::code_bytes(D);
  a.pad = (int)(sff8::scale_bytes(D) - sff8::blocks_of(D));
  hipStream_t s = (hipStream_t)stream;
  switch (x_dt) {
    case SF_F32: return q ? forward_typed<SF_F32, true>(a, s) : forward_typed<SF_F32, false>(a, s);
    case SF_BF16: return q ? forward_typed<SF_BF16, true>(a, s) : forward_typed<SF_BF16, false>(a, s);
    default: return q ? forward_typed<SF_F16, true>(a, s) : forward_typed<SF_F16, false>(a, s);
  }
}

extern "C" int sf_layer_norm_backward_workspace_size(int64_t M, int64_t D, int64_t* bytes) {
  sf_clear_error();
  if (const int rc = check_shape(M, D)) return rc;
  SF_REQUIRE(bytes, "sf_layer_norm_backward_workspace_size: NULL result");
  *bytes = backward_plan(M, D).blocks * 2 * D * (int64_t)sizeof(float);
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
  const BwdPlan p = backward_plan(M, D);
  const bool pg = dw || db;
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
    const int64_t need = pg && (p.T == 0 || p.blocks > 1) ? p.blocks * 2 * D * 4 : 0;
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
    const int xt = x ? x_dt : X_FP8;
    const bool g4 = g_dt == SF_F32;
    int rc;
    switch (xt) {
      case SF_F32: rc = g4 ? backward_typed<SF_F32, 4>(a, p, s) : backward_typed<SF_F32, 2>(a, p, s); break;
      case SF_BF16: rc = g4 ? backward_typed<SF_BF16, 4>(a, p, s) : backward_typed<SF_BF16, 2>(a, p, s); break;
      case SF_F16: rc = g4 ? backward_typed<SF_F16, 4>(a, p, s) : backward_typed<SF_F16, 2>(a, p, s); break;
      default: rc = g4 ? backward_typed<X_FP8, 4>(a, p, s) : backward_typed<X_FP8, 2>(a, p, s);
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
  if (h_dt == SF_F32) hipLaunchKernelGGL(undo_kernel<4>, grid, dim3(256), 0, (hipStream_t)stream, a, h_dt);
  else hipLaunchKernelGGL(undo_kernel<2>, grid, dim3(256), 0, (hipStream_t)stream, a, h_dt);
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
  const bool g4 = g_dt == SF_F32, h4 = drstd && h_dt == SF_F32;
  hipStream_t s = (hipStream_t)stream;
  if (g4) {
    if (h4) hipLaunchKernelGGL((undo_backward_kernel<4, 4>), grid, dim3(256), 0, s, a, g_dt, h_dt);
    else hipLaunchKernelGGL((undo_backward_kernel<4, 2>), grid, dim3(256), 0, s, a, g_dt, h_dt);
  } else {
    if (h4) hipLaunchKernelGGL((undo_backward_kernel<2, 4>), grid, dim3(256), 0, s, a, g_dt, h_dt);
    else hipLaunchKernelGGL((undo_backward_kernel<2, 2>), grid, dim3(256), 0, s, a, g_dt, h_dt);
  }
  SF_LAUNCH_CHECK("undo_backward_kernel");
  return SF_OK;
}
