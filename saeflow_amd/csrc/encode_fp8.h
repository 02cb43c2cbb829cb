#pragma once
// The encoder product on 8-bit rows (format: fp8.h):
//   out[m, n] = act(sum_k x[m, k] w[n, k] + b_enc[n]),  x and w the values that codes and scales stand for
// on v_mfma_scale_f32_32x32x64_f8f6f4, whose operands carry a power-of-two scale: each lane hands over
// the scale byte of its row's block, so the scales cost no arithmetic and the sum over K stays in one
// fp32 accumulator from b_enc on. Both operands are rows along K, a K-step is one block of 128
// codes (one cache line of a row), and any order of K within a block that both operands share is
// right, so fragments are read as the 16-bit kernels read theirs (encode_kernels.h).
//
// How exact the 8-bit instruction is (measured with single products, scaled and unscaled forms
// alike): of each eight consecutive products it drops what lies below 2^-13 of the largest of the eight,
// and adds their sum to the accumulator in fp32. Over a row that is an error of 5.5e-5 of the result
// (root mean square, d_in 768, normal operands), a fortieth of a bf16 rounding and a quarter of an fp16 one,
// which stays out of sight there. fp32 results are to be as good as fp32 sums: they take the wide
// form, where fragments become bf16 (exact: four significant bits and a power of two) and the 16-bit
// instruction, which drops nothing above 2^-23, adds them up at half the rate (error 1e-7).
#include "encode_slim.h"
#include "fp8.h"

namespace sff8 {

using sfenc::f32x16;
using sfenc::lds_void;
typedef int i32x8 __attribute__((ext_vector_type(8)));

// The base's xw, Kp (row stride), w, swn (row stride) are the codes; its epilogue fields as elsewhere.
struct F8Args : sfenc::GemmArgs {
  const uint8_t* xs;  // scale bytes, 4-B aligned rows
  int64_t sxs;
  const uint8_t* ws;
  int64_t sws;
};

constexpr int SG = 8;              // groups of four blocks whose scales LDS holds at a time
constexpr int SG_STEPS = 4 * SG;   // K-steps (blocks) they cover: 4096 elements

// acc += A (8 codes x 4 dwords of one feature row) * B (one token row), scale bytes in byte 0
__device__ __forceinline__ void mfma_f8(f32x16& acc, const i32x8& a, const i32x8& b, int sa, int sb) {
  acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, acc, 0, 0, 0, sa, 0, sb);
}

// The wide form: the 32 codes a lane holds of each operand as four bf16 MFMAs of 16 (fa, fb: the rows'
// scales).
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ sfenc::bf16x8 widen8(const i32x8& v, int part, float scale) {
  const bf16x2 w[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * part], scale, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * part], scale, true),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * part + 1], scale, false),
                       __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[2 * part + 1], scale, true)};
  return __builtin_bit_cast(sfenc::bf16x8, w);
}

__device__ __forceinline__ i32x8 join(const sfenc::u32x4& lo, const sfenc::u32x4& hi) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// One workgroup per tile of TL (encode_slim.h: 128-B K-steps), NS stage buffers, NS - 1 in flight; the
// pipeline, its waits and the epilogues are gemm_slim_kernel's. The scale bytes of the tile's rows
// lie in LDS as [group of four blocks][row] dwords, loaded for 4096 elements of K at a time.
template <typename TL, int EPI, int AUX, bool WIDE>
__global__ __launch_bounds__(TL::NT, TL::ST * TL::NS > 81920 ? (TL::NW + 3) / 4 : (TL::NW + 1) / 2) void gemm_f8_kernel(F8Args a) {
  using namespace sfenc;
  constexpr int MB = TL::MB, NB = TL::NB, KC = TL::KC, NS = TL::NS, NW = TL::NW, TN = TL::TN, TM = TL::TM, NT = TL::NT;
  constexpr int PW = TL::PW, PX = TL::PX, ROWS = TM + TN;
  static_assert(KC == 8 && NS >= 2 && NS <= 6 && NS != 5, "128-B rows");
  __shared__ __attribute__((aligned(1024))) char s0[TL::ST];
  __shared__ __attribute__((aligned(1024))) char s1[TL::ST];
  __shared__ __attribute__((aligned(1024))) char s2[NS > 2 ? TL::ST : 16];
  __shared__ __attribute__((aligned(1024))) char s3[NS > 3 ? TL::ST : 16];
  __shared__ __attribute__((aligned(1024))) char s4[NS > 4 ? TL::ST : 16];
  __shared__ __attribute__((aligned(1024))) char s5[NS > 5 ? TL::ST : 16];
  __shared__ __attribute__((aligned(16))) uint32_t s_sc[SG * ROWS];  // features first, then tokens
  __shared__ __attribute__((aligned(16))) float s_benc[TN];
  __shared__ __attribute__((aligned(16))) float s_thr[TN];

  const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = w / TL::WN, wn = w % TL::WN;
  const int total = a.tiles_m * a.tiles_n;
  const int b = blockIdx.x, per = total / 8, rem = total % 8, xcd = b % 8, loc = b / 8;
  const TilePos tp = tile_of(a, xcd * per + min(xcd, rem) + loc);
  const int64_t m0 = (int64_t)tp.m * TM, n0 = (int64_t)tp.n * TN;
  const int KT = a.ksteps, KB = KT * BLOCK;
  const int groups = (KT + 3) >> 2;

  uint32_t xo[PX], wo[PW];
#pragma unroll
  for (int i = 0; i < PX; ++i) {
    const int P = (i * NW + w) * 64 + lane, m = P / KC;
    xo[i] = (uint32_t)(m * a.Kp + ((P % KC) ^ slim_swz<KC>(m)) * 16);
  }
#pragma unroll
  for (int i = 0; i < PW; ++i) {
    const int P = (i * NW + w) * 64 + lane, n = P / KC;
    wo[i] = (uint32_t)(n * a.swn + ((P % KC) ^ slim_swz<KC>(n)) * 16);
  }
  // rows past M and N lie behind these ranges and read as zeros
  const int64_t xbytes = (min((int64_t)TM, a.M - m0) - 1) * a.Kp + KB;
  const int64_t wbytes = (min((int64_t)TN, a.N - n0) - 1) * a.swn + KB;
  auto issue = [&](int kt, char* st) {
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.xw + m0 * a.Kp, kt < KT ? xbytes : 0);
    const __amdgpu_buffer_rsrc_t wr = rsrc(a.w + n0 * a.swn, kt < KT ? wbytes : 0);
#pragma unroll
    for (int i = 0; i < PX; ++i) dma16(xr, st + TL::WT + (i * NW + w) * 1024, xo[i], (uint32_t)(kt * BLOCK));
#pragma unroll
    for (int i = 0; i < PW; ++i) dma16_w<AUX>(wr, st + (i * NW + w) * 1024, wo[i], (uint32_t)(kt * BLOCK));
  };
  // scale dwords of groups [g0, g0 + SG) of the tile's rows (the last valid row's past M and N, whose
  // codes are zeros), into registers and from there into LDS
  constexpr int PS = (SG * ROWS + NT - 1) / NT;
  uint32_t sc[PS];
  auto load_scales = [&](int g0) {
#pragma unroll
    for (int i = 0; i < PS; ++i) {
      const int at = i * NT + t, g = at / ROWS, r = at % ROWS;
      sc[i] = 0;
      if (g < SG && g0 + g < groups) {
        const uint8_t* src = r < TN ? a.ws + min(n0 + r, a.N - 1) * a.sws : a.xs + min(m0 + r - TN, a.M - 1) * a.sxs;
        sc[i] = *(const uint32_t*)(src + (g0 + g) * 4);
      }
    }
  };
  auto put_scales = [&] {
#pragma unroll
    for (int i = 0; i < PS; ++i)
      if (i * NT + t < SG * ROWS) s_sc[i * NT + t] = sc[i];
  };

  // loaded before the first stages, so that awaiting them does not await those
  const int64_t nb_ = min(n0 + t % TN, a.N - 1);
  const uint32_t rb = a.b_enc ? load_bits(a.b_enc, a.benc_dt, nb_) : 0u;
  const uint32_t rt = a.act == SF_ACT_JUMPRELU ? load_bits(a.thr, a.thr_dt, nb_) : 0u;
  load_scales(0);
  issue(0, s0);
  if constexpr (NS > 2) issue(1, s1);
  if constexpr (NS > 3) issue(2, s2);
  if constexpr (NS > 4) issue(3, s3);
  if constexpr (NS > 5) issue(4, s4);
  for (int i = t; i < TN; i += NT) {  // (TN <= NT, or each thread's one feature)
    const int64_t n = n0 + i;
    const float h = a.out_dt == SF_F32 ? 0.f : (a.out_dt == SF_BF16 ? 0x1p-126f : 0x1p-25f);
    float tv = a.act == SF_ACT_NONE ? __builtin_nanf("") : h;
    if (n >= a.N) {
      tv = __builtin_inff();
    } else if (a.act == SF_ACT_JUMPRELU) {
      const float th = bits_as_f32(rt, a.thr_dt);
      tv = th != th ? __builtin_inff() : fmaxf(th, h);
    }
    s_benc[i] = n < a.N ? bits_as_f32(rb, a.benc_dt) : 0.f;
    s_thr[i] = tv;
  }
  static_assert(TN <= NT, "a thread's bias");
  put_scales();
  wait_lgkmcnt0();
  barrier_no_fence();
  f32x16 acc[NB][MB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 be = *(const float4*)(s_benc + (wn * NB + nb) * 32 + g * 8 + (lane >> 5) * 4);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        acc[nb][mb][g * 4 + 0] = be.x;
        acc[nb][mb][g * 4 + 1] = be.y;
        acc[nb][mb][g * 4 + 2] = be.z;
        acc[nb][mb][g * 4 + 3] = be.w;
      }
    }

  struct Frag {
    i32x8 a[NB], b[MB];
  };
  // the 64 elements of half s: chunks 4s and 4s + 1 of the row, then 4s + 2 and 4s + 3, by lane half
  auto row_frag = [&](const char* tile, int row, int s) {
    const int z = slim_swz<KC>(row), c = 4 * s + (lane >> 5);
    return join(*(const sfenc::u32x4*)(tile + row * 128 + ((c ^ z) << 4)),
                *(const sfenc::u32x4*)(tile + row * 128 + (((c + 2) ^ z) << 4)));
  };
  auto load_frag = [&](Frag& f, const char* st, int s) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) f.b[mb] = row_frag(st + TL::WT, (wm * MB + mb) * 32 + (lane & 31), s);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) f.a[nb] = row_frag(st, (wn * NB + nb) * 32 + (lane & 31), s);
  };
  auto step = [&](int kt, char* cur, char* nxt) {
    wait_vm_lgkm0<(NS - 2) * (PW + PX)>();
    barrier_no_fence();
    if ((kt & (SG_STEPS - 1)) == 0 && kt) {  // every wave is done with the last groups' scales
      load_scales(kt >> 2);
      put_scales();
      wait_lgkmcnt0();
      barrier_no_fence();
    }
    issue(kt + NS - 1, nxt);
    const char* sb = (const char*)s_sc + ((kt >> 2) & (SG - 1)) * ROWS * 4 + (kt & 3);
    int sa[NB], sx[MB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) sa[nb] = *(const uint8_t*)(sb + ((wn * NB + nb) * 32 + (lane & 31)) * 4);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) sx[mb] = *(const uint8_t*)(sb + (TN + (wm * MB + mb) * 32 + (lane & 31)) * 4);
    Frag f[2];
    load_frag(f[0], cur, 0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s == 0) load_frag(f[1], cur, 1);
      if constexpr (WIDE) {
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          bf16x8 wa[NB], wb[MB];
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) wa[nb] = widen8(f[s].a[nb], part, scale_of(sa[nb]));
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) wb[mb] = widen8(f[s].b[mb], part, scale_of(sx[mb]));
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
              acc[nb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[nb], wb[mb], acc[nb][mb], 0, 0, 0);
        }
      } else {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) mfma_f8(acc[nb][mb], f[s].a[nb], f[s].b[mb], sa[nb], sx[mb]);
      }
    }
  };
  for (int kt = 0;;) {  // KT >= 1; the buffers rotate statically
    step(kt, s0, NS == 2 ? s1 : (NS == 3 ? s2 : (NS == 4 ? s3 : s5)));
    if (++kt >= KT) break;
    step(kt, s1, s0);
    if (++kt >= KT) break;
    if constexpr (NS > 2) {
      step(kt, s2, s1);
      if (++kt >= KT) break;
    }
    if constexpr (NS > 3) {
      step(kt, s3, s2);
      if (++kt >= KT) break;
    }
    if constexpr (NS > 4) {
      step(kt, s4, s3);
      if (++kt >= KT) break;
      step(kt, s5, s4);
      if (++kt >= KT) break;
    }
  }
  const int64_t mw = m0 + wm * MB * 32, nw = n0 + wn * NB * 32;
  const float* st = s_thr + wn * NB * 32;
  wait_vmcnt0();  // no DMA (the empty-range ones included) outlives its wave or hits the staging
  if constexpr (EPI != EPI_DENSE) {
    slim_rows<MB, NB>(a, acc, mw, nw, lane, st);
  } else {
    __syncthreads();
    constexpr int RG = 32 * NB * 32 * 4, WPS = TL::ST / RG;  // staging bytes per wave, waves per buffer
    static_assert(NW <= 2 * WPS, "epilogue staging");
    char* reg = w < WPS ? s0 + w * RG : s1 + (w - WPS) * RG;
    slim_dense<WIDE ? 4 : 2, MB, NB>(a, acc, mw, nw, lane, st, reg);  // (fp32 results are wide)
  }
}

}  // namespace sff8
