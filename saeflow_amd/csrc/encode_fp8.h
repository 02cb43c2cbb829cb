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
// (root mean square, d_in 768, normal operands; 9e-5 with one to four dimensions 300 to 3000 times the others), a
// fortieth of a bf16 rounding and a quarter (0.4) of an fp16 one. It is at most 7 * 2^-13 of sum |x w|, which is more of
// a result whose terms cancel. fp32 results are to be as good as fp32 sums: they take the wide
// form, where fragments become bf16 (exact down to 2^-133: four significant bits and a power of two) and the 16-bit
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
  // The fused form's tokens: x [M, K] of x_dt minus shift, quantised by each workgroup for itself.
  const void* x;
  int64_t sxm, sxk;
  int x_dt, x_rows;  // x_rows: rows contiguous and 16-B aligned
  const void* shift;
  int shift_dt, shift_vec;
  int stream;  // result rows begin on whole cache lines (Out)
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

// Feature (within a block of 32) that row i of a W fragment holds. Lane half h of an MFMA result has the
// rows 8 g + 4 h + r; with this order they are the consecutive features 16 h + 4 g + r, 32 B of a row.
__device__ __forceinline__ int frag_feature(int i) { return (i & 4) * 4 + (i >> 3) * 4 + (i & 3); }

// 16 B of a result row, at any element's address
typedef sfenc::u32x4 u32x4_any __attribute__((aligned(2)));

// What an epilogue writes to. stream: rows begin on whole cache lines, and stores go past the caches; lines that
// two stores share are put together in L2 instead.
// Either kind of store for all rows (us, d_in 120 / 768 / 2304): past the caches 197 / 334 / 722 against 204 / 464 / 836
// for 16000 tokens over 24576 features in bf16 with 256x256 tiles, 272 / 648 / 1428 against 350 / 712 / 1459 in fp32, but
// 57 / 82 / 137 against 42 / 66 / 122 for 4096 tokens over 12936 in bf16.
struct Out {
  char* out;
  int64_t som;
  int32_t* row_nnz;
  int64_t M, N;
  int act, stream;
};
// (the empty asm keeps the compiler from making one ordinary store of the two)
__device__ __forceinline__ void put16(const sfenc::u32x4& v, char* dst, int stream) {
  if (stream) {
    asm volatile("");
    __builtin_nontemporal_store(v, (u32x4_any*)dst);
    asm volatile("");
  } else {
    *(u32x4_any*)dst = v;
  }
}
// Epilogue of a wave's (32 MB x 32 NB) tile at token m0, feature n0, 32 tokens at a time through `reg` (32
// rows of 32 NB features, this wave's own), fragment rows in frag_feature order: 16-B stores at any
// alignment, element by element only across the last feature. ES: bytes of a result.
template <int ES, int MB, int NB, bool PLAIN>
__device__ __forceinline__ void tile_epilogue(const Out& a, int out_dt, f32x16 (&acc)[NB][MB], int64_t m0, int64_t n0,
                                              int lane, const float* s_t, char* reg) {
  using namespace sfenc;
  constexpr int RB = NB * 32 * ES, UPR = RB / 16, RPI = 64 / UPR, EPU = 16 / ES;
  float lo = a.act == SF_ACT_NONE ? -__builtin_inff() : 0.f;
  asm volatile("" : "+v"(lo));
  const int h = lane >> 5, rl = lane & 31, unit = lane % UPR;
  const int rows = (int)max((int64_t)0, min((int64_t)32 * MB, a.M - m0));
  const int cols = (int)max((int64_t)0, min((int64_t)32 * NB, a.N - n0));
  char* dst = a.out + ((m0 + lane / UPR) * a.som + n0 + unit * EPU) * ES;
  const int64_t step = (int64_t)RPI * a.som * ES;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    int cnt = 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int g = 0; g < 16 / EPU; ++g) {
        const int cl = nb * 32 + h * 16 + g * EPU;
        float o[EPU];
#pragma unroll
        for (int e = 0; e < EPU; ++e) {
          const float pre = acc[nb][mb][g * EPU + e];
          if constexpr (PLAIN) {
            o[e] = __builtin_elementwise_maximum(pre, lo);
          } else {
            const bool keep = !(pre <= s_t[cl + e]);
            o[e] = keep ? pre : 0.f;
            cnt += keep && cl + e < cols ? 1 : 0;
          }
        }
        sfenc::u32x4 v;
        if constexpr (ES == 4)
          v = sfenc::u32x4{__float_as_uint(o[0]), __float_as_uint(o[1]), __float_as_uint(o[2]), __float_as_uint(o[3])};
        else if (out_dt == SF_F16)
          v = sfenc::u32x4{pack2<SF_F16>(o[0], o[1]), pack2<SF_F16>(o[2], o[3]), pack2<SF_F16>(o[4], o[5]), pack2<SF_F16>(o[6], o[7])};
        else
          v = sfenc::u32x4{pack2<SF_BF16>(o[0], o[1]), pack2<SF_BF16>(o[2], o[3]), pack2<SF_BF16>(o[4], o[5]), pack2<SF_BF16>(o[6], o[7])};
        *(sfenc::u32x4*)(reg + rl * RB + (((cl / EPU) ^ (rl & (UPR - 1))) << 4)) = v;
      }
    }
    if constexpr (!PLAIN) {
      if (a.row_nnz) {
        const int c = cnt + __shfl_xor(cnt, 32);
        if (lane < 32 && mb * 32 + lane < rows && c > 0) atomicAdd(a.row_nnz + m0 + mb * 32 + lane, c);
      }
    }
    __builtin_amdgcn_wave_barrier();  // the staged rows are this wave's own (in-order LDS)
#pragma unroll
    for (int it = 0; it < 32 / RPI; ++it) {
      const int row = it * RPI + lane / UPR;
      const sfenc::u32x4 v = *(const sfenc::u32x4*)(reg + row * RB + ((unit ^ (row & (UPR - 1))) << 4));
      if (mb * 32 + row < rows) {
        if (unit * EPU + EPU <= cols) {
          put16(v, dst, a.stream);
        } else {
#pragma unroll
          for (int e = 0; e < EPU; ++e)
            if (unit * EPU + e < cols) {
              if constexpr (ES == 4) ((uint32_t*)dst)[e] = v[e];
              else ((u16*)dst)[e] = (u16)(v[e >> 1] >> ((e & 1) * 16));
            }
        }
      }
      dst += step;
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// One workgroup per tile of TL (encode_slim.h: 128-B K-steps), NS stage buffers, NS - 1 in flight; the
// pipeline and its waits are gemm_slim_kernel's. The scale bytes of the tile's rows lie in LDS as [group of
// four blocks][row] dwords, loaded for 4096 elements of K at a time.
//
// Bound by the pass over W where tokens are few (32 tokens over 65536 features of d_in 2304, bf16: 25 us, 6.2
// TB/s), by the latency of a K-step where tiles are one round, by that and LDS where they are many (128x128:
// eight waves of 32x64 read 96 KB a K-step, 768 cycles of LDS and 512 of the matrix cores; 4096 tokens 626 us,
// 1.98 PFLOP/s).
//
// FUSED (tokens of at most FUSED_BLOCKS blocks in all): the tokens come as they are; each workgroup, its
// first stages of W under way, quantises all of them into LDS, where they stay, and a launch is saved.
constexpr int FUSED_BLOCKS = 32;
template <typename TL, bool WIDE, bool PLAIN, bool FUSED>
__global__ __launch_bounds__(TL::NT, TL::ST * TL::NS > 81920 ? (TL::NW + 3) / 4 : (TL::NW + 1) / 2) void gemm_f8_kernel(F8Args a) {
  using namespace sfenc;
  constexpr int MB = TL::MB, NB = TL::NB, KC = TL::KC, NS = TL::NS, NW = TL::NW, TN = TL::TN, TM = TL::TM, NT = TL::NT;
  constexpr int PW = TL::PW, PX = FUSED ? 0 : TL::PX, ROWS = FUSED ? TN : TM + TN;
  constexpr int ST = FUSED ? TL::WT : TL::ST;
  static_assert(!FUSED || (TM == 32 && TL::WM == 1), "one block of tokens");
  static_assert(KC == 8 && NS >= 2 && NS <= 6 && NS != 5, "128-B rows");
  __shared__ __attribute__((aligned(1024))) char s0[ST];
  __shared__ __attribute__((aligned(1024))) char s1[ST];
  __shared__ __attribute__((aligned(1024))) char s2[NS > 2 ? ST : 16];
  __shared__ __attribute__((aligned(1024))) char s3[NS > 3 ? ST : 16];
  __shared__ __attribute__((aligned(1024))) char s4[NS > 4 ? ST : 16];
  __shared__ __attribute__((aligned(1024))) char s5[NS > 5 ? ST : 16];
  __shared__ __attribute__((aligned(16))) uint32_t s_sc[SG * ROWS];  // features first, then tokens
  __shared__ __attribute__((aligned(16))) char s_x[FUSED ? FUSED_BLOCKS * BLOCK : 16];  // codes [token][block]
  __shared__ __attribute__((aligned(16))) uint8_t s_xsc[FUSED ? FUSED_BLOCKS : 16];  // their scales
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

  uint32_t xo[FUSED ? 1 : PX], wo[PW];
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
    for (int i = 0; i < PW; ++i) dma16(wr, st + (i * NW + w) * 1024, wo[i], (uint32_t)(kt * BLOCK));
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
  // FUSED: the raw bits of a thread's tokens and their shift, loaded before the stages of W (loads return in
  // order: behind them they would arrive when all of those have), where they are whole 16-B units
  constexpr int Q = NT / 16, XI = FUSED ? FUSED_BLOCKS / Q : 1;  // blocks taken at a time, and per sixteen lanes
  sff8::u32x4 xraw[XI][2], craw[XI][2];
  const int all = (int)min((int64_t)FUSED_BLOCKS, a.M * KT);  // blocks there are
  const bool raw = FUSED && a.x_rows && a.K % 8 == 0 && (!a.shift || a.shift_vec);
  if constexpr (FUSED) {
#pragma unroll
    for (int i = 0; i < XI; ++i) {
      xraw[i][0] = xraw[i][1] = craw[i][0] = craw[i][1] = sff8::u32x4{0, 0, 0, 0};
      const int b = min((t >> 4) + i * Q, all - 1), m = b / KT;
      const int64_t k0 = (int64_t)(b - m * KT) * BLOCK + (t & 15) * 8;
      if (raw && k0 < a.K) {
        const int E = sf_dtype_size(a.x_dt);
        const char* px = (const char*)a.x + (m * a.sxm + k0) * E;
        const char* pc = (const char*)a.shift + k0 * E;
        xraw[i][0] = *(const sff8::u32x4*)px;
        if (E == 4) xraw[i][1] = *(const sff8::u32x4*)(px + 16);
        if (a.shift) craw[i][0] = *(const sff8::u32x4*)pc;
        if (a.shift && E == 4) craw[i][1] = *(const sff8::u32x4*)(pc + 16);
      }
    }
  }
  load_scales(0);
  issue(0, s0);
  if constexpr (NS > 2) issue(1, s1);
  if constexpr (NS > 3) issue(2, s2);
  if constexpr (NS > 4) issue(3, s3);
  if constexpr (NS > 5) issue(4, s4);
  for (int i = t; i < TN; i += NT) {  // (TN <= NT, or each thread's one feature)
    const int64_t n = n0 + i;
    // keep-threshold: the largest value that rounds to zero in the result's type (subnormals of bf16 are kept, as
    // PLAIN keeps them), or the feature's own
    const float h = a.out_dt == SF_F32 ? 0.f : (a.out_dt == SF_BF16 ? 0x1p-134f : 0x1p-25f);
    float tv = h;
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
  if constexpr (FUSED) {
    auto put = [&](int i, float (&v)[8]) {
      const int b = min((t >> 4) + i * Q, all - 1);
      uint32_t byte;
      *(sff8::u32x2*)(s_x + b * BLOCK + (t & 15) * 8) = quantize8(v, byte);
      if ((t & 15) == 0) s_xsc[b] = (uint8_t)byte;
    };
    if (raw) {
#pragma unroll
      for (int i = 0; i < XI; ++i) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (a.x_dt == SF_F32) {
            v[e] = __uint_as_float(xraw[i][e >> 2][e & 3]) - __uint_as_float(craw[i][e >> 2][e & 3]);
          } else {
            const int at = (e & 1) * 16;
            v[e] = bits_as_f32((xraw[i][0][e >> 1] >> at) & 0xffffu, a.x_dt) -
                   bits_as_f32((craw[i][0][e >> 1] >> at) & 0xffffu, a.x_dt);
          }
        }
        put(i, v);
      }
    } else {
      for (int i = 0; i < XI; ++i) {
        const int b = min((t >> 4) + i * Q, all - 1), m = b / KT;
        const int64_t k0 = (int64_t)(b - m * KT) * BLOCK + (t & 15) * 8;
        float v[8];
        if (a.x_dt == SF_BF16) load_shifted<SF_BF16, SRC_ANY>(a.x, a.sxm, a.sxk, a.shift, a.shift_dt, 0, a.K, m, k0, v);
        else if (a.x_dt == SF_F16) load_shifted<SF_F16, SRC_ANY>(a.x, a.sxm, a.sxk, a.shift, a.shift_dt, 0, a.K, m, k0, v);
        else load_shifted<SF_F32, SRC_ANY>(a.x, a.sxm, a.sxk, a.shift, a.shift_dt, 0, a.K, m, k0, v);
        put(i, v);
      }
    }
  }
  wait_lgkmcnt0();
  barrier_no_fence();
  f32x16 acc[NB][MB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 be = *(const float4*)(s_benc + (wn * NB + nb) * 32 + (lane >> 5) * 16 + g * 4);
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
  auto load_frag = [&](Frag& f, const char* st, int s, int kt) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
      if constexpr (FUSED) {
        const char* row = s_x + (min(lane & 31, (int)a.M - 1) * KT + kt) * BLOCK;
        const int c = 4 * s + (lane >> 5);
        f.b[mb] = join(*(const sfenc::u32x4*)(row + (c << 4)), *(const sfenc::u32x4*)(row + ((c + 2) << 4)));
      } else {
        f.b[mb] = row_frag(st + TL::WT, (wm * MB + mb) * 32 + (lane & 31), s);
      }
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) f.a[nb] = row_frag(st, (wn * NB + nb) * 32 + frag_feature(lane & 31), s);
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
    for (int nb = 0; nb < NB; ++nb) sa[nb] = *(const uint8_t*)(sb + ((wn * NB + nb) * 32 + frag_feature(lane & 31)) * 4);
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
      sx[mb] = FUSED ? s_xsc[min(lane & 31, (int)a.M - 1) * KT + kt]
                     : *(const uint8_t*)(sb + (TN + (wm * MB + mb) * 32 + (lane & 31)) * 4);
    Frag f[2];
    load_frag(f[0], cur, 0, kt);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      if (s == 0) load_frag(f[1], cur, 1, kt);
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
  __syncthreads();
  constexpr int ES = WIDE ? 4 : 2;  // (fp32 results are wide)
  constexpr int RG = 32 * NB * 32 * ES, WPS = ST / RG;  // staging bytes per wave, waves per buffer
  static_assert(NW <= 2 * WPS, "epilogue staging");
  char* reg = w < WPS ? s0 + w * RG : s1 + (w - WPS) * RG;
  tile_epilogue<ES, MB, NB, PLAIN>(Out{(char*)a.out, a.som, a.row_nnz, a.M, a.N, a.act, a.stream}, a.out_dt, acc, mw, nw, lane, st, reg);
}


// dword of a scale row to LDS at wave_base + 4 * lane
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t r, char* wave_base, uint32_t voff, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)wave_base, 4, (int)voff, (int)soff, 0, 0);
}

// Three bf16 pieces of a fp32 value, whose sum it is (8 significant bits each, cut off, so that none passes the
// value; a lone first piece for infinities and NaN; what lies below bf16's smallest subnormal 2^-133 is lost, which
// concerns values below 2^-109), as two dwords.
__device__ __forceinline__ sfenc::u32x2 pieces(float v) {
  const uint32_t u = __float_as_uint(v);
  const bool fine = fabsf(v) < __builtin_inff();
  const float r = v - __uint_as_float(u & 0xffff0000u);
  const uint32_t p1 = __float_as_uint(r) & 0xffff0000u, p2 = __float_as_uint(r - __uint_as_float(p1)) >> 16;
  return sfenc::u32x2{fine ? u >> 16 | p1 : f32_to_bf16(v), fine ? p2 : 0u};
}

// Epilogue of a wave's 128x128 tile of 16-bit results at token m0, feature n0, through 16 KiB of LDS, two
// passes of 64 tokens; fragment rows in frag_feature order. PLAIN: relu or none and no counts, one
// instruction an element (gfx950's v_maximum3_f32 keeps a NaN) before the conversion; otherwise as
// sfenc::epilogue, with the thresholds s_t. RAGGED: the tile reaches past M or N.
template <int ODT, bool PLAIN, bool RAGGED>
__device__ __forceinline__ void f8_epilogue(const Out& a, f32x16 (&acc)[4][4], int64_t m0, int64_t n0, int lane,
                                            const float* s_t, char* reg) {
  using namespace sfenc;
  float lo = a.act == SF_ACT_NONE ? -__builtin_inff() : 0.f;
  asm volatile("" : "+v"(lo));  // (opaque: else a maximum with 0 and a select)
  const int h = lane >> 5, unit = lane & 15;
  const int rows = RAGGED ? (int)max((int64_t)0, min((int64_t)128, a.M - m0)) : 128;
  const int cols = RAGGED ? (int)max((int64_t)0, min((int64_t)128, a.N - n0)) : 128;
  // (opaque, so that no multiples of it are formed ahead of the tile loop and spilled)
  int64_t som = a.som;
  asm volatile("" : "+s"(som));
  char* dst = (char*)a.out + ((m0 + lane / 16) * som + n0 + unit * 8) * 2;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    int cnt[2] = {0, 0};
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // eight consecutive features
        const int cl = nb * 32 + h * 16 + half * 8;
        float thv[8];
        if constexpr (!PLAIN) {
          const float4 ta = *(const float4*)(s_t + cl), tb = *(const float4*)(s_t + cl + 4);
          thv[0] = ta.x; thv[1] = ta.y; thv[2] = ta.z; thv[3] = ta.w;
          thv[4] = tb.x; thv[5] = tb.y; thv[6] = tb.z; thv[7] = tb.w;
        }
#pragma unroll
        for (int mi = 0; mi < 2; ++mi) {
          const int rl = mi * 32 + (lane & 31);
          float o[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float pre = acc[nb][pass * 2 + mi][half * 8 + e];
            if constexpr (PLAIN) {
              o[e] = __builtin_elementwise_maximum(pre, lo);
            } else {
              const bool keep = !(pre <= thv[e]);
              o[e] = keep ? pre : 0.f;
              cnt[mi] += keep && (!RAGGED || cl + e < cols) ? 1 : 0;
            }
          }
          if constexpr (!PLAIN) asm volatile("" : "+v"(cnt[mi]));  // keep the count from sinking
          *(sfenc::u32x4*)(reg + rl * 256 + (((cl >> 3) ^ (rl & 15)) << 4)) =
              sfenc::u32x4{pack2<ODT>(o[0], o[1]), pack2<ODT>(o[2], o[3]), pack2<ODT>(o[4], o[5]), pack2<ODT>(o[6], o[7])};
        }
        __builtin_amdgcn_sched_barrier(0);  // (bounds what the compiler holds in registers at once)
      }
    }
    if constexpr (!PLAIN) {
      if (a.row_nnz) {
#pragma unroll
        for (int mi = 0; mi < 2; ++mi) {
          const int c = cnt[mi] + __shfl_xor(cnt[mi], 32), r = (pass * 2 + mi) * 32 + lane;
          if (lane < 32 && c > 0 && (!RAGGED || r < rows)) atomicAdd(a.row_nnz + m0 + r, c);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();  // the staged rows are this wave's own (in-order LDS)
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      sfenc::u32x4 v[8];
#pragma unroll
      for (int it = 0; it < 8; ++it) {
        const int rl = (part * 8 + it) * 4 + lane / 16;
        v[it] = *(const sfenc::u32x4*)(reg + rl * 256 + ((unit ^ (rl & 15)) << 4));
      }
      auto store = [&](auto put) {
#pragma unroll
        for (int it = 0; it < 8; ++it) {
          const int rl = pass * 64 + (part * 8 + it) * 4;
          if (!RAGGED || (rl + lane / 16 < rows && unit * 8 + 8 <= cols)) {
            put(v[it], (u32x4_any*)dst);
          } else if (rl + lane / 16 < rows) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (unit * 8 + e < cols) ((u16*)dst)[e] = (u16)(v[it][e >> 1] >> ((e & 1) * 16));
          }
          dst += 8 * som;
        }
      };
      if (a.stream) {  // (as put16)
        asm volatile("");
        store([](const sfenc::u32x4& x, u32x4_any* d) { __builtin_nontemporal_store(x, d); });
        asm volatile("");
      } else {
        store([](const sfenc::u32x4& x, u32x4_any* d) { *d = x; });
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// Persistent form for 256x256 tiles: gemm_persist_kernel's walk of an XCD's tiles, its claims, its alternating stage buffers
// and its epilogue, four waves of 128x128 (one per SIMD; eight waves of 128x64 would need the registers of
// both halves' fragments twice), with a K loop of its own:
//   Y(kt)      16 MFMAs on the first half (64 elements) of block kt, the second half's fragments read
//              under the first of them. After 12 the wave has read all it needs of kt's buffer and
//              meets the others: past that barrier block kt + 1 has landed and kt's buffer is free, so the
//              DMAs of block kt + 2 go into it at once, a whole K-step before they are awaited.
//   X(kt + 1)  16 MFMAs on the second half of kt, the first half of kt + 1 read under them.
// The order of MFMAs, LDS reads and DMAs is pinned (a scheduling barrier after each MFMA): left to itself
// the compiler puts all reads of a half before its first MFMA (16384 x 2304 x 65536, bf16 results: 1.67
// PFLOP/s so, 2.58 pinned, 1920 us). Bound there by the power limit: the matrix cores are busy 66% of 1.78 GHz,
// waves wait 15% of their time, no LDS bank conflicts; fp32 results (the wide form) take 2.0 times as long,
// bound by the 16-bit instruction. Thresholds and counts (PLAIN false) spill 312 scalar registers (fp32 1305) and one
// vector register at tile ends: JumpReLU 2052 us, with counts 2096, ReLU with counts 2056, where ReLU alone takes 1940 to
// 2008. An odd number of blocks is rounded
// up; the one past the end reads zeros.
template <int ODT, bool PLAIN>
__global__ __launch_bounds__(256, 1) void gemm_f8_persist_kernel(F8Args a) {
  using namespace sfenc;
  constexpr int NW = 4, NB = 4, MB = 4, NMF = NB * MB;
  constexpr bool WIDE = ODT == SF_F32;
  constexpr int NST = WIDE ? 63 : 32;     // the epilogue's stores per lane (64 of fp32; vmcnt counts to 63)
  constexpr int PER = 32 / NW;            // DMAs a wave issues per operand and K-step
  // Y's schedule: two reads after each of the first YD MFMAs and one after the others, the barrier after
  // MFMA YB, one DMA an MFMA from there on
  constexpr int YD = 4, YB = 13;
  __shared__ __attribute__((aligned(1024))) char lds0[STAGE];
  __shared__ __attribute__((aligned(1024))) char lds1[STAGE];
  __shared__ __attribute__((aligned(1024))) char s_sc[2][2048];  // dwords of four blocks: features, then tokens
  __shared__ __attribute__((aligned(16))) float s_bias[2][BN];
  __shared__ __attribute__((aligned(16))) float s_thr[2][BN];
  __shared__ int s_claim;

  // The arguments that only a tile's ends need, read again from the kernel's argument block there: held in
  // scalar registers throughout, they spill into vector registers, and those into memory, whose loads then
  // wait for the tile's stores.
  auto cold = [] {
    const __attribute__((address_space(4))) F8Args* p =
        (const __attribute__((address_space(4))) F8Args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
  };
  // The thread's index, formed anew (and opaquely) where it is used, so that it and what derives from it
  // take no registers in between.
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto thread = [&] {
    int zero = 0;
    asm volatile("" : "+s"(zero));
    return w * 64 + __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
  };
  const int total = a.tiles_m * a.tiles_n;
  const int b = blockIdx.x;
  const int per = total / 8, rem = total % 8, xcd = b % 8, loc = b / 8;
  const int first = xcd * per + min(xcd, rem), last = first + per + (xcd < rem ? 1 : 0);
  const int step = gridDim.x / 8;  // workgroups per XCD: the fixed first tiles
  int32_t* const ctr = a.tile_ctr + xcd * TILE_CTR_STRIDE;
  int lid = first + loc;
  if (lid >= last) return;  // the whole workgroup
  const int KB = a.ksteps, KT = (KB + 1) & ~1;

  // A tile. Its DMAs fill LDS rows (i * NW + w) * 8 + lane / 8; rows past M or N are the last valid one again
  // (rm, rn).
  struct Tile {
    int64_t m0, n0;
    int rm, rn;
  };
  auto open_tile = [&](int lid) {
    const auto c = cold();
    // runs of group_n feature panels, token panel by token panel (tile_of)
    const int g = c->group_n, per_group = g * c->tiles_m;
    const int first = lid / per_group * g, at = lid % per_group, gs = min(c->tiles_n - first, g);
    Tile T;
    T.m0 = (int64_t)(at / gs) * BM;
    T.n0 = (int64_t)(first + at % gs) * BN;
    T.rm = (int)min((int64_t)BM, c->M - T.m0) - 1;
    T.rn = (int)min((int64_t)BN, c->N - T.n0) - 1;
    return T;
  };
  // Bias and keep-threshold (as gemm_f8_kernel forms it) of feature t of a tile: raw bits, loaded while the
  // tile before ends, and their values in LDS, read past the tile's first barrier.
  struct Raw {
    uint32_t bias, thr;
  };
  auto load_raw = [&](const Tile& T, int t) {
    const auto c = cold();
    const int64_t n = T.n0 + min(t, T.rn);
    Raw r;
    r.bias = c->b_enc ? load_bits(c->b_enc, c->benc_dt, n) : 0u;
    r.thr = !PLAIN && c->act == SF_ACT_JUMPRELU ? load_bits(c->thr, c->thr_dt, n) : 0u;
    return r;
  };
  auto put_raw = [&](const Tile& T, const Raw& r, int slot, int t) {
    const auto c = cold();
    s_bias[slot][t] = bits_as_f32(r.bias, c->benc_dt);
    if constexpr (!PLAIN) {
      constexpr float h = ODT == SF_F32 ? 0.f : (ODT == SF_BF16 ? 0x1p-134f : 0x1p-25f);
      float tv = h;
      if (t > T.rn) {
        tv = __builtin_inff();
      } else if (c->act == SF_ACT_JUMPRELU) {
        const float th = bits_as_f32(r.thr, c->thr_dt);
        tv = th != th ? __builtin_inff() : fmaxf(th, h);
      }
      s_thr[slot][t] = tv;
    }
  };
  // A lane's offsets of its DMAs of a K-step, within the tile's rows.
  struct Offsets {
    uint32_t x[PER], w[PER];
  };
  auto offsets_of = [&](const Tile& T, int t) {
    Offsets o;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int row = ((t >> 3) & 31) + i * 32;
      const uint32_t c = (((t & 7) ^ ((t >> 3) & 7) ^ (i & 1) * 4 ^ ((t >> 6) & 3)) & 7) * 16;  // swz(row)
      o.x[i] = (uint32_t)(min(row, T.rm) & 255) * ((uint32_t)a.Kp & 0xffffffu) + c;
      o.w[i] = (uint32_t)(min(row, T.rn) & 255) * ((uint32_t)a.swn & 0xffffffu) + c;
    }
    return o;
  };
  // DMAs [q0, q1) of a K-step's 2 PER, x' and W in turn
  auto stage = [&](const Tile& T, const Offsets& o, int kt, char* buf, int q0, int q1) {
    const __amdgpu_buffer_rsrc_t xr = rsrc(a.xw + T.m0 * a.Kp, kt < KB ? T.rm * a.Kp + (int64_t)KB * BLOCK : 0);
    const __amdgpu_buffer_rsrc_t wr = rsrc(a.w + T.n0 * a.swn, kt < KB ? T.rn * a.swn + (int64_t)KB * BLOCK : 0);
#pragma unroll
    for (int q = 0; q < 2 * PER; ++q) {
      if (q < q0 || q >= q1) continue;
      const int i = q >> 1;
      if (q & 1) dma16(wr, buf + (i * NW + w) * 1024, o.w[i], (uint32_t)(kt * BLOCK));
      else dma16(xr, buf + TILE + (i * NW + w) * 1024, o.x[i], (uint32_t)(kt * BLOCK));
    }
  };
  auto stage_scales = [&](const Tile& T, int g, int w, int t) {
    dma4(rsrc(a.ws + T.n0 * a.sws, 256 * a.sws), s_sc[g & 1] + w * 256,
         (uint32_t)(min(t, T.rn) & 255) * ((uint32_t)a.sws & 0xffffffu), (uint32_t)(g * 4));
    dma4(rsrc(a.xs + T.m0 * a.sxs, 256 * a.sxs), s_sc[g & 1] + 1024 + w * 256,
         (uint32_t)(min(t, T.rm) & 255) * ((uint32_t)a.sxs & 0xffffffu), (uint32_t)(g * 4));
  };

  Tile T = open_tile(lid);
  {
    const int t0 = thread();
    const Raw r = load_raw(T, t0);
    stage(T, offsets_of(T, t0), 0, lds0, 0, 2 * PER);
    stage_scales(T, 0, w, t0);
    put_raw(T, r, 0, t0);
    wait_vmcnt0();
  }

  auto tile = [&](auto par_tag) -> bool {
    constexpr int P = decltype(par_tag)::value;
    char* const B0 = P ? lds1 : lds0;
    char* const B1 = P ? lds0 : lds1;
    int t = thread(), lane = t & 63;
    const int wm = w >> 1, wn = w & 1;
    // past this barrier block 0 and its scales have landed, and B1 is no longer staging space
    wait_lgkmcnt0();
    barrier_no_fence();
    const Offsets off = offsets_of(T, t);
    stage(T, off, 1, B1, 0, 2 * PER);
    // The accumulators start at b_enc: one bf16 MFMA each, of the bias in three exact pieces with ones (a
    // quarter of the time that writing 256 registers takes).
    f32x16 acc[NB][MB];
    {
      uint32_t one2 = 0x3f803f80u, one1 = 0x3f80u, none = 0;  // (opaque: not kept across tiles)
      asm volatile("" : "+v"(one2), "+v"(one1), "+v"(none));
      const bf16x8 ones = __builtin_bit_cast(bf16x8, sfenc::u32x4{one2, one1, none, none});
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const sfenc::u32x2 p = pieces(lane < 32 ? s_bias[P][wn * 128 + nb * 32 + frag_feature(lane)] : 0.f);
        const bf16x8 pb = __builtin_bit_cast(bf16x8, sfenc::u32x4{p[0], p[1], none, none});
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          acc[nb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pb, ones, f32x16{}, 0, 0, 0);
          asm volatile("" : "+a"(acc[nb][mb]));  // (four MFMAs, not one and copies)
        }
      }
    }
    if (t == 0) s_claim = a.tile_ctr ? atomicAdd(ctr, 1) : 1 << 28;  // visible past the next barrier

    struct Frag {
      sfenc::u32x4 lo[8], hi[8];  // x' fragments 0 to 3, W fragments 4 to 7
    };
    // Where a lane reads: chunk 4 s + 2 j + lane / 32 of row r of block q of the wave's rows (r: lane % 32
    // of x', frag_feature of it of W). swz of row 32 q + r is swz(r), with bit 2 flipped where q is odd, so s and q only decide bit 6 of the
    // offset: four offsets per operand, which the compiler is kept from working out anew per read.
    int at_x[2][2], at_w[2][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int rx = lane & 31, rw = frag_feature(rx), c = 2 * j + (lane >> 5);
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        at_x[j][p] = TILE + (wm * 128 + rx) * ROWB + (((c ^ swz(rx)) << 4) ^ (p * 64));
        at_w[j][p] = (wn * 128 + rw) * ROWB + (((c ^ swz(rw)) << 4) ^ (p * 64));
        asm volatile("" : "+v"(at_x[j][p]), "+v"(at_w[j][p]));
      }
    }
    // LDS read i of a half's 16, in the order in which the MFMAs want them
    auto read = [&](Frag& f, const char* cur, int s, int i) {
      constexpr int order[8] = {0, 4, 1, 2, 3, 5, 6, 7};
      const int q = order[i >> 1], p = (s ^ q) & 1;
      const char* at = cur + (q < 4 ? at_x : at_w)[i & 1][p] + (q & 3) * 32 * ROWB;
      if (i & 1) f.hi[q] = *(const sfenc::u32x4*)at;
      else f.lo[q] = *(const sfenc::u32x4*)at;
    };
    int sc[8], scn[8];  // scale bytes of the block in use and of the next
    auto read_scales = [&](int (&v)[8], int kt) {
      const char* sb = s_sc[(kt >> 2) & 1] + (kt & 3);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = *(const uint8_t*)(sb + (256 + wm * 128 + q * 32 + (lane & 31)) * 4);
        v[4 + q] = *(const uint8_t*)(sb + (wn * 128 + q * 32 + frag_feature(lane & 31)) * 4);
      }
    };
    auto mma = [&](const Frag& f, int i) {
      const int nb = i >> 2, mb = i & 3;
      mfma_f8(acc[nb][mb], join(f.lo[4 + nb], f.hi[4 + nb]), join(f.lo[mb], f.hi[mb]), sc[4 + nb], sc[mb]);
      asm volatile("" : "+a"(acc[nb][mb]));  // keeps the MFMA in its place among the memory operations
    };
    Frag F0, F1;
    // DMA: block kt + 2 goes into cur
    auto phase_y = [&](auto dma_tag, char* cur, int kt) {
      constexpr bool DMA = decltype(dma_tag)::value;
#pragma unroll
      for (int i = 0; i < NMF; ++i) {
        mma(F0, i);
        if (i < YD) {
          read(F1, cur, 1, 2 * i);
          read(F1, cur, 1, 2 * i + 1);
        } else if (i < 16 - YD) {
          read(F1, cur, 1, YD + i);
        }
        if (i == YB) {
          wait_vm_lgkm0<0>();
          barrier_no_fence();
          read_scales(scn, kt + 1);
        }
        if (DMA && i > YB) stage(T, off, kt + 2, cur, i - YB - 1, i - YB);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    auto phase_x = [&](auto dma_tag, const char* nxt, char* cur, int kt) {  // kt: the block just left (cur)
      constexpr bool DMA = decltype(dma_tag)::value;
#pragma unroll
      for (int i = 0; i < NMF; ++i) {
        mma(F1, i);
        read(F0, nxt, 0, i);
        if (DMA) stage(T, off, kt + 2, cur, 15 - YB + i, 16 - YB + i);
        __builtin_amdgcn_sched_barrier(0);
      }
      if (DMA && ((kt + 2) & 3) == 0) stage_scales(T, (kt + 2) >> 2, w, thread());
#pragma unroll
      for (int q = 0; q < 8; ++q) sc[q] = scn[q];
    };
    // The wide form of both phases: four parts of 16 bf16 MFMAs each. b: this part's and the next part's x'
    // fragments, a: this group of four MFMAs' W fragment and the next's, widened one dword each an
    // MFMA ahead of their use; the last part prepares the next phase's first (its fragments g, scales gs).
    // Reads, barrier and DMAs lie where they lie among a quarter as many MFMAs in the narrow form.
    bf16x8 wb[2][MB], wa[2];
    auto widen = [&](const Frag& f, const int (&s)[8], int q, int part) {
      return widen8(join(f.lo[q], f.hi[q]), part, scale_of(s[q]));
    };
    auto phase_wide = [&](auto y_tag, auto dma_tag, const Frag& f, const int (&fs)[8], Frag& g, const int (&gs)[8],
                          char* cur, const char* nxt, int kt) {
      constexpr bool Y = decltype(y_tag)::value, DMA = decltype(dma_tag)::value;
#pragma unroll
      for (int part = 0; part < 4; ++part) {
#pragma unroll
        for (int i = 0; i < NMF; ++i) {
          const int j = part * NMF + i, nb = i >> 2, mb = i & 3;
          acc[nb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[nb & 1], wb[part & 1][mb], acc[nb][mb], 0, 0, 0);
          asm volatile("" : "+a"(acc[nb][mb]));
          if (j % 2 == 0 && j < 32) {
            if constexpr (Y) read(g, cur, 1, j / 2);
            else read(g, nxt, 0, j / 2);
          }
          if (Y && j == 4 * YB) {
            wait_vm_lgkm0<0>();
            barrier_no_fence();
            read_scales(scn, kt + 1);
          }
          if constexpr (DMA) {
            const int e = j / 4;
            if (j % 4 == 2 && (!Y || e > YB)) {
              if constexpr (Y) stage(T, off, kt + 2, cur, e - YB - 1, e - YB);
              else stage(T, off, kt + 2, cur, 15 - YB + e, 16 - YB + e);
            }
          }
          if (mb == 2) {
            // the next group's W fragment, and one of the next part's x' fragments
            const int na = (nb + 1) & 3, pa = nb == 3 ? part + 1 : part;
            if (pa < 4) wa[(nb + 1) & 1] = widen(f, fs, 4 + na, pa);
            else wa[(nb + 1) & 1] = widen(g, gs, 4 + na, 0);
          }
          if (mb == 0) {
            if (part < 3) wb[(part + 1) & 1][nb] = widen(f, fs, nb, part + 1);
            else wb[(part + 1) & 1][nb] = widen(g, gs, nb, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };
    // K-step kt from its first half on: Y, then (more than one K-step left) X into kt + 1
    auto wide_y = [&](auto dma_tag, char* cur, int kt) { phase_wide(std::true_type{}, dma_tag, F0, sc, F1, sc, cur, nullptr, kt); };
    auto wide_x = [&](auto dma_tag, const char* nxt, char* cur, int kt) {
      phase_wide(std::false_type{}, dma_tag, F1, sc, F0, scn, cur, nxt, kt);
      if (decltype(dma_tag)::value && ((kt + 2) & 3) == 0) stage_scales(T, (kt + 2) >> 2, w, thread());
#pragma unroll
      for (int q = 0; q < 8; ++q) sc[q] = scn[q];
    };
    auto run_y = [&](auto dma_tag, char* cur, int kt) {
      if constexpr (WIDE) wide_y(dma_tag, cur, kt);
      else phase_y(dma_tag, cur, kt);
    };
    auto run_x = [&](auto dma_tag, const char* nxt, char* cur, int kt) {
      if constexpr (WIDE) wide_x(dma_tag, nxt, cur, kt);
      else phase_x(dma_tag, nxt, cur, kt);
    };
    read_scales(sc, 0);
#pragma unroll
    for (int i = 0; i < 16; ++i) read(F0, B0, 0, i);
    if constexpr (WIDE) {
      wa[0] = widen(F0, sc, 4, 0);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) wb[0][mb] = widen(F0, sc, mb, 0);
    }
    using Yes = std::true_type;
    using No = std::false_type;
    int end = KT;
    asm volatile("" : "+s"(end));  // (opaque: whether there is a loop is not remembered across tiles)
    for (int kt = 0; kt + 2 < end; kt += 2) {
      run_y(Yes{}, B0, kt);
      run_x(Yes{}, B1, B0, kt);
      run_y(Yes{}, B1, kt + 1);
      run_x(Yes{}, B0, B1, kt + 1);
    }
    run_y(No{}, B0, KT - 2);
    // (behind a barrier of this tile, even where it has two K-steps only: s_claim is this tile's)
    const int nlid = first + step + s_claim;  // claims past the range fail: the loop ends
    const bool more = nlid < last;
    const Tile U = open_tile(more ? nlid : lid);
    const Raw raw = load_raw(U, thread());
    run_x(No{}, B1, B0, KT - 2);
    run_y(No{}, B1, KT - 1);
    // both buffers are free past the last barrier: the next tile's block 0 goes to B1 (its B0), the
    // epilogue stages through B0
    t = thread();
    lane = t & 63;
    put_raw(U, raw, 1 - P, t);
    const int64_t mw = T.m0 + wm * 128, nw = T.n0 + wn * 128;
    if (more) {
      stage(U, offsets_of(U, t), 0, B1, 0, 2 * PER);
      stage_scales(U, 0, w, t);
    }
    T = U;
    if constexpr (WIDE) {
      // the last half: its fragments are in F1, its first part is widened
#pragma unroll
      for (int part = 0; part < 4; ++part) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const bf16x8 pa = widen(F1, sc, 4 + nb, part);
#pragma unroll
          for (int mb = 0; mb < MB; ++mb)
            acc[nb][mb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(pa, widen(F1, sc, mb, part), acc[nb][mb], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NMF; ++i) mma(F1, i);
    }
    const Out out = {(char*)cold()->out, cold()->som, cold()->row_nnz, cold()->M, cold()->N, cold()->act, cold()->stream};
    if (mw + 128 <= out.M && nw + 128 <= out.N) {
      if constexpr (WIDE) tile_epilogue<4, MB, NB, PLAIN>(out, SF_F32, acc, mw, nw, lane, s_thr[P] + wn * 128, B0 + w * 16384);
      else f8_epilogue<ODT, PLAIN, false>(out, acc, mw, nw, lane, s_thr[P] + wn * 128, B0 + w * 16384);
      // vector-memory operations retire in issue order: at most the epilogue's NST stores outstanding
      // means that the next tile's DMAs have landed
      __builtin_amdgcn_s_waitcnt(0x0F70 | (NST & 15) | (((NST >> 4) & 3) << 14));
    } else {
      if constexpr (WIDE) tile_epilogue<4, MB, NB, PLAIN>(out, SF_F32, acc, mw, nw, lane, s_thr[P] + wn * 128, B0 + w * 16384);
      else f8_epilogue<ODT, PLAIN, true>(out, acc, mw, nw, lane, s_thr[P] + wn * 128, B0 + w * 16384);
      wait_vmcnt0();
    }
    return more;
  };
  for (;;) {
    if (!tile(std::integral_constant<int, 0>{})) break;
    if (!tile(std::integral_constant<int, 1>{})) break;
  }
}

// The persistent kernels' tile counters, before each launch.
__global__ void clear_counters_kernel(int32_t* ctr) {
  if (threadIdx.x < 8) ctr[threadIdx.x * sfenc::TILE_CTR_STRIDE] = 0;
}

}  // namespace sff8
