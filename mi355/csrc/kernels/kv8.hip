// A key/value cache held in 8 bits, its append and the single-token attention
// that reads it.
//
//   k        (B, H, NB*64, D)  e4m3     token-major
//   v        (B, H, NB, D, 64) e4m3     a block of 64 tokens is d-major
//   k_scale, v_scale (B, H, NB) fp32    a power of two for 64 tokens of a head
//
//   value = code * scale,  scale = 2^ceil(log2(amax/448)),  code = rne(x/scale)
//
// Powers of two make a block's growth cheap: when a later token needs a larger
// scale, the block's old codes are divided by a power of two, which e4m3 holds
// exactly except where a code becomes subnormal.  V is transposed inside a
// block because the product P V contracts over tokens: a lane then reads 16
// tokens of one d as 16 bytes, the operand layout of the matrix instruction.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <limits>

#include "../common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

constexpr int BLK = 64;       // tokens that share a scale
constexpr int E_MIN = -120, E_MAX = 120;

// ---------------------------------------------------------------------------
// 8-bit codes
// ---------------------------------------------------------------------------
// 2^ceil(log2(amax/448)) from the exponent field: 448 = 1.75 * 2^8, so the
// exponent of amax, less 8, plus one where the significand is over 1.75.
// Zero and everything below gets 2^E_MIN.
DEVINL float scale_for(float amax) {
  const unsigned u = __builtin_bit_cast(unsigned, amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = min(max(e, E_MIN), E_MAX);
  return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}

// what counts for a scale: NaN and infinities do not
DEVINL float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

// four floats, already divided by the scale -> four codes.  Infinities
// saturate, NaN stays NaN.
DEVINL unsigned encode4(float a, float b, float c, float d) {
  auto sat = [](float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); };
  unsigned r = 0;
  r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), r, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), r, true);
  return r;
}

DEVINL void decode4(unsigned codes, float* out) {
  const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
  const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
  out[0] = lo[0]; out[1] = lo[1]; out[2] = hi[0]; out[3] = hi[1];
}

DEVINL unsigned char encode1(float x) { return (unsigned char)(encode4(x, 0.f, 0.f, 0.f) & 0xff); }
DEVINL float decode1(unsigned char c) {
  float o[4];
  decode4(c, o);
  return o[0];
}

struct Str3 { long b, h, s; };

// start / counts / lengths: a number for all sequences, or one each
struct PerSeq {
  const int* each;
  int all;
  DEVINL int at(int b) const { return each ? each[b] : all; }
};

// ---------------------------------------------------------------------------
// Append: one workgroup for a (sequence, head, touched block) of K or of V.
// Bound by the bytes it moves: the new tokens are read once into registers,
// their largest value is found across the group, and codes are written 8 or 16
// bytes at a time (V through LDS, where it is turned).  512 tokens of 256 x 12
// heads of 64 in fp16: 126 us a call in a stream of them, 4.8 TB/s (a large copy
// reaches 4.9), 134 and more alone.  8 x 8 chunks of up to 137 tokens, D 128: 7.2 us;
// K alone 5.1, latency, V alone 6.8.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_append_kernel(const T* __restrict__ knew, const T* __restrict__ vnew, Str3 kst, Str3 vst,
                  unsigned char* __restrict__ kc, unsigned char* __restrict__ vc,
                  float* __restrict__ ks, float* __restrict__ vs, PerSeq start, PerSeq counts,
                  int H, int S, int NB, int NW) {
  constexpr int PER_ROW = D / 8;                 // 8-wide pieces of a token
  constexpr int PIECES = BLK * PER_ROW / 256;    // pieces a thread holds
  static_assert(PIECES >= 1, "");
  const int win = blockIdx.x % NW;
  const long bh = blockIdx.x / NW;
  const int b = bh / H, h = bh % H;
  const bool is_v = blockIdx.y;
  const int st = start.at(b);
  const int cnt = min(counts.at(b), S);
  if (st < 0 || cnt <= 0) return;
  const long blk = (long)(st / BLK) + win;
  const long end = (long)st + cnt;
  if (blk >= NB || blk * BLK >= end) return;
  const int first = max((int)(st - blk * BLK), 0);            // first new token in the block
  const int last = (int)min((long)BLK, end - blk * BLK);      // one past the last

  const T* src = is_v ? vnew + b * vst.b + h * vst.h : knew + b * kst.b + h * kst.h;
  const long ss = is_v ? vst.s : kst.s;
  unsigned char* codes = (is_v ? vc : kc) + (bh * NB + blk) * (BLK * D);
  float* scale_at = (is_v ? vs : ks) + bh * NB + blk;

  __shared__ float red[16];
  __shared__ alignas(16) unsigned char turn[D][BLK + 16];

  // read by every thread before the reduction's barriers, written after them
  const float old = first > 0 ? *scale_at : 0.f;
  float val[PIECES][8];
  float amax = 0.f;
#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int piece = threadIdx.x + p * 256;
    const int tok = piece / PER_ROW, d0 = (piece % PER_ROW) * 8;
#pragma unroll
    for (int u = 0; u < 8; ++u) val[p][u] = 0.f;
    if (tok >= first && tok < last) {
      const VecT<T, 8> in = vload<T, 8>(src + (blk * BLK + tok - st) * ss + d0);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        val[p][u] = DT<T>::to_f32(in.data[u]);
        amax = fmaxf(amax, finite_abs(val[p][u]));
      }
    }
  }
  amax = block_reduce_max(amax, red);
  float scale = scale_for(amax);
  scale = fmaxf(scale, old);
  const float inv = 1.f / scale;                    // exact: a power of two
  const bool regrow = first > 0 && scale > old;     // old codes are re-expressed

#pragma unroll
  for (int p = 0; p < PIECES; ++p) {
    const int piece = threadIdx.x + p * 256;
    const int tok = piece / PER_ROW, d0 = (piece % PER_ROW) * 8;
    const bool fresh = tok >= first && tok < last;
    if (!(fresh || (regrow && tok < first))) continue;
    u32x2 c;
    if (fresh) {
      c[0] = encode4(val[p][0] * inv, val[p][1] * inv, val[p][2] * inv, val[p][3] * inv);
      c[1] = encode4(val[p][4] * inv, val[p][5] * inv, val[p][6] * inv, val[p][7] * inv);
    } else {
      float o[8];
      if (is_v) {
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = decode1(codes[(d0 + u) * BLK + tok]);
      } else {
        const u32x2 was = *reinterpret_cast<const u32x2*>(codes + tok * D + d0);
        decode4(was[0], o);
        decode4(was[1], o + 4);
      }
      const float ratio = old * inv;
      c[0] = encode4(o[0] * ratio, o[1] * ratio, o[2] * ratio, o[3] * ratio);
      c[1] = encode4(o[4] * ratio, o[5] * ratio, o[6] * ratio, o[7] * ratio);
    }
    if (!is_v) {
      *reinterpret_cast<u32x2*>(codes + tok * D + d0) = c;
    } else {
#pragma unroll
      for (int u = 0; u < 8; ++u) turn[d0 + u][tok] = (unsigned char)(c[u >> 2] >> (8 * (u & 3)));
    }
  }
  if (is_v) {
    __syncthreads();
    const int lo = regrow ? 0 : first;              // tokens [lo, last) are in `turn`
#pragma unroll
    for (int p = 0; p < D * 4 / 256 + (D * 4 % 256 ? 1 : 0); ++p) {
      const int q = threadIdx.x + p * 256;
      const int d = q >> 2, t0 = (q & 3) * 16;
      if (d >= D) continue;
      if (lo <= t0 && last >= t0 + 16) {
        *reinterpret_cast<u32x4*>(codes + d * BLK + t0) =
            *reinterpret_cast<const u32x4*>(&turn[d][t0]);
      } else {
        for (int t = max(lo, t0); t < min(last, t0 + 16); ++t) codes[d * BLK + t] = turn[d][t];
      }
    }
  }
  if (threadIdx.x == 0) *scale_at = scale;
}

// four codes at another scale: `ratio` is a power of two of at most 1
DEVINL unsigned rescale4(unsigned codes, float ratio) {
  float o[4];
  decode4(codes, o);
  return encode4(o[0] * ratio, o[1] * ratio, o[2] * ratio, o[3] * ratio);
}

// ---------------------------------------------------------------------------
// Append of one token, a wave for a (sequence, head) of K or of V: a load, a
// reduction over the wave and a byte a lane to store.  The codes of the block
// are touched only if its scale has to grow, which happens to few tokens.
// Bound by latency: alone 3.2 us for 12 heads, 5 to 6 for 256 x 12 (as a block 13); a
// call whose 256 x 12 heads all grow 13.8 us, 9.0 where none does, launch included.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(256)
kv8_append_one_kernel(const T* __restrict__ knew, const T* __restrict__ vnew, Str3 kst, Str3 vst,
                      unsigned char* __restrict__ kc, unsigned char* __restrict__ vc,
                      float* __restrict__ ks, float* __restrict__ vs, PerSeq start, PerSeq counts,
                      int BH, int H, int NB) {
  constexpr int PER = D > 64 ? D / 64 : 1;        // values a lane holds
  const int lane = threadIdx.x & 63;
  const int bh = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool is_v = blockIdx.y;
  if (bh >= BH) return;
  const int b = bh / H, h = bh % H;
  const int st = start.at(b);
  if (st < 0 || st / BLK >= NB || counts.at(b) <= 0) return;
  const int at = st % BLK;
  const long blk = (long)bh * NB + st / BLK;
  const T* src = is_v ? vnew + b * vst.b + h * vst.h : knew + b * kst.b + h * kst.h;
  unsigned char* codes = (is_v ? vc : kc) + blk * (BLK * D);
  float* scale_at = (is_v ? vs : ks) + blk;
  const float old = at > 0 ? *scale_at : 0.f;
  const int d0 = lane * PER;
  float x[PER];
  float amax = 0.f;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    x[u] = d0 + u < D ? DT<T>::to_f32(src[d0 + u]) : 0.f;
    amax = fmaxf(amax, finite_abs(x[u]));
  }
  const float scale = fmaxf(scale_for(wave_reduce_max(amax)), old);
  const float inv = 1.f / scale;                  // exact: a power of two
  if (at > 0 && scale > old) {
    const float ratio = old * inv;
    const int t0 = lane % 16 * 4;                 // this lane's word of every fourth row of V
    if (!is_v) {
      for (int i = lane * 4; i < at * D; i += 256) {
        unsigned* c = reinterpret_cast<unsigned*>(codes + i);
        *c = rescale4(*c, ratio);
      }
    } else {
      // whole words before the new token's
      if (t0 + 4 <= at) {
        unsigned w[D / 4];
#pragma unroll
        for (int i = 0; i < D / 4; ++i) w[i] = *reinterpret_cast<const unsigned*>(codes + (lane / 16 + 4 * i) * BLK + t0);
#pragma unroll
        for (int i = 0; i < D / 4; ++i)
          *reinterpret_cast<unsigned*>(codes + (lane / 16 + 4 * i) * BLK + t0) = rescale4(w[i], ratio);
      }
      // the new token's word, by the lane that has its code: bytes before it
      // follow the scale, those behind it stay
      if (const int byte = at & 3) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          if (d0 + u >= D) break;
          unsigned* c = reinterpret_cast<unsigned*>(codes + (d0 + u) * BLK + at - byte);
          const unsigned before = (1u << (8 * byte)) - 1u, here = 0xffu << (8 * byte);
          const unsigned was = *c;
          *c = (rescale4(was, ratio) & before) | (unsigned)encode1(x[u] * inv) << (8 * byte) |
               (was & ~(before | here));
        }
        if (lane == 0) *scale_at = scale;
        return;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (d0 + u >= D) break;
    const unsigned char c = encode1(x[u] * inv);
    if (is_v) codes[(d0 + u) * BLK + at] = c;
    else codes[at * D + d0 + u] = c;
  }
  if (lane == 0) *scale_at = scale;
}

// ---------------------------------------------------------------------------
// Attention of one query token over the cache.
//
// A wave takes a block of 64 tokens at a time.  Scores: S^T = K Q^T, the K rows
// as matrix rows and up to 16 query heads of the group as columns; row i of
// tile t is token 16*(i/4) + 4t + i%4, so that lane group g = lane/16 ends up
// with the scores of tokens 16g..16g+15 - the very tokens whose V bytes it
// loads as one 16-byte piece per d.  P thus goes from one matrix instruction
// to the next without leaving its registers.  K codes are converted exactly to
// the query's type and the block's scale is multiplied into the score; V codes
// are converted to bf16 with the scale applied by the conversion (exact).
//
// A group has GP = 1, 2, 4, 8 or 16 query heads (the next power of two) for the
// matrix instruction's 16 columns.  Column c takes head c % GP and, of each
// lane group's 16 tokens, the GP from c / GP * GP on: its other weights are 0,
// and the columns of a head are summed at the end.  So a lane makes GP weights,
// not 16, and a token's weight is made once.
//
// P is split into three bf16 numbers, p = hi + mid + lo, 8 significant bits
// each: all of its 24.  (With two a weight is off by up to 2^-18, and ten times
// as many outputs land a step beside the nearest one.)  A column's other weights
// are 0, so mid and lo go there, one column and two columns of the same head
// further: up to 4 heads take one matrix instruction a tile for all three, up to
// 8 two, 16 three.  64 x 4 x 8 heads of 128 over 1024 tokens 26.7 us with two, 27.1
// with three.  The reference m that is subtracted in the exponent is raised, and
// what was summed rescaled, only when a score is over it by more than 8: weights
// then stay under e^8, which costs no precision in fp32 and bf16, and most blocks do
// without a reduction over the wave.  Scores, statistics and sums are fp32.
//
// Few rows and a long cache: the blocks of a sequence are dealt to `nsplit`
// workgroups, whose (o, m, l) a second kernel joins.  Short ones: the four
// waves of a workgroup take one, two or four sequences and heads.
//
// Bound by the codes' bytes where there are enough of them: 8 x 32 heads of 64
// over 5000 padded tokens 31 us (5.2 TB/s; a library's sum reads 4.0), 16 x 8
// x 4 heads of 128 over 8000 to 16384 tokens 80 us (5.0), 256 x 12 heads over
// 128 tokens 11.7 us (4.3); 12 heads over 45 tokens 4.1 us, all latency.  With
// the sixteen weights of a lane made in every column, the first of these took
// 38 us and the second, whose columns are half used, 77.
// ---------------------------------------------------------------------------
template <typename T> struct KFrag;
template <> struct KFrag<__hip_bfloat16> {
  using vec = bf16x8;
  static DEVINL vec load(u32x2 c) {
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], 1.f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[0], 1.f, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], 1.f, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[1], 1.f, true));
    return __builtin_bit_cast(vec, r);
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct KFrag<__half> {
  using vec = f16x8;
  static DEVINL vec load(u32x2 c) {
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], 1.f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[0], 1.f, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], 1.f, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c[1], 1.f, true));
    return __builtin_bit_cast(vec, r);
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

DEVINL bf16x8 v_frag(unsigned c0, unsigned c1, float scale) {
  u32x4 r;
  r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, scale, false));
  r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c0, scale, true));
  r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, scale, false));
  r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c1, scale, true));
  return __builtin_bit_cast(bf16x8, r);
}

struct AttnArgs {
  const float* bias;   // (1 or B, Hq, width) or null
  const float* kpad;   // (B, width) or null
  long bias_b, bias_h, kpad_b;
  float scale;
  int BH, Hq, H, G, NB, max_len, nsplit;
  int share;           // waves of a workgroup's 4 that share a sequence and head: 1, 2 or 4
};

constexpr int MAX_SPLIT = 256;
constexpr float LOG2E = 1.4426950408889634f;

// x of the lane that is BY away, round a row of 16
template <int BY, typename X> DEVINL X turned(X x) {
  static_assert(BY > 0 && BY < 16 && sizeof(X) == 4, "");
  return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x120 + BY,
                                                           0xf, 0xf, false));
}

// op over the columns of a head: lanes of a row of 16 that are GP apart
template <int GP, typename Op> DEVINL float over_columns(float x, Op op) {
  if (GP < 16) x = op(x, turned<8>(x));
  if (GP < 8) x = op(x, turned<4>(x));
  if (GP < 4) x = op(x, turned<2>(x));
  if (GP < 2) x = op(x, turned<1>(x));
  return x;
}

template <typename T, int D, int GP>
__global__ void __launch_bounds__(256)
kv8_attn_kernel(const T* __restrict__ q, long qsb, long qsh, const unsigned char* __restrict__ kc,
                const unsigned char* __restrict__ vc, const float* __restrict__ ksc,
                const float* __restrict__ vsc, PerSeq lengths, AttnArgs a, T* __restrict__ out,
                float* __restrict__ part) {
  constexpr int WAVES = 4;
  constexpr int KSTEP = D / 32;        // matrix instructions along d
  constexpr int DT16 = D / 16;         // tiles of 16 d
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // known to be uniform
  const int g = lane >> 4, c16 = lane & 15;
  const int sub = wave & (a.share - 1);                // of the waves that share
  const long bh_at = (long)blockIdx.x * (WAVES / a.share) + wave / a.share;
  const bool there = bh_at < a.BH;
  const long bh = there ? bh_at : 0;
  const int b = bh / a.H, h = bh % a.H;
  const int split = blockIdx.y;
  const int q0 = blockIdx.z * GP;                      // first query head of the group
  const int col = c16 % GP, part16 = c16 / GP;         // this lane's head, and its tokens
  // the tokens whose mid and lo it takes
  const int mid_part = GP <= 8 ? turned<GP <= 8 ? GP : 1>(part16) : part16;
  const int lo_part = GP <= 4 ? turned<GP <= 4 ? 2 * GP : 1>(part16) : part16;
  const bool col_ok = q0 + col < a.G;
  const int hq = h * a.G + q0 + (col_ok ? col : 0);
  const int len = min(max(lengths.at(b), 0), a.max_len);
  const int nblk = there ? (len + BLK - 1) / BLK : 0;
  const float* bias = a.bias ? a.bias + b * a.bias_b + hq * a.bias_h : nullptr;
  const float* kpad = a.kpad ? a.kpad + b * a.kpad_b : nullptr;

  // queries: lane (column, g) holds d = g*(D/4) + 8s + j
  typename KFrag<T>::vec qf[KSTEP];
#pragma unroll
  for (int s = 0; s < KSTEP; ++s) {
    u32x4 v = u32x4{0u, 0u, 0u, 0u};
    if (col_ok) v = *reinterpret_cast<const u32x4*>(q + b * qsb + hq * qsh + g * (D / 4) + 8 * s);
    qf[s] = __builtin_bit_cast(typename KFrag<T>::vec, v);
  }

  f32x4 acc[DT16];
#pragma unroll
  for (int i = 0; i < DT16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;       // m: of the head; l: this lane's share

  const int krow = (c16 >> 2) * 16 + (c16 & 3);
  for (int blk = split * a.share + sub; blk < nblk; blk += a.nsplit * a.share) {
    const unsigned char* kb = kc + (bh * a.NB + blk) * (long)(BLK * D);
    const unsigned char* vb = vc + (bh * a.NB + blk) * (long)(BLK * D);
    const float kscale = ksc[bh * a.NB + blk] * a.scale;
    const float vscale = vsc[bh * a.NB + blk];
    const int tok0 = blk * BLK + 16 * g;               // this lane group's 16 tokens
    const int tok = tok0 + part16 * GP;                // this lane's GP of them
    float add[GP], pad[GP];
#pragma unroll
    for (int i = 0; i < GP; ++i) {
      const int at = min(tok + i, len - 1);
      add[i] = bias ? bias[at] : 0.f;
      pad[i] = kpad ? kpad[at] : 0.f;
    }
    // loads in the order of their use: V's are in flight while scores are made
    u32x2 kr[4][KSTEP];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int s = 0; s < KSTEP; ++s)
        kr[t][s] = *reinterpret_cast<const u32x2*>(kb + (krow + 4 * t) * D + g * (D / 4) + 8 * s);
    u32x4 vr[DT16];
#pragma unroll
    for (int i = 0; i < DT16; ++i)
      vr[i] = *reinterpret_cast<const u32x4*>(vb + (16 * i + c16) * BLK + 16 * g);
    f32x16 sc;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 s4 = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KSTEP; ++s) s4 = KFrag<T>::mfma(KFrag<T>::load(kr[t][s]), qf[s], s4);
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[4 * t + r] = s4[r];
    }
    // this lane's GP scores to the front
#pragma unroll
    for (int n = 8; n >= GP; n >>= 1) {
      const bool upper = part16 & (n / GP);
#pragma unroll
      for (int i = 0; i < n; ++i) sc[i] = upper ? sc[i + n] : sc[i];
    }
    bool hole = (blk + 1) * BLK > len;                 // the sequence ends in this block
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < GP; ++i) {
      sc[i] = fmaf(sc[i], kscale, add[i]) + pad[i];
      const bool gone = tok + i >= len || pad[i] == -INFINITY;
      sc[i] = gone ? -INFINITY : sc[i];
      hole |= gone;
      mx = fmaxf(mx, sc[i]);
    }
    if (__any(hole)) {
      // what is not there counts for nothing whatever its bytes hold, NaN codes
      // among them
      unsigned gone = 0xffffu & ~((1u << min(max(len - tok0, 0), 16)) - 1u);
      if (kpad) {
#pragma unroll 4
        for (int j = 0; j < 16; ++j)
          gone |= kpad[min(tok0 + j, len - 1)] == -INFINITY ? 1u << j : 0u;
      }
      u32x4 keep;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        keep[t] = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) keep[t] |= gone >> (4 * t + r) & 1u ? 0u : 0xffu << (8 * r);
      }
#pragma unroll
      for (int i = 0; i < DT16; ++i) vr[i] &= keep;
    }
    if (__any(mx > m + 8.f)) {
      mx = over_columns<GP>(mx, [](float x, float y) { return fmaxf(x, y); });
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float mn = fmaxf(m, mx);
      const float alpha = __builtin_amdgcn_exp2f((m - (mn == -INFINITY ? 0.f : mn)) * LOG2E);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < DT16; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    constexpr int PAIRS = GP > 1 ? GP / 2 : 1;
    unsigned hi[PAIRS], mid[PAIRS], lo[PAIRS];         // two tokens each
    if (GP == 1) {
      const float p = __builtin_amdgcn_exp2f((sc[0] - ref) * LOG2E);
      l += p;
      const __bf16 h1 = (__bf16)p;
      const float rest = p - (float)h1;
      const __bf16 m1 = (__bf16)rest;
      const __bf16 l1 = (__bf16)(rest - (float)m1);
      const int odd = 16 * (c16 & 1);
      hi[0] = (unsigned)__builtin_bit_cast(unsigned short, h1) << odd;
      mid[0] = (unsigned)__builtin_bit_cast(unsigned short, m1) << odd;
      lo[0] = (unsigned)__builtin_bit_cast(unsigned short, l1) << odd;
    } else {
#pragma unroll
      for (int i = 0; i < GP / 2; ++i) {
        const float p0 = __builtin_amdgcn_exp2f((sc[2 * i] - ref) * LOG2E);
        const float p1 = __builtin_amdgcn_exp2f((sc[2 * i + 1] - ref) * LOG2E);
        l += p0;
        l += p1;
        const bf16x2 h2 = bf16x2{(__bf16)p0, (__bf16)p1};
        const float r0 = p0 - (float)h2[0], r1 = p1 - (float)h2[1];
        const bf16x2 m2 = bf16x2{(__bf16)r0, (__bf16)r1};
        const bf16x2 l2 = bf16x2{(__bf16)(r0 - (float)m2[0]), (__bf16)(r1 - (float)m2[1])};
        hi[i] = __builtin_bit_cast(unsigned, h2);
        mid[i] = __builtin_bit_cast(unsigned, m2);
        lo[i] = __builtin_bit_cast(unsigned, l2);
      }
    }
    // The column's weights, tokens 2e and 2e + 1 in a word: hi of this lane's
    // tokens; mid and lo of those of the head's next two columns, as far as it has
    // as many, else in operands of their own.
    if (GP <= 8) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) mid[i] = turned<GP <= 8 ? GP : 1>(mid[i]);
    }
    if (GP <= 4) {
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) lo[i] = turned<GP <= 4 ? 2 * GP : 1>(lo[i]);
    }
    u32x4 p[1 + (GP > 8) + (GP > 4)][2];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const auto of = [&](int part, const unsigned (&w)[PAIRS]) {
        return (GP > 1 ? part == e / PAIRS : part >> 1 == e) ? w[e % PAIRS] : 0u;
      };
      const unsigned h = of(part16, hi), m_ = of(mid_part, mid), l_ = of(lo_part, lo);
      p[0][e >> 2][e & 3] = GP <= 4 ? h | m_ | l_ : GP <= 8 ? h | m_ : h;
      if (GP > 8) p[1][e >> 2][e & 3] = m_;
      if (GP > 4) p[GP > 8 ? 2 : 1][e >> 2][e & 3] = l_;
    }
#pragma unroll
    for (int i = 0; i < DT16; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bf16x8 v = v_frag(vr[i][2 * e], vr[i][2 * e + 1], vscale);
#pragma unroll
        for (int j = 0; j < (int)(sizeof(p) / sizeof(p[0])); ++j)
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, __builtin_bit_cast(bf16x8, p[j][e]), acc[i], 0, 0, 0);
      }
  }
  const auto sum = [](float x, float y) { return x + y; };
  l = over_columns<GP>(l, sum);
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
#pragma unroll
  for (int i = 0; i < DT16; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) acc[i][r] = over_columns<GP>(acc[i][r], sum);

  // join the waves
  __shared__ float so[WAVES][GP][D + 4];
  __shared__ float sm[WAVES][GP], sl[WAVES][GP];
  if (c16 < GP) {
    // D layout: column = query, row d = 16i + 4g + r
#pragma unroll
    for (int i = 0; i < DT16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[wave][c16][16 * i + 4 * g + r] = acc[i][r];
    if (g == 0) { sm[wave][c16] = m; sl[wave][c16] = l; }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < WAVES / a.share * GP * D; e += 256) {
    const int d = e % D, c = e / D % GP, pair = e / D / GP, w0 = pair * a.share;
    const long row = (long)blockIdx.x * (WAVES / a.share) + pair;
    if (row >= a.BH || q0 + c >= a.G) continue;
    float mm = -INFINITY;
    for (int w = w0; w < w0 + a.share; ++w) mm = fmaxf(mm, sm[w][c]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float o = 0.f, ll = 0.f;
    for (int w = w0; w < w0 + a.share; ++w) {
      const float f = __builtin_amdgcn_exp2f((sm[w][c] - ref) * LOG2E);
      o += so[w][c][d] * f;
      ll += sl[w][c] * f;
    }
    const long head = row * a.G + q0 + c;            // of B * Hq
    if (a.nsplit == 1) {
      // l is NaN where a score was: then so is the output
      out[head * D + d] = DT<T>::from_f32(ll == 0.f ? 0.f : o / ll);
    } else {
      part[(head * a.nsplit + split) * D + d] = o;
      if (d == 0) {
        float* ml = part + (long)a.BH * a.G * a.nsplit * D + (head * a.nsplit + split) * 2;
        ml[0] = mm;
        ml[1] = ll;
      }
    }
  }
}

// Joins the nsplit parts of each query head: a workgroup of whole waves a head,
// a thread a d.
template <typename T, int D>
__global__ void __launch_bounds__(D < 64 ? 64 : D) kv8_join_kernel(const float* __restrict__ part,
                                                     T* __restrict__ out, long heads, int nsplit) {
  __shared__ float f[MAX_SPLIT];
  const long head = blockIdx.x;
  const int d = threadIdx.x, lane = d & 63;
  const float* p = part + head * nsplit * D + min(d, D - 1);
  const float2* ml = reinterpret_cast<const float2*>(part + heads * nsplit * D) + head * nsplit;
  float mm = -INFINITY, ll = 0.f;
  // each wave for itself: a lane a part
  for (int s = lane; s < nsplit; s += 64) mm = fmaxf(mm, ml[s].x);
  mm = wave_reduce_max(mm);
  const float ref = mm == -INFINITY ? 0.f : mm;
  for (int s = lane; s < nsplit; s += 64) {
    const float2 v = ml[s];
    const float w = __builtin_amdgcn_exp2f((v.x - ref) * LOG2E);
    f[s] = w;                                        // the same from every wave
    ll += v.y * w;
  }
  ll = wave_reduce_sum(ll);
  __syncthreads();
  float o = 0.f;
#pragma unroll 8
  for (int s = 0; s < nsplit; ++s) o += p[(long)s * D] * f[s];
  if (d < D) out[head * D + d] = DT<T>::from_f32(ll == 0.f ? 0.f : o / ll);
}

struct Cache {
  const torch::Tensor &k, &v, &ks, &vs;
  long B, H, NB, D;
};

Cache check_cache(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ks,
                  const torch::Tensor& vs) {
  VALUE_CHECK(k.dim() == 4 && v.dim() == 5 && ks.dim() == 3 && vs.dim() == 3,
              "kv8: k (B,H,NB*64,D), v (B,H,NB,D,64), scales (B,H,NB)");
  const Cache c{k, v, ks, vs, v.size(0), v.size(1), v.size(2), v.size(3)};
  VALUE_CHECK(v.size(4) == BLK && k.size(0) == c.B && k.size(1) == c.H &&
                  k.size(2) == c.NB * BLK && k.size(3) == c.D,
              "kv8: k and v are not of one cache");
  VALUE_CHECK(c.D == 32 || c.D == 64 || c.D == 128, "kv8: head dim 32, 64 or 128, got ", c.D);
  for (const auto* s : {&ks, &vs})
    VALUE_CHECK(s->size(0) == c.B && s->size(1) == c.H && s->size(2) == c.NB && s->is_contiguous() &&
                    s->scalar_type() == torch::kFloat && s->device() == k.device(),
                "kv8: scales must be contiguous fp32 (B,H,NB) on the cache's device");
  for (const auto* t : {&k, &v})
    VALUE_CHECK(t->is_contiguous() && t->element_size() == 1 && t->is_cuda() &&
                    t->device() == k.device() &&
                    reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "kv8: codes must be contiguous 8-bit device tensors, 16-byte aligned");
  VALUE_CHECK(c.NB < (1L << 24) && c.B * c.H < (1L << 31), "kv8: cache too large");
  return c;
}

// `each`, if given, as int32 (kept alive by the caller's tensor)
PerSeq per_seq(c10::optional<torch::Tensor>& each, long all, const Cache& c, const char* what) {
  if (each.has_value() && each->defined()) {
    VALUE_CHECK(each->dim() == 1 && each->size(0) == c.B && each->device() == c.k.device() &&
                    c10::isIntegralType(each->scalar_type(), /*includeBool=*/false),
                "kv8: ", what, " must be a number or an int32 (", c.B, ",) tensor on ",
                c.k.device(), ", got ", each->sizes(), " on ", each->device());
    if (each->scalar_type() == torch::kLong)        // past every capacity, or under 0, either way
      each = each->clamp(std::numeric_limits<int>::min(), std::numeric_limits<int>::max());
    if (each->scalar_type() != torch::kInt || !each->is_contiguous())
      each = each->to(torch::kInt).contiguous();
    return {each->data_ptr<int>(), 0};
  }
  VALUE_CHECK(all >= 0 && all < (1L << 30), "kv8: ", what, " out of range: ", all);
  return {nullptr, (int)all};
}

void check_tokens(const torch::Tensor& t, const Cache& c, const char* what) {
  VALUE_CHECK(t.device() == c.k.device(), what, ": tokens on ", t.device(), ", cache on ", c.k.device());
  VALUE_CHECK(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kHalf, what,
              " takes bf16 or fp16 on a GPU, got ", t.scalar_type());
  NO_GRAD_CHECK(t, "an 8-bit cache");
}

// (B,H,S,D) with D contiguous and every row 16-byte aligned
torch::Tensor rows16(torch::Tensor t) {
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % 8 == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

}  // namespace

void kv8_append(torch::Tensor k, torch::Tensor v, torch::Tensor kc, torch::Tensor vc,
                torch::Tensor ks, torch::Tensor vs, c10::optional<torch::Tensor> starts, long start,
                c10::optional<torch::Tensor> counts) {
  const Cache c = check_cache(kc, vc, ks, vs);
  check_tokens(k, c, "kv8_append");
  check_tokens(v, c, "kv8_append");
  VALUE_CHECK(k.dim() == 4 && k.size(0) == c.B && k.size(1) == c.H && k.size(3) == c.D &&
                  v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
              "kv8_append: k ", k.sizes(), " and v ", v.sizes(), " of one type do not fit a cache of ",
              kc.sizes());
  const long S = k.size(2);
  c10::DeviceGuard guard(kc.device());
  const PerSeq st = per_seq(starts, start, c, "start");
  VALUE_CHECK(st.each || start + S <= c.NB * BLK, "kv8_append: ", S, " tokens at ", start,
              " do not fit a cache of ", c.NB * BLK);
  const PerSeq ct = per_seq(counts, S, c, "counts");
  if (S == 0 || c.B * c.H == 0) return;
  const long NW = (S + BLK - 2) / BLK + 1;
  VALUE_CHECK(S < (1L << 30) && fits_a_launch(S == 1 ? (c.B * c.H + 3) / 4 : c.B * c.H * NW, 256),
              "kv8_append: too many tokens at once: ", k.sizes());
  k = rows16(k);
  v = rows16(v);
  auto stream = at::hip::getCurrentHIPStream().stream();
  const Str3 kst{k.stride(0), k.stride(1), k.stride(2)}, vst{v.stride(0), v.stride(1), v.stride(2)};
#define APPEND(T, DD)                                                                            \
  if (S == 1)                                                                                    \
    hipLaunchKernelGGL((kv8_append_one_kernel<T, DD>), dim3((c.B * c.H + 3) / 4, 2), dim3(256),   \
                       0, stream, (const T*)k.data_ptr(), (const T*)v.data_ptr(), kst, vst,       \
                       (unsigned char*)kc.data_ptr(), (unsigned char*)vc.data_ptr(),              \
                       ks.data_ptr<float>(), vs.data_ptr<float>(), st, ct, (int)(c.B * c.H),      \
                       (int)c.H, (int)c.NB);                                                      \
  else                                                                                            \
  hipLaunchKernelGGL((kv8_append_kernel<T, DD>), dim3(c.B* c.H* NW, 2), dim3(256), 0, stream,     \
                     (const T*)k.data_ptr(), (const T*)v.data_ptr(), kst, vst,                    \
                     (unsigned char*)kc.data_ptr(), (unsigned char*)vc.data_ptr(),                \
                     ks.data_ptr<float>(), vs.data_ptr<float>(), st, ct, (int)c.H, (int)S,        \
                     (int)c.NB, (int)NW)
#define BY_DIM(T, F)                            \
  do {                                          \
    if (c.D == 32) { F(T, 32); }                \
    else if (c.D == 64) { F(T, 64); }           \
    else { F(T, 128); }                         \
  } while (0)
  if (k.scalar_type() == torch::kBFloat16) BY_DIM(__hip_bfloat16, APPEND);
  else BY_DIM(__half, APPEND);
#undef APPEND
  HIP_CHECK_KERNEL();
}

torch::Tensor kv8_attn(torch::Tensor q, torch::Tensor kc, torch::Tensor vc, torch::Tensor ks,
                       torch::Tensor vs, c10::optional<torch::Tensor> lengths, long length,
                       long max_len, bool has_max_len, c10::optional<torch::Tensor> bias,
                       c10::optional<torch::Tensor> kpad, double scale) {
  const Cache c = check_cache(kc, vc, ks, vs);
  check_tokens(q, c, "decode_attention_kv8");
  VALUE_CHECK(q.dim() == 4 && q.size(0) == c.B && q.size(2) == 1 && q.size(3) == c.D && c.H > 0 &&
                  q.size(1) % c.H == 0,
              "decode_attention_kv8: q ", q.sizes(), " does not fit a cache of ", kc.sizes());
  const long Hq = q.size(1), cap = c.NB * BLK;
  c10::DeviceGuard guard(kc.device());
  const PerSeq ln = per_seq(lengths, length, c, "lengths");
  VALUE_CHECK(ln.each || length <= cap, "decode_attention_kv8: length ", length, " in a cache of ", cap);
  VALUE_CHECK(!has_max_len || (max_len >= 0 && (ln.each || max_len >= length)),
              "decode_attention_kv8: max_len ", max_len, " under the length");
  if (!has_max_len) max_len = ln.each ? cap : length;
  max_len = std::min(max_len, cap);
  AttnArgs a{};
  torch::Tensor masks[2];
  auto mask = [&](c10::optional<torch::Tensor>& t, int i, const char* what) -> const torch::Tensor& {
    NO_GRAD_CHECK(*t, "decode_attention_kv8");
    VALUE_CHECK(t->device() == kc.device() && t->size(-1) >= max_len, "decode_attention_kv8: ", what, " ",
                t->sizes(), " on ", t->device(), " for max_len ", max_len, " on ", kc.device());
    masks[i] = t->scalar_type() == torch::kFloat && t->stride(-1) == 1 ? *t : t->to(torch::kFloat).contiguous();
    return masks[i];
  };
  if (bias.has_value() && bias->defined()) {
    VALUE_CHECK(bias->dim() == 4 && (bias->size(0) == 1 || bias->size(0) == c.B) &&
                    bias->size(1) == Hq && bias->size(2) == 1,
                "decode_attention_kv8: bias ", bias->sizes(), " is not (1 or ", c.B, ", ", Hq, ", 1, .)");
    const auto& m = mask(bias, 0, "bias");
    a.bias = m.data_ptr<float>();
    a.bias_b = m.size(0) > 1 ? m.stride(0) : 0;
    a.bias_h = m.stride(1);
  }
  if (kpad.has_value() && kpad->defined()) {
    VALUE_CHECK(kpad->dim() == 2 && kpad->size(0) == c.B,
                "decode_attention_kv8: kpad ", kpad->sizes(), " is not (", c.B, ", .)");
    const auto& m = mask(kpad, 1, "kpad");
    a.kpad = m.data_ptr<float>();
    a.kpad_b = m.stride(0);
  }
  q = rows16(q);
  auto out = at::empty({c.B, Hq, 1, c.D}, q.options().memory_format(at::MemoryFormat::Contiguous));
  if (c.B == 0 || Hq == 0) return out;
  if (max_len == 0) return out.zero_();
  const int G = Hq / c.H;
  const int GP = G > 8 ? 16 : G > 4 ? 8 : G > 2 ? 4 : G;
  const int nz = (G + GP - 1) / GP;
  const long nblk = (max_len + BLK - 1) / BLK;
  // Split a long cache over workgroups until there are 512 of them, two for
  // each CU (ragged lengths even out), but leave each 8 blocks of tokens, and
  // leave caches alone whose blocks take less time than the join: one sequence
  // of 32 heads over 16384 tokens 111 -> 32 us, of 12 heads over 512 tokens
  // (8 blocks) 5.1 -> 7.2 us.
  const long nsplit = nblk < 32 ? 1 : std::max(1L, std::min({512 / (c.B * c.H * nz), nblk / 8, (long)MAX_SPLIT}));
  VALUE_CHECK(nz < 65536, "decode_attention_kv8: too many heads");
  a.scale = (float)scale;
  a.share = nsplit > 1 || nblk > 3 ? 4 : nblk > 1 ? 2 : 1;
  a.BH = c.B * c.H; a.Hq = Hq; a.H = c.H; a.G = G; a.NB = c.NB; a.max_len = max_len; a.nsplit = nsplit;
  torch::Tensor part;
  if (nsplit > 1) part = torch::empty({c.B * Hq * nsplit * (c.D + 2)}, ks.options());
  auto stream = at::hip::getCurrentHIPStream().stream();
  const long groups = (c.B * c.H + 4 / a.share - 1) / (4 / a.share);
  VALUE_CHECK(fits_a_launch(groups, 256), "decode_attention_kv8: too many heads: ", kc.sizes());
  const dim3 grid(groups, nsplit, nz);
  auto run = [&](auto kernel, auto* type) {
    using T = std::remove_pointer_t<decltype(type)>;
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, (const T*)q.data_ptr(),
                       (long)q.stride(0), (long)q.stride(1), (const unsigned char*)kc.data_ptr(),
                       (const unsigned char*)vc.data_ptr(), ks.data_ptr<float>(),
                       vs.data_ptr<float>(), ln, a, (T*)out.data_ptr(),
                       nsplit > 1 ? part.data_ptr<float>() : nullptr);
  };
#define ATTN(T, DD)                                                                              \
  do {                                                                                           \
    T* type = nullptr;                                                                           \
    if (GP == 1) run(kv8_attn_kernel<T, DD, 1>, type);                                           \
    else if (GP == 2) run(kv8_attn_kernel<T, DD, 2>, type);                                      \
    else if (GP == 4) run(kv8_attn_kernel<T, DD, 4>, type);                                      \
    else if (GP == 8) run(kv8_attn_kernel<T, DD, 8>, type);                                      \
    else run(kv8_attn_kernel<T, DD, 16>, type);                                                  \
    if (nsplit > 1)                                                                              \
      hipLaunchKernelGGL((kv8_join_kernel<T, DD>), dim3(c.B* Hq), dim3(DD < 64 ? 64 : DD), 0,    \
                         stream, part.data_ptr<float>(), (T*)out.data_ptr(), c.B* Hq,            \
                         (int)nsplit);                                                           \
  } while (0)
  if (q.scalar_type() == torch::kBFloat16) BY_DIM(__hip_bfloat16, ATTN);
  else BY_DIM(__half, ATTN);
#undef ATTN
#undef BY_DIM
  HIP_CHECK_KERNEL();
  return out;
}
