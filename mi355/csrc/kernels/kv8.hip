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

#include "../common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
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
// bytes at a time (V through LDS, where it is turned).
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
// P is split into two bf16 numbers, p = hi + lo (16 significant bits, so P
// adds no error beside the output's own rounding).  With at most 8 query heads
// a group, columns 8..15 repeat the queries of 0..7 and carry `lo`: the same
// instruction does both.  Scores, statistics and sums are fp32.
//
// Few rows and a long cache: the blocks of a sequence are dealt to `nsplit`
// workgroups, whose (o, m, l) a second kernel joins.
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

// the first n of 16 bytes
DEVINL u32x4 keep_bytes(u32x4 x, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int k = min(max(n - 4 * i, 0), 4);
    x[i] &= k == 4 ? 0xffffffffu : (1u << (8 * k)) - 1u;
  }
  return x;
}

struct AttnArgs {
  const float* bias;   // (1 or B, Hq, width) or null
  const float* kpad;   // (B, width) or null
  long bias_b, bias_h, kpad_b;
  float scale;
  int Hq, H, G, NB, max_len, nsplit;
  bool mask16;         // mask rows are 16-byte aligned
};

constexpr float LOG2E = 1.4426950408889634f;

// sixteen values of a mask row from token tok0; behind the sequence's end the
// last one again
DEVINL void mask16(const float* row, int tok0, int len, bool aligned, f32x4* out) {
  if (aligned && tok0 + 16 <= len) {
#pragma unroll
    for (int t = 0; t < 4; ++t) out[t] = *reinterpret_cast<const f32x4*>(row + tok0 + 4 * t);
  } else {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) out[t][r] = row[min(tok0 + 4 * t + r, len - 1)];
  }
}

// WIDE: more than 8 query heads a cache head
template <typename T, int D, bool WIDE, bool BIAS, bool KPAD>
__global__ void __launch_bounds__(256)
kv8_attn_kernel(const T* __restrict__ q, long qsb, long qsh, const unsigned char* __restrict__ kc,
                const unsigned char* __restrict__ vc, const float* __restrict__ ksc,
                const float* __restrict__ vsc, PerSeq lengths, AttnArgs a, T* __restrict__ out,
                float* __restrict__ part) {
  constexpr int WAVES = 4;
  constexpr int KSTEP = D / 32;        // matrix instructions along d
  constexpr int DT16 = D / 16;         // tiles of 16 d
  constexpr int COLS = WIDE ? 16 : 8;  // query heads a workgroup takes
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c16 = lane & 15;
  const long bh = blockIdx.x;
  const int b = bh / a.H, h = bh % a.H;
  const int split = blockIdx.y;
  const int q0 = blockIdx.z * COLS;                    // first query head of the group
  const int col = WIDE ? c16 : (c16 & 7);
  const bool lo_half = !WIDE && c16 >= 8;
  const bool col_ok = q0 + col < a.G;
  const int hq = h * a.G + q0 + (col_ok ? col : 0);
  const int len = min(max(lengths.at(b), 0), a.max_len);
  const int nblk = (len + BLK - 1) / BLK;

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
  float m = -INFINITY, l = 0.f;       // l: this lane group's share

  const int krow = (c16 >> 2) * 16 + (c16 & 3);
  for (int blk = split * WAVES + wave; blk < nblk; blk += a.nsplit * WAVES) {
    const unsigned char* kb = kc + (bh * a.NB + blk) * (long)(BLK * D);
    const unsigned char* vb = vc + (bh * a.NB + blk) * (long)(BLK * D);
    const float kscale = ksc[bh * a.NB + blk] * a.scale;
    const float vscale = vsc[bh * a.NB + blk];
    // loads first: V's are in flight while the scores are made
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

    f32x4 sc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < KSTEP; ++s) sc[t] = KFrag<T>::mfma(KFrag<T>::load(kr[t][s]), qf[s], sc[t]);
    }
    const int tok0 = blk * BLK + 16 * g;     // this lane group's 16 tokens
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) sc[t][r] *= kscale;
    if (BIAS) {
      f32x4 m4[4];
      mask16(a.bias + b * a.bias_b + hq * a.bias_h, tok0, len, a.mask16, m4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[t][r] += m4[t][r];
    }
    unsigned gone = 0;                       // tokens of this lane group that are not there
    if (KPAD) {
      f32x4 m4[4];
      mask16(a.kpad + b * a.kpad_b, tok0, len, a.mask16, m4);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          sc[t][r] += m4[t][r];
          gone |= m4[t][r] == -INFINITY ? 1u << (4 * t + r) : 0u;
        }
    }
    if ((blk + 1) * BLK > len) {             // the sequence ends in this block
      const int n = min(max(len - tok0, 0), 16);
      gone |= 0xffffu & ~((1u << n) - 1u);
    }
    if (__any(gone != 0)) {
      // what is not there counts for nothing whatever its bytes hold, NaN codes
      // and NaN masks among them
      u32x4 keep;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        unsigned bytes = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool is_gone = gone >> (4 * t + r) & 1u;
          if (is_gone) sc[t][r] = -INFINITY;
          bytes |= is_gone ? 0u : 0xffu << (8 * r);
        }
        keep[t] = bytes;
      }
#pragma unroll
      for (int i = 0; i < DT16; ++i) vr[i] &= keep;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sc[t][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((m - ref) * LOG2E);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < DT16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
    bf16x8 ph[2], pl[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = __builtin_amdgcn_exp2f((sc[t][r] - ref) * LOG2E);
        l += p;
        const __bf16 hi = (__bf16)p;
        const __bf16 low = (__bf16)(p - (float)hi);
        const int e = 4 * (t & 1) + r;
        ph[t >> 1][e] = !WIDE && lo_half ? low : hi;
        if (WIDE) pl[t >> 1][e] = low;
      }
#pragma unroll
    for (int i = 0; i < DT16; ++i) {
      const bf16x8 v0 = v_frag(vr[i][0], vr[i][1], vscale);
      const bf16x8 v1 = v_frag(vr[i][2], vr[i][3], vscale);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, ph[0], acc[i], 0, 0, 0);
      acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, ph[1], acc[i], 0, 0, 0);
      if (WIDE) {
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pl[0], acc[i], 0, 0, 0);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pl[1], acc[i], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (!WIDE) {                       // hi and lo columns
#pragma unroll
    for (int i = 0; i < DT16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][r] += __shfl_xor(acc[i][r], 8);
  }

  // join the waves
  __shared__ float so[WAVES][COLS][D + 4];
  __shared__ float sm[WAVES][COLS], sl[WAVES][COLS];
  if (c16 < COLS) {
    // D layout: column = query, row d = 16i + 4g + r
#pragma unroll
    for (int i = 0; i < DT16; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) so[wave][c16][16 * i + 4 * g + r] = acc[i][r];
    if (g == 0) { sm[wave][c16] = m; sl[wave][c16] = l; }
  }
  __syncthreads();
  const int ncol = min(COLS, a.G - q0);
  for (int e = threadIdx.x; e < ncol * D; e += 256) {
    const int c = e / D, d = e % D;
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) mm = fmaxf(mm, sm[w][c]);
    const float ref = mm == -INFINITY ? 0.f : mm;
    float o = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = __builtin_amdgcn_exp2f((sm[w][c] - ref) * LOG2E);
      o += so[w][c][d] * f;
      ll += sl[w][c] * f;
    }
    const int head = h * a.G + q0 + c;
    if (a.nsplit == 1) {
      // l is NaN where a score was: then so is the output
      out[((long)b * a.Hq + head) * D + d] = DT<T>::from_f32(ll == 0.f ? 0.f : o / ll);
    } else {
      float* p = part + (((long)b * a.Hq + head) * a.nsplit + split) * (D + 2);
      p[d] = o;
      if (d == 0) { p[D] = mm; p[D + 1] = ll; }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(D) kv8_join_kernel(const float* __restrict__ part,
                                                     T* __restrict__ out, int nsplit) {
  const float* p = part + (long)blockIdx.x * nsplit * (D + 2);
  const int d = threadIdx.x;
  float mm = -INFINITY;
  for (int s = 0; s < nsplit; ++s) mm = fmaxf(mm, p[s * (D + 2) + D]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float o = 0.f, ll = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float f = __builtin_amdgcn_exp2f((p[s * (D + 2) + D] - ref) * LOG2E);
    o += p[s * (D + 2) + d] * f;
    ll += p[s * (D + 2) + D + 1] * f;
  }
  out[(long)blockIdx.x * D + d] = DT<T>::from_f32(ll == 0.f ? 0.f : o / ll);
}

struct Cache {
  torch::Tensor k, v, ks, vs;
  long B, H, NB, D;
};

Cache check_cache(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& ks,
                  const torch::Tensor& vs) {
  TORCH_CHECK(k.dim() == 4 && v.dim() == 5 && ks.dim() == 3 && vs.dim() == 3,
              "kv8: k (B,H,NB*64,D), v (B,H,NB,D,64), scales (B,H,NB)");
  Cache c{k, v, ks, vs, v.size(0), v.size(1), v.size(2), v.size(3)};
  TORCH_CHECK(v.size(4) == BLK && k.size(0) == c.B && k.size(1) == c.H &&
                  k.size(2) == c.NB * BLK && k.size(3) == c.D,
              "kv8: k and v are not of one cache");
  TORCH_CHECK(c.D == 32 || c.D == 64 || c.D == 128, "kv8: head dim 32, 64 or 128, got ", c.D);
  for (const auto& s : {ks, vs})
    TORCH_CHECK(s.size(0) == c.B && s.size(1) == c.H && s.size(2) == c.NB && s.is_contiguous() &&
                    s.scalar_type() == torch::kFloat && s.device() == k.device(),
                "kv8: scales must be contiguous fp32 (B,H,NB) on the cache's device");
  for (const auto& t : {k, v})
    TORCH_CHECK(t.is_contiguous() && t.element_size() == 1 && t.is_cuda() &&
                    t.device() == k.device() &&
                    reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0,
                "kv8: codes must be contiguous 8-bit device tensors, 16-byte aligned");
  TORCH_CHECK(c.NB < (1L << 24) && c.B * c.H < (1L << 31), "kv8: cache too large");
  return c;
}

PerSeq per_seq(const c10::optional<torch::Tensor>& each, long all, const Cache& c, const char* what) {
  if (each.has_value() && each->defined()) {
    TORCH_CHECK(each->dim() == 1 && each->size(0) == c.B && each->scalar_type() == torch::kInt &&
                    each->is_contiguous() && each->device() == c.k.device(),
                "kv8: ", what, " must be an int or a contiguous int32 (B,) tensor on the cache's device");
    return {each->data_ptr<int>(), 0};
  }
  TORCH_CHECK(all >= 0 && all < (1L << 30), "kv8: ", what, " out of range: ", all);
  return {nullptr, (int)all};
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
  for (const auto& t : {k, v})
    TORCH_CHECK(t.dim() == 4 && t.size(0) == c.B && t.size(1) == c.H && t.size(3) == c.D &&
                    t.size(2) == k.size(2) && t.device() == kc.device() &&
                    t.scalar_type() == k.scalar_type(),
                "kv8_append: k and v must be (B,H,S,D) of one type on the cache's device");
  const long S = k.size(2);
  const PerSeq st = per_seq(starts, start, c, "start");
  TORCH_CHECK(st.each || start + S <= c.NB * BLK, "kv8_append: ", start, " + ", S,
              " tokens do not fit a cache of ", c.NB * BLK);
  const PerSeq ct = per_seq(counts, S, c, "counts");
  if (S == 0 || c.B * c.H == 0) return;
  c10::DeviceGuard guard(kc.device());
  k = rows16(k);
  v = rows16(v);
  const long NW = (S + BLK - 2) / BLK + 1;
  TORCH_CHECK(c.B * c.H * NW < (1L << 31), "kv8_append: too many tokens at once");
  auto stream = at::hip::getCurrentHIPStream().stream();
  const Str3 kst{k.stride(0), k.stride(1), k.stride(2)}, vst{v.stride(0), v.stride(1), v.stride(2)};
#define APPEND(T, DD)                                                                            \
  hipLaunchKernelGGL((kv8_append_kernel<T, DD>), dim3(c.B* c.H* NW, 2), dim3(256), 0, stream,     \
                     (const T*)k.data_ptr(), (const T*)v.data_ptr(), kst, vst,                    \
                     (unsigned char*)kc.data_ptr(), (unsigned char*)vc.data_ptr(),                \
                     ks.data_ptr<float>(), vs.data_ptr<float>(), st, ct, (int)c.H, (int)S,        \
                     (int)c.NB, (int)NW)
#define BY_DIM(T, F)                            \
  do {                                          \
    if (c.D == 32) F(T, 32);                    \
    else if (c.D == 64) F(T, 64);               \
    else F(T, 128);                             \
  } while (0)
  if (k.scalar_type() == torch::kBFloat16) BY_DIM(__hip_bfloat16, APPEND);
  else if (k.scalar_type() == torch::kHalf) BY_DIM(__half, APPEND);
  else TORCH_CHECK(false, "kv8_append: bf16 or fp16 tokens, got ", k.scalar_type());
#undef APPEND
  HIP_CHECK_KERNEL();
}

torch::Tensor kv8_attn(torch::Tensor q, torch::Tensor kc, torch::Tensor vc, torch::Tensor ks,
                       torch::Tensor vs, c10::optional<torch::Tensor> lengths, long length,
                       long max_len, c10::optional<torch::Tensor> bias,
                       c10::optional<torch::Tensor> kpad, double scale) {
  const Cache c = check_cache(kc, vc, ks, vs);
  TORCH_CHECK(q.dim() == 4 && q.size(0) == c.B && q.size(2) == 1 && q.size(3) == c.D &&
                  q.device() == kc.device(),
              "kv8_attn: q must be (B,Hq,1,D) on the cache's device");
  const long Hq = q.size(1);
  TORCH_CHECK(c.H > 0 && Hq % c.H == 0, "kv8_attn: ", Hq, " query heads over ", c.H, " cache heads");
  const PerSeq ln = per_seq(lengths, length, c, "lengths");
  TORCH_CHECK(ln.each || length <= c.NB * BLK, "kv8_attn: length ", length,
              " over the cache's capacity ", c.NB * BLK);
  max_len = std::min(max_len, c.NB * BLK);
  TORCH_CHECK(max_len >= 0 && (ln.each || max_len >= length), "kv8_attn: max_len ", max_len,
              " under the length");
  AttnArgs a{};
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->dim() == 4 && (bias->size(0) == 1 || bias->size(0) == c.B) &&
                    bias->size(1) == Hq && bias->size(2) == 1 && bias->size(3) >= max_len &&
                    bias->scalar_type() == torch::kFloat && bias->stride(3) == 1 &&
                    bias->device() == kc.device(),
                "kv8_attn: bias must be fp32 (1 or B,Hq,1,>=max_len)");
    a.bias = bias->data_ptr<float>();
    a.bias_b = bias->size(0) > 1 ? bias->stride(0) : 0;
    a.bias_h = bias->stride(1);
  }
  if (kpad.has_value() && kpad->defined()) {
    TORCH_CHECK(kpad->dim() == 2 && kpad->size(0) == c.B && kpad->size(1) >= max_len &&
                    kpad->scalar_type() == torch::kFloat && kpad->stride(1) == 1 &&
                    kpad->device() == kc.device(),
                "kv8_attn: kpad must be fp32 (B,>=max_len)");
    a.kpad = kpad->data_ptr<float>();
    a.kpad_b = kpad->stride(0);
  }
  c10::DeviceGuard guard(kc.device());
  q = rows16(q);
  auto out = torch::empty({c.B, Hq, 1, c.D}, q.options().memory_format(at::MemoryFormat::Contiguous));
  if (c.B == 0 || Hq == 0) return out;
  if (max_len == 0) return out.zero_();
  const int G = Hq / c.H;
  const bool wide = G > 8;
  const int nz = (G + (wide ? 15 : 7)) / (wide ? 16 : 8);
  const long nblk = (max_len + BLK - 1) / BLK;
  // Enough workgroups to fill 256 CUs a few times over, and at least two
  // blocks of tokens for each of a workgroup's four waves.
  long nsplit = std::max(1L, std::min(1024 / std::max(1L, c.B * c.H * nz), nblk / 8));
  TORCH_CHECK(c.B * c.H < (1L << 31) && nz < 65536, "kv8_attn: too many heads");
  a.scale = (float)scale;
  a.Hq = Hq; a.H = c.H; a.G = G; a.NB = c.NB; a.max_len = max_len; a.nsplit = nsplit;
  torch::Tensor part;
  if (nsplit > 1) part = torch::empty({c.B * Hq * nsplit * (c.D + 2)}, ks.options());
  auto stream = at::hip::getCurrentHIPStream().stream();
  const dim3 grid(c.B * c.H, nsplit, nz);
  a.mask16 = (!a.bias || (reinterpret_cast<uintptr_t>(a.bias) % 16 == 0 && a.bias_b % 4 == 0 &&
                          a.bias_h % 4 == 0)) &&
             (!a.kpad || (reinterpret_cast<uintptr_t>(a.kpad) % 16 == 0 && a.kpad_b % 4 == 0));
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
    if (a.bias && a.kpad)                                                                        \
      wide ? run(kv8_attn_kernel<T, DD, true, true, true>, type)                                 \
           : run(kv8_attn_kernel<T, DD, false, true, true>, type);                               \
    else if (a.bias)                                                                             \
      wide ? run(kv8_attn_kernel<T, DD, true, true, false>, type)                                \
           : run(kv8_attn_kernel<T, DD, false, true, false>, type);                              \
    else if (a.kpad)                                                                             \
      wide ? run(kv8_attn_kernel<T, DD, true, false, true>, type)                                \
           : run(kv8_attn_kernel<T, DD, false, false, true>, type);                              \
    else                                                                                         \
      wide ? run(kv8_attn_kernel<T, DD, true, false, false>, type)                               \
           : run(kv8_attn_kernel<T, DD, false, false, false>, type);                             \
    if (nsplit > 1)                                                                              \
      hipLaunchKernelGGL((kv8_join_kernel<T, DD>), dim3(c.B* Hq), dim3(DD), 0, stream,           \
                         part.data_ptr<float>(), (T*)out.data_ptr(), (int)nsplit);               \
  } while (0)
  if (q.scalar_type() == torch::kBFloat16) BY_DIM(__hip_bfloat16, ATTN);
  else if (q.scalar_type() == torch::kHalf) BY_DIM(__half, ATTN);
  else TORCH_CHECK(false, "kv8_attn: bf16 or fp16 queries, got ", q.scalar_type());
#undef ATTN
#undef BY_DIM
  HIP_CHECK_KERNEL();
  return out;
}
