// Products of a few rows with 4-bit weights:  y[m,n] = sum_k x[m,k] * w[n,k],
// w[n,k] = e2m1(code[n,k]) * 2^(exp[n, k/32] - 127).
//
// Codes are two a byte (low nibble: even k), row-major (N, K/2), one exponent
// byte for 32 inputs (N, K/32): 4.25 bits a weight, laid out as the checkpoint
// holds them.  With few rows the weight bytes bound the product, so every
// weight is read once from memory, straight into registers, 16 bytes a lane:
// lane (n = lane%16, g = lane/16) owns the 32 codes of ONE scale group, row n,
// k = 128c + 32g .. +32.  CDNA4 converts two codes with a per-lane power-of-two
// scale in one instruction, so the group scale costs nothing, and the order of
// k inside a matrix instruction is free, so MFMA i takes bytes 4i..4i+3 of each
// lane (k = 128c + 32g + 8i + j) and x is read at the same k: no shuffle.
//
// Roundings: a converted weight has 2 significant bits and is exact in bf16 and
// fp16 as far as their exponents reach.  So its exponent is taken relative to
// the row's largest (put back in 32 bits at the end), in fp16 2^13 over it: from
// 6 * 2^13 = 49152 down to 2^-14, half of the smallest scale, a row may span 26
// octaves.  (Smaller ones would be exact as subnormal numbers, but a matrix
// instruction loses bits of their sum: 6 units of 2^-24 of the sum of sizes at 35
// octaves, 20 at 36, against 0.7 at up to 30.)  Groups of zeros do not count.
// Rows that span more, which hardly a trained weight has, are summed group by group
// in fp32 by the wave that stores them (far_outputs); their row exponent is given
// as 255.  One of them takes the product of one row by 20480 x 4096 from 12.7 to
// 13.0 us, of 16 rows by 10240 x 2048 from 8 to 21, of 256 from 25 to 92 (a lane an
// output: 74, 133, 619).  Sums are fp32; y is rounded once.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "../common.h"

namespace {

typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

template <typename T> struct Frag;
template <> struct Frag<__hip_bfloat16> {
  using vec = bf16x8;
  static constexpr int BIAS = 0;      // octaves that weights stand over their row's scale
  template <int S> static DEVINL unsigned cvt2(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, S));
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Frag<__half> {
  using vec = f16x8;
  static constexpr int BIAS = 13;
  template <int S> static DEVINL unsigned cvt2(unsigned codes, float scale) {
    return __builtin_bit_cast(unsigned,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, S));
  }
  static DEVINL f32x4 mfma(vec a, vec b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

// eight codes of one scale group -> eight weights
template <typename T>
DEVINL typename Frag<T>::vec decode8(unsigned codes, float scale) {
  u32x4 r;
  r[0] = Frag<T>::template cvt2<0>(codes, scale);
  r[1] = Frag<T>::template cvt2<1>(codes, scale);
  r[2] = Frag<T>::template cvt2<2>(codes, scale);
  r[3] = Frag<T>::template cvt2<3>(codes, scale);
  return __builtin_bit_cast(typename Frag<T>::vec, r);
}

// 2^(e - row_e + BIAS) as a float.  Of groups that are not all zeros the
// difference is from -26 to 0 (or the row is FAR).
template <typename T> DEVINL float group_scale(int e, int row_e) {
  const int d = min(max(e - row_e, -100), 0) + Frag<T>::BIAS;
  return __builtin_bit_cast(float, (unsigned)(d + 127) << 23);
}

// a sum of inputs times weights at group_scale, at the row's scale
template <typename T> DEVINL float at_row_scale(float sum, int row_e) {
  return __builtin_amdgcn_ldexpf(sum, row_e - 127 - Frag<T>::BIAS);
}

struct Args {
  const unsigned char *codes, *exps, *row_exp;
  int M, N, K;
  long ldx;
};

constexpr int FAR = 255;                // the row exponent of rows without one scale for all

constexpr int SPAN = 26;                // octaves that a row may span otherwise

// Each row's exponent, a wave a row and a lane a group: the largest of groups that
// hold more than zeros, or FAR.  Once for a weight; bound by reading its codes.
__global__ void __launch_bounds__(256)
w4_row_exp_kernel(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ exps,
                  unsigned char* __restrict__ row_exp, int N, int groups) {
  const int lane = threadIdx.x & 63;
  const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (n >= N) return;
  int most = 0, least = 255, no_scale = 0;
  for (int g = lane; g < groups; g += 64) {
    const long at = (long)n * groups + g;
    u32x4 c;
    __builtin_memcpy(&c, codes + 16 * at, 16);      // of any alignment
    const int e = exps[at];
    const bool there = ((c[0] | c[1] | c[2] | c[3]) & 0x77777777u) != 0;
    most = max(most, there ? e : 0);
    least = min(least, there ? e : 255);
    no_scale |= e == 255;
  }
#pragma unroll
  for (int by = 32; by > 0; by >>= 1) {
    most = max(most, __shfl_xor(most, by));
    least = min(least, __shfl_xor(least, by));
    no_scale |= __shfl_xor(no_scale, by);
  }
  if (lane == 0) row_exp[n] = no_scale || most - least > SPAN ? FAR : most;
}

// One output of such a row, by a wave: a sum in fp32 for each group, a lane a
// group, at its scale, and their sum.
template <typename T> DEVINL float far_output(const T* x, const Args& a, int m, int n) {
  const unsigned char* codes = a.codes + (long)n * (a.K >> 1);
  const unsigned char* exps = a.exps + (long)n * (a.K >> 5);
  x += m * a.ldx;
  float sum = 0.f;
#pragma unroll 1
  for (int k = 32 * (threadIdx.x & 63); k < a.K; k += 32 * 64) {
    const int e = exps[k >> 5];
    float s = 0.f;
#pragma unroll 1
    for (int i = k; i < k + 32; i += 8) {
      const unsigned c = *reinterpret_cast<const unsigned*>(codes + (i >> 1));
      const VecT<T, 8> v = vload<T, 8>(x + i);
      auto two = [&](auto w, int at) {
        s = fmaf(DT<T>::to_f32(v.data[at]), w[0], s);
        s = fmaf(DT<T>::to_f32(v.data[at + 1]), w[1], s);
      };
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 0), 0);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 1), 2);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 2), 4);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.f, 3), 6);
    }
    sum += e == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(s, e - 127);
  }
  return wave_reduce_sum(sum);
}

// The outputs (m, n) of the lanes that are `mine`, one after the other.  Every lane
// of the wave calls it.
template <typename T> DEVINL void far_outputs(bool mine, const T* x, T* y, const Args& a, int m, int n) {
  unsigned long long todo = __ballot(mine);
#pragma unroll 1
  while (todo) {
    const int from = __builtin_ctzll(todo);
    todo &= todo - 1;
    const int mm = __builtin_amdgcn_readlane(m, from), nn = __builtin_amdgcn_readlane(n, from);
    const float sum = far_output(x, a, mm, nn);
    if ((int)(threadIdx.x & 63) == from) y[(long)mm * a.N + nn] = DT<T>::from_f32(sum);
  }
}

// The block's waves hold sums over parts of K, each for the 16 * NT outputs from
// n0 - lane%16 on: added through LDS in wave order (the same sum every time) and
// stored.  D layout: column n = lane%16, row m = 4*(lane/16) + r.
template <typename T, int NT, int WAVES>
DEVINL void add_waves(f32x4 (*part)[NT][64], const f32x4* acc, int n0, const T* x, T* y, const Args& a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < NT; ++u) part[wave][u][lane] = acc[u];
  __syncthreads();
  for (int u = wave; u < NT; u += WAVES) {
    const int n = n0 + 16 * u;
    f32x4 s = part[0][u][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) {
      const f32x4 p = part[v][u][lane];
#pragma unroll
      for (int r = 0; r < 4; ++r) s[r] += p[r];
    }
    const int row_e = a.row_exp[min(n, a.N - 1)];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int m = 4 * (lane >> 4) + r;
      if (m < a.M && n < a.N) y[(long)m * a.N + n] = DT<T>::from_f32(at_row_scale<T>(s[r], row_e));
    }
    if (__any(row_e == FAR)) {
#pragma unroll 1
      for (int r = 0; r < 4; ++r) {
        const int m = 4 * (lane >> 4) + r;
        far_outputs(row_e == FAR && n < a.N && m < a.M, x, y, a, m, n);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Up to 16 rows, x straight from the caches: one wave owns 16*NT outputs and
// every WAVES-th 128-wide piece of K, the next piece's weights and x on their
// way while this one is multiplied.  NT tiles of outputs share a wave's x: as few
// as leave at most 256 workgroups, one a CU, and four beyond.  A call with 16 rows
// and K = 2048 takes with one, two and four tiles 5.5, 5.9 and 7.9 us for 4096
// outputs; 7.6, 5.9 and 7.9 for 4608; 7.8, 6.0 and 7.9 for 8192; 10.3, 9.5 and 8.0
// for 8704; 19.4, 14.0 and 14.1 for 20480; 27.1, 17.9 and 14.3 for 32128.
// ---------------------------------------------------------------------------
template <typename T, int NT, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
w4_few_rows(const T* __restrict__ x, T* __restrict__ y, Args a) {
  using vec = typename Frag<T>::vec;
  __shared__ f32x4 part[WAVES][NT][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c16 = lane & 15;
  const int n0 = blockIdx.x * (16 * NT) + c16;
  int row_e[NT];
  const unsigned char *crow[NT], *erow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min(n0 + 16 * t, a.N - 1);      // the last row again: not stored
    row_e[t] = a.row_exp[n];
    crow[t] = a.codes + (long)n * (a.K >> 1);
    erow[t] = a.exps + (long)n * (a.K >> 5);
  }

  struct Piece {
    u32x4 w[NT], x[4];
    int e[NT];
  };
  auto load = [&](int k0) {
    Piece p;
    const int k = k0 + 32 * g;                    // K is a multiple of 32
    const bool k_ok = k < a.K;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      p.w[t] = u32x4{0u, 0u, 0u, 0u};
      p.e[t] = 127;
      if (k_ok) {
        p.w[t] = *reinterpret_cast<const u32x4*>(crow[t] + (k >> 1));
        p.e[t] = erow[t][k >> 5];
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p.x[i] = u32x4{0u, 0u, 0u, 0u};
      if (k_ok && c16 < a.M) p.x[i] = *reinterpret_cast<const u32x4*>(x + c16 * a.ldx + k + 8 * i);
    }
    return p;
  };

  f32x4 acc[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  Piece next = load(wave * 128);
  for (int k0 = wave * 128; k0 < a.K; k0 += WAVES * 128) {
    const Piece p = next;
    if (k0 + WAVES * 128 < a.K) next = load(k0 + WAVES * 128);
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const float scale = group_scale<T>(p.e[u], row_e[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[u] = Frag<T>::mfma(__builtin_bit_cast(vec, p.x[i]), decode8<T>(p.w[u][i], scale), acc[u]);
    }
  }
  add_waves<T, NT, WAVES>(part, acc, n0, x, y, a);
}

// Elements of a row of x in LDS: zeros behind K as far as a wave's pieces reach
// (a repeated infinity would meet a weight of 0), and 16 bytes between rows.
__host__ __device__ constexpr int lds_row(int K) { return (K + 255) / 256 * 256 + 8; }

// The same with x in LDS, for few enough rows that a workgroup's copy is small
// beside its weights: of the 64 lanes that the matrix instruction has for x only
// M in 16 hold a row (the others repeat the last; their sums are not stored),
// and fetching those from the caches takes as many memory instructions as the
// weights.  One row by 20480 x 4096: 12.0 us (3.7 TB/s), 17 with x from the caches;
// by 10240 x 2048 a call with 4 rows takes 6.2 us, 7.2 with x from the caches, with
// 8 rows 7.3 and 7.5, with 12 rows 10.2 and 7.7.
// U pieces of 128 lie next to each other.  Eight waves of one piece, but four of
// two for many outputs and a K under 1024, of which either takes all at once and
// more, smaller workgroups fill the CUs better: one row by 32128 x 768 5.0 us (6.0
// with eight waves), 8 rows 6.9 (7.2), one by 50257 x 768 7.7 (8.0); by 18432 x 768
// 5.5 and 5.4; by 32128 x 1024 6.9 and 6.8, x 2048 10.7 and 10.4, with 8 rows x 2304
// 19.6 and 16.3.
// Registers are held to what leaves room for all 8 waves of a SIMD.
template <typename T, int NT, int U, int WAVES>
__global__ void __launch_bounds__(WAVES * 64, 8)
w4_lds_rows(const T* __restrict__ x, T* __restrict__ y, Args a) {
  using vec = typename Frag<T>::vec;
  __shared__ f32x4 part[WAVES][NT][64];
  extern __shared__ u32x4 shared[];
  T* xs = reinterpret_cast<T*>(shared);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c16 = lane & 15;
  const int n0 = blockIdx.x * (16 * NT) + c16;
  static_assert(U <= 2, "lds_row()");
  const int LD = lds_row(a.K);
  int row_e[NT];
  const unsigned char *crow[NT], *erow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min(n0 + 16 * t, a.N - 1);      // the last row again: not stored
    row_e[t] = a.row_exp[n];
    crow[t] = a.codes + (long)n * (a.K >> 1);
    erow[t] = a.exps + (long)n * (a.K >> 5);
  }
  struct Piece {
    u32x4 w[U][NT];
    int e[U][NT];
  };
  auto load = [&](int k0) {
    Piece p;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = k0 + 128 * j + 32 * g;          // K is a multiple of 32
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        p.w[j][t] = u32x4{0u, 0u, 0u, 0u};
        p.e[j][t] = 127;
        if (k < a.K) {
          p.w[j][t] = *reinterpret_cast<const u32x4*>(crow[t] + (k >> 1));
          p.e[j][t] = erow[t][k >> 5];
        }
      }
    }
    return p;
  };
  constexpr int RUN = WAVES * 128 * U;
  Piece next = load(wave * 128 * U);
  for (int i = threadIdx.x * 8; i < a.M * LD; i += WAVES * 64 * 8) {
    const int m = i / LD, k = i - m * LD;
    u32x4 v = u32x4{0u, 0u, 0u, 0u};
    if (k < a.K) v = *reinterpret_cast<const u32x4*>(x + m * a.ldx + k);
    *reinterpret_cast<u32x4*>(xs + i) = v;
  }
  __syncthreads();
  f32x4 acc[NT];
#pragma unroll
  for (int u = 0; u < NT; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T* xrow = xs + min(c16, a.M - 1) * LD;
  for (int k0 = wave * 128 * U; k0 < a.K; k0 += RUN) {
    const Piece p = next;
    if (k0 + RUN < a.K) next = load(k0 + RUN);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int k = k0 + 128 * j + 32 * g;
      float scale[NT];
#pragma unroll
      for (int u = 0; u < NT; ++u) scale[u] = group_scale<T>(p.e[j][u], row_e[u]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const vec xf = *reinterpret_cast<const vec*>(xrow + k + 8 * i);
#pragma unroll
        for (int u = 0; u < NT; ++u)
          acc[u] = Frag<T>::mfma(xf, decode8<T>(p.w[j][u][i], scale[u]), acc[u]);
      }
    }
  }
  add_waves<T, NT, WAVES>(part, acc, n0, x, y, a);
}

// ---------------------------------------------------------------------------
// Many rows: a workgroup of 2 x WN waves makes 32*MT rows by 16*NT*WN outputs.
// x goes through LDS, 128 of K at a time in two buffers (two pieces are on
// their way in registers while one is multiplied); weights go from memory to
// registers as above, converted once for MT tiles of rows.  LDS holds the 32 k
// of a lane group as a plane of its own, rows 80 bytes apart and planes a
// multiple of 256: sixteen rows at one k are in different banks, in whichever
// lane groups the hardware takes them.
// 256 rows by 10240 x 2048 take 25, 34 and 53 us in tiles of 128 x 128, 64 x 64 and
// 32 x 32, by 4096 x 768 11, 6.6 and 9.5 us, by 768 x 2048 23, 12 and 8.9 us (the
// library on 16-bit weights: 23, 6.8 and 8.4 us).  Which it is follows from rounds
// of workgroups on the 256 CUs; of each border both sides, in us a call:
//  - 128 x 128 for over 64 rows and over 512 tiles of 64 x 64.  256 rows by 8448 x
//    2048 25.6 (64 x 64: 34.8), by 8192 x 2048 24.6 (23.9); 96 rows by 32128 x 768
//    12.9 (18.1), 64 rows by 40000 x 768 21.9 (15.8).
//  - 64 x 64 for over 32 rows and over 128 tiles.  256 rows by 2560 x 2048 13.1 (32 x
//    32: 17.4), by 2048 x 2048 13.0 (12.5); 33 rows by 10240 x 2048 13.6 (18.0),
//    32 rows 13.4 (12.5).
//  - Up to 128 tiles of 64 x 64 and K from 4096: they share K, in runs of 512 and
//    more, and a second kernel adds their fp32 sums in order.  64 rows by 4096 x
//    10240 24.2 (32 x 32: 42.5), 256 by 2048 x 4096 18.4 (21.5); 192 by 4096 x 4096,
//    192 tiles, 29.9 (64 x 64: 24.6); 64 by 4096 x 2816 10.9 (10.5).
// Four waves of 64 x 64 read half as much LDS as eight of 64 x 32, but 30 us, one
// for each SIMD, is more than 25.
// ---------------------------------------------------------------------------
template <typename T, int MT, int NT, int WN>
__global__ void __launch_bounds__(128 * WN)
w4_many_rows(const T* __restrict__ x, T* __restrict__ y, float* __restrict__ part, int run, Args a) {
  using vec = typename Frag<T>::vec;
  constexpr int THREADS = 128 * WN, BM = 32 * MT, BN = 16 * NT * WN, KC = 128;
  constexpr int LD = 40, PLANE = BM * LD;         // elements: a row of 32 k, 32 k of all rows
  constexpr int LOADS = BM * KC / 8 / THREADS;       // 16-byte pieces of x a thread brings
  __shared__ alignas(256) T lds[2][4 * PLANE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c16 = lane & 15;
  const int wm = wave & 1, wn = wave >> 1;
  const int k_at = blockIdx.z * run, k_end = min(k_at + run, a.K);   // this workgroup's part of K
  const int m_at = blockIdx.x * BM, n0 = blockIdx.y * BN + wn * 16 * NT + c16;
  int row_e[NT];
  const unsigned char *crow[NT], *erow[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int n = min(n0 + 16 * t, a.N - 1);      // the last row again: not stored
    row_e[t] = a.row_exp[n];
    crow[t] = a.codes + (long)n * (a.K >> 1);
    erow[t] = a.exps + (long)n * (a.K >> 5);
  }
  // Loads carry no condition, so that the compiler can count them and wait for
  // no younger ones: addresses are clamped, what they are clamped for becomes 0
  // where it is used.
  struct Piece {
    u32x4 x[LOADS], w[NT];
    int e[NT];
  } ahead[2];
  // piece p of x: 8 of k at 8 * (p % 4) of row p / 4 % BM of plane p / (4 * BM)
  const int xrow = threadIdx.x / 4 % BM, xk = threadIdx.x % 4 * 8;
  const T* xat = x + min(m_at + xrow, a.M - 1) * a.ldx;
  static_assert(THREADS % (4 * BM) == 0, "the same row for all of a thread's pieces");
  auto plane = [&](int i) { return (int)(threadIdx.x + THREADS * i) / (4 * BM); };
  auto load = [&](Piece& p, int k0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      p.x[i] = *reinterpret_cast<const u32x4*>(xat + min(k0 + 32 * plane(i) + xk, a.K - 8));
    const int kk = min(k0 + 32 * g, a.K - 32);      // K is a multiple of 32
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      p.w[t] = *reinterpret_cast<const u32x4*>(crow[t] + (kk >> 1));
      p.e[t] = erow[t][kk >> 5];
    }
  };
  auto stage = [&](const Piece& p, int k0, int buf) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const unsigned keep = k0 + 32 * plane(i) < k_end ? 0xffffffffu : 0u;
      *reinterpret_cast<u32x4*>(&lds[buf][plane(i) * PLANE + xrow * LD + xk]) = p.x[i] & keep;
    }
  };
  // orders LDS alone: a plain barrier would wait for the loads on their way
  auto lds_barrier = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  };

  f32x4 acc[MT][NT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < NT; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};

  // multiplies the piece in `buf`, whose weights are in `now`, while that after
  // the next is loaded
  auto step = [&](int k0, Piece& now, const Piece& next, int buf) {
    const unsigned keep = k0 + 32 * g < k_end ? 0xffffffffu : 0u;
    u32x4 w[NT];
    float scale[NT];
#pragma unroll
    for (int u = 0; u < NT; ++u) { w[u] = now.w[u] & keep; scale[u] = group_scale<T>(now.e[u], row_e[u]); }
    load(now, k0 + 2 * KC);
    const T* row = &lds[buf][g * PLANE + (wm * 16 * MT + c16) * LD];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      vec xf[MT];
#pragma unroll
      for (int t = 0; t < MT; ++t) xf[t] = *reinterpret_cast<const vec*>(row + 16 * t * LD + 8 * i);
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const vec wf = decode8<T>(w[u][i], scale[u]);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t][u] = Frag<T>::mfma(xf[t], wf, acc[t][u]);
      }
    }
    stage(next, k0 + KC, buf ^ 1);
    lds_barrier();
  };
  load(ahead[0], k_at);
  load(ahead[1], k_at + KC);
  stage(ahead[0], k_at, 0);
  lds_barrier();
  // in pairs; of an odd number of pieces the last is multiplied by zeros
  for (int k0 = k_at; k0 < k_end; k0 += 2 * KC) {
    step(k0, ahead[0], ahead[1], 0);
    step(k0 + KC, ahead[1], ahead[0], 1);
  }
#pragma unroll
  for (int u = 0; u < NT; ++u) {
    const int n = n0 + 16 * u;
    if (n >= a.N) continue;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int m = m_at + wm * 16 * MT + 16 * t + 4 * g + r;
        if (m >= a.M) continue;
        if (part) part[((long)blockIdx.z * a.M + m) * a.N + n] = acc[t][u][r];
        else y[(long)m * a.N + n] = DT<T>::from_f32(at_row_scale<T>(acc[t][u][r], row_e[u]));
      }
  }
  bool far = false;
#pragma unroll
  for (int u = 0; u < NT; ++u) far |= row_e[u] == FAR;
  if (__any(far) && !part) {                        // w4_add_parts makes them otherwise
#pragma unroll 1
    for (int i = 0; i < 4 * NT * MT; ++i) {
      const int n = n0 + 16 * (i / (4 * MT)), m = m_at + wm * 16 * MT + 16 * (i / 4 % MT) + 4 * g + i % 4;
      far_outputs(n < a.N && m < a.M && a.row_exp[min(n, a.N - 1)] == FAR, x, y, a, m, n);
    }
  }
}

// The sum over parts of K, in their order, and the rows' scales.
template <typename T>
__global__ void __launch_bounds__(256)
w4_add_parts(const T* __restrict__ x, const float* __restrict__ part, T* __restrict__ y, int parts, Args a) {
  const long mn = (long)a.M * a.N, i = (long)blockIdx.x * 256 + threadIdx.x;
  const bool there = i < mn;
  const int m = there ? i / a.N : 0, n = there ? i - (long)m * a.N : 0, row_e = a.row_exp[n];
  if (there) {
    float s = 0.f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) s += part[p * mn + i];
    y[i] = DT<T>::from_f32(at_row_scale<T>(s, row_e));
  }
  far_outputs(there && row_e == FAR, x, y, a, m, n);
}

}  // namespace

torch::Tensor w4_row_exp(torch::Tensor codes, torch::Tensor exps) {
  VALUE_CHECK(codes.dim() == 2 && exps.dim() == 2 && codes.size(0) == exps.size(0) &&
                  codes.size(1) == 16 * exps.size(1) && exps.size(1) < (1L << 25) &&
                  fits_a_launch((codes.size(0) + 3) / 4, 256),
              "w4_row_exp: codes (N,K/2) and exponents (N,K/32), got ", codes.sizes(), " and ", exps.sizes());
  for (const auto* t : {&codes, &exps})
    VALUE_CHECK(t->scalar_type() == torch::kByte && t->is_contiguous() && t->is_cuda() &&
                    t->device() == codes.device(),
                "w4_row_exp: contiguous uint8 tensors of one GPU");
  c10::DeviceGuard guard(codes.device());
  auto row_exp = at::empty({codes.size(0)}, exps.options());
  if (codes.size(0) == 0) return row_exp;
  hipLaunchKernelGGL(w4_row_exp_kernel, dim3((codes.size(0) + 3) / 4), dim3(256), 0,
                     at::hip::getCurrentHIPStream().stream(), codes.data_ptr<unsigned char>(),
                     exps.data_ptr<unsigned char>(), row_exp.data_ptr<unsigned char>(),
                     (int)codes.size(0), (int)exps.size(1));
  HIP_CHECK_KERNEL();
  return row_exp;
}

torch::Tensor w4_linear(torch::Tensor x, torch::Tensor codes, torch::Tensor exps,
                        torch::Tensor row_exp) {
  NO_GRAD_CHECK(x, "linear_w4");
  VALUE_CHECK(codes.dim() == 2 && exps.dim() == 2 && row_exp.dim() == 1,
              "linear_w4: codes (N,K/2), exps (N,K/32), row_exp (N)");
  const long N = codes.size(0), K = 2 * codes.size(1);
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) == K && K > 0, "linear_w4: x ", x.sizes(),
              ", the weight has ", K, " inputs");
  VALUE_CHECK(K % 32 == 0 && exps.size(0) == N && exps.size(1) * 32 == K && row_exp.size(0) == N,
              "linear_w4: codes ", codes.sizes(), " and exponents ", exps.sizes(), " do not match");
  for (const auto* t : {&codes, &exps, &row_exp})
    VALUE_CHECK(t->scalar_type() == torch::kByte && t->is_contiguous() && t->device() == x.device(),
                "linear_w4: codes and exponents must be contiguous uint8 on x's device, ",
                x.device(), ", got ", t->device());
  VALUE_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0,
              "linear_w4: codes must be 16-byte aligned");
  VALUE_CHECK(x.scalar_type() == torch::kBFloat16 || x.scalar_type() == torch::kHalf,
              "linear_w4 takes bf16 or fp16 on a GPU, got ", x.scalar_type());
  c10::DeviceGuard guard(x.device());
  const long M = x.numel() / K;
  // tiles of 32 rows take 256 threads and of 64 rows 512; a grid's second dimension, of
  // tiles of 32 outputs and more, is 16 bits wide
  VALUE_CHECK(fits_a_launch((M + 31) / 32, 256) && N < 65535L * 32 && K < (1L << 30),
              "linear_w4: too large: ", M, " rows of ", K, " by ", N);
  auto sizes = x.sizes().vec();
  sizes.back() = N;
  auto y = at::empty(sizes, x.options().memory_format(at::MemoryFormat::Contiguous));
  if (x.dim() != 2) x = x.reshape({-1, K});
  if (M == 0 || N == 0) return y;
  // rows of x are read 16 bytes at a time
  if (x.stride(1) != 1 || (M > 1 && x.stride(0) % 8 != 0) ||
      reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0)
    x = x.clone(at::MemoryFormat::Contiguous);
  auto stream = at::hip::getCurrentHIPStream().stream();
  const Args a{codes.data_ptr<unsigned char>(), exps.data_ptr<unsigned char>(),
               row_exp.data_ptr<unsigned char>(), (int)M, (int)N, (int)K, (long)x.stride(0)};
  auto go = [&](auto tag) {
    using T = decltype(tag);
    const auto up = [](long n, long by) { return (n + by - 1) / by; };
    auto launch = [&](auto kernel, dim3 grid, int threads, long lds, auto... more) {
      hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, stream, (const T*)x.data_ptr(),
                         (T*)y.data_ptr(), more..., a);
    };
    auto many = [&](auto kernel, dim3 grid, int threads, long parts) {
      const long run = up(up(K, parts), 128) * 128;
      parts = up(K, run);
      grid.z = parts;
      torch::Tensor part;
      if (parts > 1) part = at::empty({parts * M * N}, x.options().dtype(torch::kFloat));
      float* p = parts > 1 ? part.data_ptr<float>() : nullptr;
      launch(kernel, grid, threads, 0, p, (int)run);
      if (parts > 1)
        hipLaunchKernelGGL(w4_add_parts<T>, dim3(up(M * N, 256)), dim3(256), 0, stream,
                           (const T*)x.data_ptr(), p, (T*)y.data_ptr(), (int)parts, a);
    };
    const auto tiles = [&](long t) { return dim3(up(M, t), up(N, t)); };
    const auto count = [](dim3 d) { return (long)d.x * d.y; };
    const long copy = M * lds_row(K) * 2;           // x in LDS
    // What bounds a launch is rounds of workgroups on the 256 CUs; the borders, with
    // both sides of each, are at the kernels.
    if (M <= 8 && copy <= 56 * 1024) {
      if (N >= 20480 && K < 1024) launch(w4_lds_rows<T, 1, 2, 4>, dim3(up(N, 16)), 256, copy);
      else launch(w4_lds_rows<T, 1, 1, 8>, dim3(up(N, 16)), 512, copy);
    } else if (M <= 16) {
      if (N <= 4096) launch(w4_few_rows<T, 1, 8>, dim3(up(N, 16)), 512, 0);
      else if (N <= 8192) launch(w4_few_rows<T, 2, 8>, dim3(up(N, 32)), 512, 0);
      else launch(w4_few_rows<T, 4, 8>, dim3(up(N, 64)), 512, 0);
    } else if (M > 64 && count(tiles(64)) > 512) {
      many(w4_many_rows<T, 4, 2, 4>, tiles(128), 512, 1);
    } else if (K >= 4096 && count(tiles(64)) <= 128) {
      many(w4_many_rows<T, 2, 1, 4>, tiles(64), 512, std::min(up(256, count(tiles(64))), K / 512));
    } else if (M > 32 && count(tiles(64)) > 128) {
      many(w4_many_rows<T, 2, 1, 4>, tiles(64), 512, 1);
    } else {
      many(w4_many_rows<T, 1, 1, 2>, tiles(32), 256, 1);
    }
  };
  if (x.scalar_type() == torch::kBFloat16) go(__hip_bfloat16());
  else go(__half());
  HIP_CHECK_KERNEL();
  return y;
}
