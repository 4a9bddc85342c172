// One token per row of logits from a given uniform number, after temperature,
// top-k, top-p and min-p.
//
//   w_i = exp((x_i - max)/T);  order: x descending, ties by index ascending
//   K = the first k;  P = the shortest prefix of K with sum w >= top_p * sum_K w
//   A = those of P with w >= min_p;  the lowest i of A, in index order, whose
//   running sum is over u * sum_A w
//
// Every cut is a prefix of ONE order, so the kept set is "everything up to a
// border element (value, index)" and nothing is sorted: a histogram over the
// distance from the maximum gives the border's bin, the bin's few elements are
// ranked against each other, and the kept ones - usually some hundred - go to a
// list in LDS that the later steps work on.  If they do not fit, the later
// steps run over the row again with the border as a filter.
//
// A token is a comparison of a sum with as many borders as there are logits:
// an error e in the cumulative share moves a row's token with a probability of
// about 2 V e, one row in 150 in fp32 at V = 32128.  So weights are computed in
// fp64 (the table-driven exponential after Tang: 2^(j/32) from a table and the
// Taylor polynomial of degree 5 for what is left; relative error under 1e-14 and
// that of (x - max)/T) and summed as integers w * 2^44: exact, in any order, hence
// atomics whose order does not matter.  A weight under 2^-45 counts as none.
//
// One workgroup a row; the row is read from memory once, and a few times from
// the L2 after that.  What bounds it is one CU's instruction rate (an
// instruction for every logit of a 32128 row is 0.2 us; a weight is about 20 of
// them, 7 us a row) and, for a small top-k, the latency of its dozen steps.
// One row of 32128 with top-k 50 and top-p 10 us; 256 rows, nucleus sampling,
// 26 us (reading them: 3.3 us): the maximum 6.3, weights and histogram 9.0, the list
// 4.3, the border 2.2, sums and drawing 4.1; 33 rows of 50257 in fp32, top-k 100 to
// 300, 17 us: 5.8, listing and ranking 10.3, drawing 1.2; 52647 logits with a nucleus
// of some 10000, the longest path, 62 us.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "../common.h"

namespace {

typedef unsigned long long u64;
typedef __attribute__((ext_vector_type(8))) float f32x8;

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2 * THREADS;
constexpr int CAP = THREADS;             // elements ranked against each other at once
constexpr int LIST = 4 * THREADS;        // kept elements that the list holds
constexpr int SHORT = 192;               // lists up to this are summed pair by pair
constexpr int FEW = 512;                 // a top-k up to this is found without a histogram of the row
constexpr int MAX_V = 1 << 19;           // sums of w * 2^44 stay under 2^63
constexpr int SEG = 512;                 // logits of a segment: a wave's 64 slots of 8
constexpr int SEGS = MAX_V / SEG;
constexpr double ONE = 17592186044416.0; // 2^44
constexpr int TABLE = 32;              // 8 bytes each: one for every pair of LDS banks

struct Opt {                             // a number for all rows, or one each
  const void* each;
  double all;
  bool wide;                             // fp64 ones
  DEVINL double f(int row) const {
    return !each ? all : wide ? ((const double*)each)[row] : (double)((const float*)each)[row];
  }
  DEVINL int i(int row) const { return each ? ((const int*)each)[row] : (int)all; }
};

// The bits of 2^44 * 2^(j/32), correctly rounded, less j << 47: with n << 47
// added for n = 32 i + j, what stays of it is i in the exponent field.
__constant__ const u64 EXP2_TABLE[TABLE] = {
    0x42b0000000000000ull, 0x42afd9b0d3158574ull, 0x42afb5586cf9890full, 0x42af9301d0125b51ull,
    0x42af72b83c7d517bull, 0x42af54873168b9aaull, 0x42af387a6e756238ull, 0x42af1e9df51fdee1ull,
    0x42af06fe0a31b715ull, 0x42aef1a7373aa9cbull, 0x42aedea64c123422ull, 0x42aece086061892dull,
    0x42aebfdad5362a27ull, 0x42aeb42b569d4f82ull, 0x42aeab07dd485429ull, 0x42aea47eb03a5585ull,
    0x42aea09e667f3bcdull, 0x42ae9f75e8ec5f74ull, 0x42aea11473eb0187ull, 0x42aea589994cce13ull,
    0x42aeace5422aa0dbull, 0x42aeb737b0cdc5e5ull, 0x42aec49182a3f090ull, 0x42aed503b23e255dull,
    0x42aee89f995ad3adull, 0x42aeff76f2fb5e47ull, 0x42af199bdd85529cull, 0x42af3720dcef9069ull,
    0x42af5818dcfba487ull, 0x42af7c97337b9b5full, 0x42afa4afa2a490daull, 0x42afd0765b6e4540ull,
};

// A larger float has a larger key; with the index: one order over all elements
// of a row, larger first, then the lower index.  -0 becomes 0: they are equal.
DEVINL u64 rank_key(float x, int idx) {
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  return (u64)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (unsigned)~idx;
}
DEVINL float value_of(u64 key) {
  const unsigned u = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
DEVINL int index_of(u64 key) { return (int)~(unsigned)key; }

// exp((x - max)/T) * 2^44 as an integer.  y = (x - max) * 32/(T ln2) = n + f,
// 2^(y/32) = 2^(n/32) * e^(f ln2/32) with |f| <= 1/2.
struct Weights {
  double max, slope;
  const u64* table;
  // the integer in the low 52 bits, under the exponent field of 2^52
  DEVINL u64 raw(float x) const {
    // what is under 2^-46, and NaN, becomes 2^-47 here and 0 in the integer
    const double y = fmax(((double)x - max) * slope, -47.0 * TABLE);
    // added to 1.5 * 2^52, y is rounded to the integer in the low bits
    const double magic = 6755399441055744.0;
    const double rounded = y + magic;
    const int n = (int)__builtin_bit_cast(u64, rounded);
    const double f = y - (rounded - magic);
    double p = __builtin_fma(f, 3.973709984549416e-11, 9.172562701824643e-09);
    p = __builtin_fma(p, f, 1.693850972437182e-06);
    p = __builtin_fma(p, f, 0.0002345961982022468);
    p = __builtin_fma(p, f, 0.02166084939249829);
    p = __builtin_fma(p, f, 1.0);
    const u64 base = table[n & (TABLE - 1)] + ((u64)(unsigned)n << 47);
    // added to 2^52, the weight is rounded to the integer in the low bits
    return __builtin_bit_cast(u64, __builtin_fma(p, __builtin_bit_cast(double, base), 4503599627370496.0));
  }
  DEVINL u64 of(float x) const { return raw(x) & 0xfffffffffffffull; }
};

// A row of at least 8 logits in slots of 8.  The last slot is read from V - 8:
// what it repeats of the one before is taken as -inf.  NaN is let through: it
// is not the larger of two, not at least anything, and weighs nothing.  Rows need not
// be aligned (a 16-byte load at an element's alignment is legal here).  A pass
// reads the row anew; after the first it comes from the L2.
template <typename T> struct Row {
  const T* p;
  int V;
  bool only_inf;       // the maximum is +inf: those count as 0, others as -inf

  DEVINL int slots() const { return (V + 7) / 8; }
  DEVINL int first(int q) const { return min(q * 8, V - 8); }   // of slot q
  DEVINL float at(int i) const {
    const float x = DT<T>::to_f32(p[i]);
    return !only_inf ? x : x == INFINITY ? 0.f : -INFINITY;
  }
  struct Raw { T v[8]; };
  DEVINL Raw fetch(int q) const {
    Raw r;
    __builtin_memcpy(r.v, p + first(q), sizeof(r.v));
    return r;
  }
  DEVINL f32x8 take8(const Raw& r, int q) const {
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = DT<T>::to_f32(r.v[e]);
    if (only_inf) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] == INFINITY ? 0.f : -INFINITY;
    }
    if (q * 8 > V - 8) {
      const int skip = q * 8 - (V - 8);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = e < skip ? -INFINITY : x[e];
    }
    return x;
  }
  // f(8 logits, slot) for this thread's slots.  Every thread makes the same
  // number of calls; slots from slots() on are -inf.  each4: a call is cheap,
  // four slots are loaded at a time; each1: it is not, the next is on its way.
  template <typename F> DEVINL void each4(F f) const {
    const int n = (slots() + THREADS - 1) / THREADS;
#pragma unroll 1
    for (int i = 0; i < n; i += 4) {
      Raw r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) r[j] = fetch(threadIdx.x + (i + j) * THREADS);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = threadIdx.x + (i + j) * THREADS;
        f(take8(r[j], q), q);
      }
    }
  }
  template <typename F> DEVINL void each1(F f) const {
    const int n = (slots() + THREADS - 1) / THREADS;
    Raw next = fetch(threadIdx.x);
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int q = threadIdx.x + i * THREADS;
      const Raw r = next;
      next = fetch(q + THREADS);
      f(take8(r, q), q);
    }
  }
  DEVINL unsigned bits_from(f32x8 x, float low, float high) const {
    unsigned bits = 0;
    low = fmaxf(low, -3.402823466e38f);
#pragma unroll
    for (int e = 0; e < 8; ++e) bits |= x[e] >= low && x[e] <= high ? 1u << e : 0u;
    return bits;
  }
  // f(x, index) for the few elements from `low` to `high`
  template <typename F> DEVINL void each_from(float low, float high, F f) const {
    each1([&](f32x8 x, int q) {
      unsigned bits = bits_from(x, low, high);
#pragma unroll 1
      while (bits) {
        const int b = __builtin_ctz(bits);
        bits &= bits - 1;
        f(pick(x, b), first(q) + b);
      }
    });
  }
  static DEVINL float pick(f32x8 x, int b) {
    float v = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) v = b == e ? x[e] : v;
    return v;
  }
};

// Inclusive sum over the lanes, in six steps along the row (no LDS).
template <int CTRL, int ROWS> DEVINL int moved(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> DEVINL u64 moved(u64 x) {
  const unsigned lo = moved<CTRL, ROWS>((int)(unsigned)x);
  const unsigned hi = moved<CTRL, ROWS>((int)(unsigned)(x >> 32));
  return (u64)hi << 32 | lo;
}
template <typename I> DEVINL I wave_scan(I x) {
  x += moved<0x111, 0xf>(x);             // from the lane 1, 2, 4, 8 before, in rows of 16
  x += moved<0x112, 0xf>(x);
  x += moved<0x114, 0xf>(x);
  x += moved<0x118, 0xf>(x);
  x += moved<0x142, 0xa>(x);             // lane 15 of a row to the next row
  x += moved<0x143, 0xc>(x);             // lane 31 to the upper half
  return x;
}
DEVINL u64 last_lane(u64 x) {
  const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)x, 63);
  const unsigned hi = __builtin_amdgcn_readlane((int)(unsigned)(x >> 32), 63);
  return (u64)hi << 32 | lo;
}
DEVINL int last_lane(int x) { return __builtin_amdgcn_readlane(x, 63); }
template <typename I> DEVINL I wave_sum(I x) { return last_lane(wave_scan(x)); }

struct Shared {
  u64 hist[BINS];
  u64 cand_k[CAP], cand_w[CAP], sum[CAP];
  u64 list_k[LIST];
  union { u64 list_w[LIST]; int list_i[LIST]; };
  u64 seg[SEGS], last[SEG];
  u64 wave_tot[WAVES];
  u64 table[TABLE];
  float red[2][WAVES];
  u64 found_before, border, last_want;
  int found_bin, cand_n, list_n, last_seg, greedy;
};

// The first bin with whose elements the running sum, from `outer`, reaches what
// a cut needs: leaves it and what lies before it in s.found_*, or -1.
// `need(total)` gives the cut's test for the sum over all, which is `total`, or
// with 0 that of the histogram.  Every thread calls it, after a barrier behind
// the histogram and with s.found_bin at -1; returns the total.
template <typename Need> DEVINL u64 find_bin(Shared& s, u64 outer, u64 total, Need need) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const u64 a = s.hist[2 * t], b = s.hist[2 * t + 1];
  const u64 inc = wave_scan(a + b);
  if (lane == 63) s.wave_tot[wave] = inc;
  __syncthreads();
  u64 before = outer + inc - (a + b), all = outer;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const u64 v = s.wave_tot[w];
    before += w < wave ? v : 0;
    all += v;
  }
  if (!total) total = all;
  const auto reached = need(total);
  // at most one thread has the first bin to reach
  if (!reached(before) && reached(before + a + b)) {
    const bool second = !reached(before + a);
    s.found_bin = 2 * t + second;
    s.found_before = second ? before + a : before;
  }
  __syncthreads();
  return total;
}

// Empties the histogram and the candidates; barriers on both sides.
DEVINL void clear(Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += THREADS) s.hist[i] = 0;
  if (threadIdx.x == 0) { s.cand_n = 0; s.found_bin = -1; }
  __syncthreads();
}

// s.sum[i] = the sum of of(i, j) over all j < n, for n <= CAP elements, in
// integers of type I.  Where n is small, several waves share an element's sum.
// Barriers on both sides.
template <typename I, typename Of> DEVINL void pair_sums(Shared& s, int n, Of of) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  if (t < n) s.sum[t] = 0;
  __syncthreads();
  const int each = (n + 63) / 64;                  // waves for all elements once
  const int parts = WAVES / max(each, 1), part = wave / max(each, 1);
  const int i = (wave - part * each) * 64 + lane;
  const int run = (n + parts - 1) / parts;
  if (part < parts && i < n) {
    I sum = 0;
    const int end = min(n, (part + 1) * run);
#pragma unroll 4
    for (int j = part * run; j < end; ++j) sum += of(i, j);
    if (sum) atomicAdd(&s.sum[i], (u64)sum);
  }
  __syncthreads();
}

// Among the n candidates the one with which the running sum, from `before`,
// reaches.
template <typename Reached> DEVINL u64 rank_candidates(Shared& s, int n, u64 before, Reached reached) {
  const int t = threadIdx.x;
  pair_sums<u64>(s, n, [&](int i, int j) { return s.cand_k[j] > s.cand_k[i] ? s.cand_w[j] : 0; });
  if (t < n) {
    const u64 sum = before + s.sum[t];
    if (!reached(sum) && reached(sum + s.cand_w[t])) s.border = s.cand_k[t];
  }
  __syncthreads();
  return s.border;
}

// A running sum of integers is over u * total exactly if it is over this one;
// the last one always is.
DEVINL u64 last_before(double u, u64 total) {
  const double target = u * (double)total;
  const u64 want = target > 0.0 ? (u64)target : 0;
  return want < total ? want : total - 1;
}

DEVINL void candidate(Shared& s, u64 key, u64 w) {
  const int to = atomicAdd(&s.cand_n, 1);
  if (to < CAP) { s.cand_k[to] = key; s.cand_w[to] = w; }
}

// All elements of at least `low` to the list, as far as it goes: their indices
// first - where a wave's logit goes follows from masks in scalar registers, and
// one that no lane lists costs a comparison - then, a lane each, their keys.
template <typename T> DEVINL void list_from(Shared& s, const Row<T>& row, float low) {
  const int lane = threadIdx.x & 63;
  low = fmaxf(low, -3.402823466e38f);
  row.each4([&](f32x8 x, int q) {
    u64 who[8];
    int all = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      who[e] = __ballot(x[e] >= low);
      all += __popcll(who[e]);
    }
    if (!all) return;
    int to = 0;
    if (lane == 0) to = atomicAdd(&s.list_n, all);
    to = __builtin_amdgcn_readfirstlane(to);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!who[e]) continue;
      const int at = to + (int)__builtin_amdgcn_mbcnt_hi((unsigned)(who[e] >> 32),
                                                         __builtin_amdgcn_mbcnt_lo((unsigned)who[e], 0));
      if (x[e] >= low && at < LIST) s.list_i[at] = row.first(q) + e;
      to += __popcll(who[e]);
    }
  });
  __syncthreads();
  const int n = min(s.list_n, LIST);
  for (int i = threadIdx.x; i < n; i += THREADS) s.list_k[i] = rank_key(row.at(s.list_i[i]), s.list_i[i]);
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const T* __restrict__ logits, long ld, int V, const void* __restrict__ uniform,
              bool uniform_is_double, Opt temperature, Opt top_k, Opt top_p, Opt min_p,
              long empty_token, long* __restrict__ out) {
  __shared__ Shared s;
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  Row<T> row{logits + r * ld, V, false};

  // this thread's largest, the row's, and the smallest of the threads'
  float mine = -INFINITY;
  row.each4([&](f32x8 x, int) {
#pragma unroll
    for (int e = 0; e < 8; ++e) mine = fmaxf(mine, x[e]);
  });
  if (t < TABLE) s.table[t] = EXP2_TABLE[t];
  for (int i = t; i < BINS; i += THREADS) s.hist[i] = 0;
  s.seg[t] = 0;                                     // SEGS of them
  if (t < SEG) s.last[t] = 0;
  if (t == 0) { s.cand_n = s.list_n = 0; s.found_bin = -1; s.greedy = 0x7fffffff; }
  float mx = wave_reduce_max(mine);
  float mn = -wave_reduce_max(mine > -INFINITY ? -mine : -INFINITY);
  if (lane == 0) { s.red[0][wave] = mx; s.red[1][wave] = mn; }
  double temp = temperature.f(r);
  temp = temp > 1e30 ? 1e30 : temp;                 // infinity among a row's options
  const int k = top_k.i(r);
  const double p = top_p.f(r);
  double floor_p = min_p.f(r);
  const double u = uniform_is_double ? ((const double*)uniform)[r] : ((const float*)uniform)[r];
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    mx = fmaxf(mx, s.red[0][w]);
    mn = fminf(mn, s.red[1][w]);
  }
  if (mx == -INFINITY) {
    if (t == 0) out[r] = empty_token;
    return;
  }
  if (mx == INFINITY) {
    row.only_inf = true;
    mx = mn = 0.f;
  }
  if (!(temp > 0.0) || k == 1 || p <= 0.0) {        // the first of the order
    row.each_from(mx, mx, [&](float, int idx) { atomicMin(&s.greedy, idx); });
    __syncthreads();
    if (t == 0) out[r] = s.greedy;
    return;
  }

  // finite, so that the maximum's distance of 0 stays 0: under 1e-300 nothing but
  // the maximum weighs anything either way
  const double slope = 46.16624130844683 / fmax(temp, 1e-300);
  const Weights weight{(double)mx, slope, s.table};
  floor_p = floor_p > 1.0 ? 1.0 : floor_p;          // the maximum always stays
  const u64 min_w = floor_p > 0.0 ? (u64)__builtin_rint(floor_p * ONE) : 0;

  // Bins over the distance from the maximum that matters: the spread of the
  // threads' largest, which a few masked logits do not stretch, or three times
  // it; what is further shares the last bin.  Rounding keeps the order: a bin
  // holds a run of it.
  const float range = fminf(mx - mn, 64.f * fmaxf(1.f, (float)temp));
  const float narrow = range > 0.f ? fminf((float)(BINS - 2) / range, 1e30f) : 0.f;
  float bin_scale = narrow;
  auto bin_of = [&](float x) {
    return (int)fminf((mx - x) * bin_scale, (float)(BINS - 1));
  };
  // a value that is not above any of bins 0..b: one bin more, for its roundings
  auto low_of = [&](int b) {
    return b >= BINS - 2 || !(bin_scale > 0.f) ? -INFINITY : mx - (float)(b + 2) / bin_scale;
  };
  // and one that is not below any of bins b..
  auto high_of = [&](int b) {
    return b < 2 || !(bin_scale > 0.f) ? INFINITY : mx - (float)(b - 1) / bin_scale;
  };

  u64 border = 0;                                   // the last element kept; 0: all are
  bool ordered = false;                             // and top-p is done
  bool listed = false;                              // the list holds all up to the border
  bool counted = false;                             // the histogram was used

  // Leaves border, and the list where what is not behind `bin` fits (all that
  // the cut keeps, and a few more).  Of `bin`, what is not below floor_key and
  // reached() keeps stays.  value(x): what an element adds to the running sum,
  // which is `before` where the bin begins.
  auto cut_in_bin = [&](int bin, u64 before, u64 floor_key, auto value, auto reached) {
    list_from(s, row, low_of(bin));
    listed = s.list_n <= LIST;
    if (listed) {
      const int n = s.list_n;
      for (int i = t; i < n; i += THREADS) {
        const u64 key = s.list_k[i];
        const float x = value_of(key);
        s.list_w[i] = weight.of(x);
        if (bin_of(x) == bin && key >= floor_key) candidate(s, key, value(x));
      }
    } else {
      row.each_from(low_of(bin), high_of(bin), [&](float x, int idx) {
        const u64 key = rank_key(x, idx);
        if (bin_of(x) == bin && key >= floor_key) candidate(s, key, value(x));
      });
    }
    __syncthreads();
    const int n = s.cand_n;
    if (n <= CAP) {
      border = rank_candidates(s, n, before, reached);
      return;
    }
    // Too many share the bin (a flat row, or few distinct values): narrow the
    // border down by 11 bits of the key at a time.
    u64 prefix = 0;
#pragma unroll 1
    for (int shift = 64; shift > 0;) {
      const int up = shift, bits = min(11, shift);
      shift -= bits;
      clear(s);
      row.each_from(low_of(bin), high_of(bin), [&](float x, int idx) {
        const u64 key = rank_key(x, idx);
        if (bin_of(x) != bin || key < floor_key || (up < 64 && (key >> up) != prefix)) return;
        // bin 0 holds the largest
        atomicAdd(&s.hist[(1 << bits) - 1 - (int)(key >> shift & ((1u << bits) - 1))], value(x));
      });
      __syncthreads();
      find_bin(s, before, 0, [&](u64) { return reached; });
      before = s.found_before;
      prefix = prefix << bits | (u64)((1 << bits) - 1 - s.found_bin);
    }
    border = prefix;
  };

  if (k > 0 && k < V) {
    const u64 want = k;
    const auto reached = [want](u64 sum) { return sum >= want; };
    bool done = false;
    if (k <= FEW) {
      // The k-th largest of the threads' largest is a lower bound of the k-th
      // largest: bins behind its own hold nothing of the first k.
      if (mine > -INFINITY && !row.only_inf) atomicAdd(&s.hist[bin_of(mine)], (u64)1);
      __syncthreads();
      find_bin(s, 0, 0, [&](u64) { return reached; });
      // fewer than k threads may hold anything: then no bound
      const int bin = s.found_bin < 0 ? BINS - 1 : s.found_bin;
      list_from(s, row, low_of(bin));
      const int found = s.list_n;
      if (found <= CAP) {
        // the first k of them in the row's order, and their weights
        pair_sums<int>(s, found, [&](int i, int j) { return (int)(s.list_k[j] > s.list_k[i]); });
        const int n = min(found, k);
        const u64 key = t < found ? s.list_k[t] : 0;
        __syncthreads();
        if (t < found && s.sum[t] < (u64)k) {
          s.list_k[s.sum[t]] = key;
          s.list_w[s.sum[t]] = weight.of(value_of(key));
        }
        if (t == 0) s.list_n = n;
        __syncthreads();
        if (n <= 64) {
          // one wave, an element a lane, in the row's order
          if (wave != 0) return;
          u64 w = lane < n ? s.list_w[lane] : 0;
          const int idx = lane < n ? index_of(s.list_k[lane]) : 0x7fffffff;
          u64 end = wave_scan(w);
          if (p < 1.0 && lane > 0 && (double)(end - w) >= p * (double)last_lane(end)) w = 0;
          if (w < min_w) w = 0;
          end = wave_scan(w);
          const u64 last = last_before(u, last_lane(end));
          u64 before = 0;                           // of lower index
          for (int j = 0; j < n; ++j) {
            const u64 lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)w, j);
            const u64 hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(w >> 32), j);
            before += __builtin_amdgcn_readlane(idx, j) < idx ? hi << 32 | lo : 0;
          }
          if (before <= last && before + w > last) out[r] = idx;
          return;
        }
        if (wave == 0 && p < 1.0) {
          // the next cut, from running sums in that order
          constexpr int PER = FEW / 64;
          u64 w[PER], own = 0;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            w[j] = lane * PER + j < n ? s.list_w[lane * PER + j] : 0;
            own += w[j];
          }
          const u64 end = wave_scan(own);
          const double enough = p * (double)last_lane(end);
          u64 before = end - own;
#pragma unroll
          for (int j = 0; j < PER; ++j) {
            const int i = lane * PER + j;
            if (i > 0 && i < n && (double)before >= enough) s.list_w[i] = 0;
            before += w[j];
          }
        }
        listed = done = ordered = true;
      }
      if (!done) {
        clear(s);
        if (t == 0) s.list_n = 0;
      }
    }
    if (!done) {
      counted = true;
      bin_scale = narrow / 3;
      row.each4([&](f32x8 x, int) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (x[e] > -INFINITY) atomicAdd(&s.hist[bin_of(x[e])], (u64)1);
      });
      __syncthreads();
      find_bin(s, 0, 0, [&](u64) { return reached; });
      // fewer than k may be there: then all stay
      if (s.found_bin >= 0)
        cut_in_bin(s.found_bin, s.found_before, 0, [](float) { return (u64)1; }, reached);
    }
  }

  if (p < 1.0 && !ordered) {
    const auto need = [p](u64 total) {
      const double enough = p * (double)total;
      return [enough](u64 sum) { return sum > 0 && (double)sum >= enough; };
    };
    if (counted) clear(s);                          // also where fewer than k were there
    if (listed) {
      const int n = s.list_n;
      for (int i = t; i < n; i += THREADS) {
        if (s.list_k[i] < border) s.list_w[i] = 0;  // behind the first k
        atomicAdd(&s.hist[bin_of(value_of(s.list_k[i]))], s.list_w[i]);
      }
      __syncthreads();
      const auto reached = need(find_bin(s, 0, 0, need));
      const int bin = s.found_bin;
      const u64 before = s.found_before;
      for (int i = t; i < n; i += THREADS)
        if (bin_of(value_of(s.list_k[i])) == bin) candidate(s, s.list_k[i], s.list_w[i]);
      __syncthreads();
      if (s.cand_n <= CAP) {
        border = rank_candidates(s, s.cand_n, before, reached);
      } else {
        // rank them against the list itself, a few for each thread
        for (int i = t; i < n; i += THREADS) {
          const u64 key = s.list_k[i];
          if (bin_of(value_of(key)) != bin) continue;
          u64 sum = 0;
          for (int j = 0; j < n; ++j) sum += s.list_k[j] > key ? s.list_w[j] : 0;
          if (!reached(sum) && reached(sum + s.list_w[i])) s.border = key;
        }
        __syncthreads();
        border = s.border;
      }
    } else {
      const u64 floor_key = border;
      bin_scale = narrow;
      if (t == 0) s.list_n = 0;
      // Only what is at least every thread's largest goes to the histogram at
      // first: the border is hardly ever below, and the atomics cost as much
      // as the weights.
      float from = mn;
      u64 total = 0;
      auto weigh = [&](auto floored) {
        row.each1([&](f32x8 x, int q) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            u64 w = weight.of(x[e]);
            if (floored && rank_key(x[e], row.first(q) + e) < floor_key) w = 0;
            total += w;
            if (x[e] >= from) atomicAdd(&s.hist[bin_of(x[e])], w);
          }
        });
      };
#pragma unroll 1
      for (int turn = 0; turn < 2; ++turn) {
        total = 0;
        if (floor_key) weigh(std::true_type());
        else weigh(std::false_type());
        total = wave_sum(total);
        if (lane == 0) s.cand_w[wave] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) total += s.cand_w[w];
        find_bin(s, 0, total, need);
        if (s.found_bin >= 0) break;
        clear(s);
        bin_scale = narrow / 3;
        from = -3.402823466e38f;
      }
      cut_in_bin(s.found_bin, s.found_before, floor_key,
                 [&](float x) { return weight.of(x); }, need(total));
    }
  }

  // A short list: the running sum in index order, each element for itself.
  __syncthreads();
  if (listed && s.list_n <= SHORT) {
    const int n = s.list_n;
    u64 w = 0;
    if (t < n) {
      w = s.list_k[t] >= border && s.list_w[t] >= min_w ? s.list_w[t] : 0;
      s.list_w[t] = w;
    }
    __syncthreads();
    // keys of an index hold its complement
    pair_sums<u64>(s, n, [&](int i, int j) {
      return (unsigned)s.list_k[j] >= (unsigned)s.list_k[i] ? s.list_w[j] : 0;
    });
    u64 total = 0;                                  // the largest of the running sums
    if (wave == 0) {
      for (int i = lane; i < n; i += 64) total += s.list_w[i];
      total = wave_sum(total);
      if (lane == 0) s.last_want = last_before(u, total);
    }
    __syncthreads();
    if (t < n && s.sum[t] > s.last_want && s.sum[t] - w <= s.last_want) out[r] = index_of(s.list_k[t]);
    return;
  }

  // Kept weights in index order: a sum for each segment of 512, the segment
  // that the number falls into, and the logit in it.
  const int nseg = (V + SEG - 1) / SEG;
  auto kept = [&](float x, int idx) -> u64 {
    const u64 v = x > -INFINITY && rank_key(x, idx) >= border ? weight.of(x) : 0;
    return v >= min_w ? v : 0;
  };
  const int n_list = s.list_n;
  if (listed) {
    for (int i = t; i < n_list; i += THREADS) {
      const u64 v = s.list_k[i] >= border && s.list_w[i] >= min_w ? s.list_w[i] : 0;
      s.list_w[i] = v;
      if (v) atomicAdd(&s.seg[index_of(s.list_k[i]) / SEG], v);
    }
  } else {
    row.each1([&](f32x8 x, int q) {
      u64 sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += kept(x[e], row.first(q) + e);
      sum = wave_sum(sum);
      if (lane == 0 && (q >> 6) < nseg) s.seg[q >> 6] = sum;
    });
  }
  __syncthreads();
  if (wave == 0) {
    const int per = (nseg + 63) / 64;               // a lane's run of segments
    const int from = min(lane * per, nseg), upto = min(from + per, nseg);
    u64 own = 0;
    for (int i = from; i < upto; ++i) own += s.seg[i];
    const u64 end = wave_scan(own);
    const u64 total = last_lane(end);
    const u64 want = last_before(u, total);
    u64 before = end - own;
    if (before <= want && end > want) {
      int i = from;
      while (before + s.seg[i] <= want) before += s.seg[i++];
      s.last_seg = i;
      s.last_want = want - before;                  // what is left inside it
    }
  }
  __syncthreads();
  const int seg = s.last_seg;
  if (listed) {
    for (int i = t; i < n_list; i += THREADS) {
      const int at = index_of(s.list_k[i]);
      if (at / SEG == seg) s.last[at % SEG] = s.list_w[i];
    }
  } else if (t < SEG && seg * SEG + t < V) {
    s.last[t] = kept(row.at(seg * SEG + t), seg * SEG + t);
  }
  __syncthreads();
  if (wave == 0) {
    u64 w[8], sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) { w[e] = s.last[lane * 8 + e]; sum += w[e]; }
    const u64 want = s.last_want, end = wave_scan(sum);
    if (end - sum <= want && end > want) {
      u64 c = end - sum;
      int e = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c += w[j];
        e += c <= want;
      }
      out[r] = seg * SEG + lane * 8 + e;
    }
  }
}

}  // namespace

torch::Tensor sample_tokens(torch::Tensor logits, torch::Tensor u,
                            c10::optional<torch::Tensor> temperatures, double temperature,
                            c10::optional<torch::Tensor> top_ks, long top_k,
                            c10::optional<torch::Tensor> top_ps, double top_p,
                            c10::optional<torch::Tensor> min_ps, double min_p, long empty_token) {
  NO_GRAD_CHECK(logits, "sample_tokens");
  NO_GRAD_CHECK(u, "sample_tokens");
  VALUE_CHECK(logits.dim() == 2 && logits.is_cuda() && logits.size(1) >= 1 && logits.size(1) <= MAX_V,
              "sample_tokens: logits (B, V) with V from 1 to ", MAX_V, ", got ", logits.sizes());
  const long B = logits.size(0), V = logits.size(1);
  VALUE_CHECK(fits_a_launch(B, THREADS), "sample_tokens: too many rows: ", B);
  VALUE_CHECK(u.dim() == 1 && u.size(0) == B && u.device() == logits.device() &&
                  (u.scalar_type() == torch::kFloat || u.scalar_type() == torch::kDouble),
              "sample_tokens: u must be fp32 or fp64 (", B, ",) on ", logits.device(), ", got ",
              u.scalar_type(), " ", u.sizes(), " on ", u.device());
  c10::DeviceGuard guard(logits.device());
  if (!u.is_contiguous()) u = u.contiguous();
  auto opt = [&](c10::optional<torch::Tensor>& each, double all, double least, double most,
                 torch::ScalarType type, const char* what) -> Opt {
    if (!each.has_value() || !each->defined()) {
      VALUE_CHECK(all >= least && all <= most, "sampling: temperature and top_k are at least 0, "
                  "top_p and min_p from 0 to 1; got ", what, " = ", all);
      return {nullptr, all, false};
    }
    VALUE_CHECK(each->dim() == 1 && each->size(0) == B && each->device() == logits.device(),
                "sample_tokens: ", what, " must be a number or a (", B, ",) tensor on ",
                logits.device(), ", got ", each->sizes(), " on ", each->device());
    const bool wide = type == torch::kFloat && each->scalar_type() == torch::kDouble;
    // a top-k of another type: over MAX_V, where it keeps all, its size is not needed
    if (type == torch::kInt && each->scalar_type() != type)
      each = each->to(torch::kDouble).nan_to_num(0.0).clamp(-1.0, 2.0 * MAX_V);
    if ((!wide && each->scalar_type() != type) || !each->is_contiguous())
      each = each->to(wide ? torch::kDouble : type).contiguous();
    return {each->data_ptr(), all, wide};
  };
  const Opt ot = opt(temperatures, temperature, 0.0, 1.7e308, torch::kFloat, "temperature");
  const Opt ok = opt(top_ks, (double)std::min(top_k, V), 0.0, 1.7e308, torch::kInt, "top_k");
  const Opt op = opt(top_ps, top_p, 0.0, 1.0, torch::kFloat, "top_p");
  const Opt om = opt(min_ps, min_p, 0.0, 1.0, torch::kFloat, "min_p");
  auto out = torch::empty({B}, logits.options().dtype(torch::kLong));
  if (B == 0) return out;
  if (V < 8) logits = at::constant_pad_nd(logits, {0, 8 - V}, -INFINITY);   // a slot at least
  if (logits.stride(1) != 1) logits = logits.contiguous();
  auto stream = at::hip::getCurrentHIPStream().stream();
  const bool is_double = u.scalar_type() == torch::kDouble;
#define SAMPLE(T)                                                                                 \
  hipLaunchKernelGGL((sample_kernel<T>), dim3(B), dim3(THREADS), 0, stream,                        \
                     (const T*)logits.data_ptr(), (long)logits.stride(0), (int)logits.size(1), u.data_ptr(),    \
                     is_double, ot, ok, op, om, empty_token, out.data_ptr<long>())
  if (logits.scalar_type() == torch::kBFloat16) SAMPLE(__hip_bfloat16);
  else if (logits.scalar_type() == torch::kHalf) SAMPLE(__half);
  else if (logits.scalar_type() == torch::kFloat) SAMPLE(float);
  else TORCH_CHECK(false, "sample_tokens takes bf16, fp16 or fp32 logits on a GPU, got ", logits.scalar_type());
#undef SAMPLE
  HIP_CHECK_KERNEL();
  return out;
}
