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
// ranked against each other, and a last pass in index order finds the token.
//
// A token is a comparison of a sum with as many borders as there are logits:
// an error e in the cumulative share moves a row's token with a probability of
// about 2 V e, one row in 150 in fp32 at V = 32128.  So weights are computed in
// fp64 (table of 2^(j/64) and a polynomial of degree 5, relative error under
// 1e-14) and summed as integers w * 2^44: exact, in any order, hence atomics
// whose order does not matter.  A weight under 2^-45 counts as none.
//
// One workgroup a row; the row is read a few times, from memory once and from
// the L2 after that.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "../common.h"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2 * THREADS;
constexpr int CAP = THREADS;             // elements of a border bin ranked at once
constexpr int MAX_V = 1 << 19;           // sums stay under 2^63
constexpr int SEGS = MAX_V / 512 + 16;   // a wave's 512 logits
constexpr u64 NO_BORDER = 0;             // below every element

struct Opt {                             // a number for all rows, or one each
  const void* each;
  double all;
  DEVINL double f(int row) const { return each ? (double)((const float*)each)[row] : all; }
  DEVINL int i(int row) const { return each ? ((const int*)each)[row] : (int)all; }
};

// 2^(j/64), correctly rounded
__constant__ const double EXP2_64[64] = {
    1.0, 1.0108892860517005, 1.0218971486541166, 1.0330248790212284,
    1.0442737824274138, 1.0556451783605572, 1.0671404006768237, 1.0787607977571199,
    1.0905077326652577, 1.102382583307841, 1.1143867425958924, 1.1265216186082418,
    1.1387886347566916, 1.1511892299529827, 1.1637248587775775, 1.1763969916502812,
    1.189207115002721, 1.202156731452703, 1.215247359980469, 1.22848053610687,
    1.241857812073484, 1.255380757024691, 1.2690509571917332, 1.2828700160787783,
    1.2968395546510096, 1.3109612115247644, 1.3252366431597413, 1.339667524053303,
    1.3542555469368927, 1.3690024229745905, 1.383909881963832, 1.3989796725383112,
    1.4142135623730951, 1.42961333839197, 1.4451808069770467, 1.460917794180647,
    1.4768261459394993, 1.4929077282912648, 1.5091644275934228, 1.5255981507445384,
    1.5422108254079407, 1.559004400237837, 1.5759808451078865, 1.593142151342267,
    1.6104903319492543, 1.6280274218573478, 1.645755478153965, 1.6636765803267364,
    1.681792830507429, 1.7001063537185235, 1.718619298122478, 1.7373338352737062,
    1.7562521603732995, 1.7753764925265212, 1.7947090750031072, 1.8142521755003989,
    1.8340080864093424, 1.8539791250833855, 1.8741676341103, 1.8945759815869656,
    1.9152065613971474, 1.9360617934922943, 1.9571441241754002, 1.978456026387951,
};

// e^a for a <= 0, zero under -40:  a = n ln2/64 + r,  |r| <= ln2/128
DEVINL double exp_neg(double a, const double* table) {
  if (!(a > -40.0)) return 0.0;
  const double n = __builtin_rint(a * 92.33248261689366);        // 64/ln2
  double r = __builtin_fma(n, -0.010830424696249145, a);          // ln2/64
  r = __builtin_fma(n, -3.623510646634843e-19, r);                  // and its rest
  double p = __builtin_fma(r, 1.0 / 120, 1.0 / 24);
  p = __builtin_fma(p, r, 1.0 / 6);
  p = __builtin_fma(p, r, 0.5);
  p = __builtin_fma(p, r, 1.0);
  p = __builtin_fma(p, r, 1.0);
  const int k = (int)n;
  return __builtin_ldexp(p * table[k & 63], k >> 6);
}

// a larger float has a larger key; -inf is the lowest of what occurs
DEVINL unsigned key_of(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// one order over all elements of a row: value, then the lower index first
DEVINL u64 rank_key(float x, int idx) { return (u64)key_of(x) << 32 | (unsigned)~idx; }

template <typename T> struct Row {
  const T* p;      // the row
  int V, off;      // off: elements from the 16-byte line that p lies in
  static constexpr int N = 8;
  // element e of slot q is logit q*8 + e - off, so that whole slots are aligned
  DEVINL int index(int q, int e) const { return q * N + e - off; }
  DEVINL int slots() const { return (V + off + N - 1) / N; }
  DEVINL void load(int q, float* x) const {
    const int i0 = q * N - off;
    if (i0 >= 0 && i0 + N <= V) {
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int v = 0; v < N; v += W) {
        const VecT<T, W> in = vload<T, W>(p + i0 + v);
#pragma unroll
        for (int u = 0; u < W; ++u) x[v + u] = DT<T>::to_f32(in.data[u]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        x[e] = i0 + e >= 0 && i0 + e < V ? DT<T>::to_f32(p[i0 + e]) : -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = x[e] == x[e] ? x[e] : -INFINITY;   // NaN: not there
  }
};

DEVINL u64 shfl_up64(u64 x, int d) { return __shfl_up(x, d, 64); }

DEVINL u64 wave_sum64(u64 x) {
#pragma unroll
  for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}
DEVINL u64 wave_scan64(u64 x) {          // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const u64 y = shfl_up64(x, off);
    if (lane >= off) x += y;
  }
  return x;
}

struct Shared {
  u64 hist[BINS];
  u64 cand_w[CAP];
  u64 cand_k[CAP];
  u64 seg[SEGS];
  u64 wave_tot[WAVES];
  double table[64];
  float red[16];
  u64 found_before, border;
  int found_bin, cand_n;
};

struct Weights {
  float max;
  double inv_t;
  const double* table;
  DEVINL u64 of(float x) const {
    const double w = x == max ? 1.0 : exp_neg(((double)x - (double)max) * inv_t, table);
    // w * 2^44 in the low bits of a double over 2^52: rounded to an integer
    const double d = __builtin_fma(w, 17592186044416.0, 4503599627370496.0);
    return __builtin_bit_cast(u64, d) & 0xfffffffffffffull;
  }
};

// The first bin with whose elements the running sum reaches what a cut needs:
// leaves it and what lies before it in s.found_*.  Every thread calls it.
template <typename Reached>
DEVINL void find_bin(Shared& s, Reached reached) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const u64 a = s.hist[2 * t], b = s.hist[2 * t + 1];
  const u64 inc = wave_scan64(a + b);
  if (lane == 63) s.wave_tot[wave] = inc;
  __syncthreads();
  u64 before = inc - (a + b);
  for (int w = 0; w < wave; ++w) before += s.wave_tot[w];
  // exactly one thread finds its bin: the first to reach
  if (!reached(before) && reached(before + a)) { s.found_bin = 2 * t; s.found_before = before; }
  else if (!reached(before + a) && reached(before + a + b)) {
    s.found_bin = 2 * t + 1;
    s.found_before = before + a;
  }
  __syncthreads();
}

// The border element: the last one, in the row's order, that a cut keeps.
//   value(x): what an element adds to the running sum (1, or its weight);
//   elements below floor_key do not count.
//   reached(sum): whether a running sum is all that the cut keeps; false for 0,
//   true for the sum over all.
template <typename T, typename Value, typename Reached>
DEVINL u64 find_border(Shared& s, const Row<T>& row, float max, float bin_scale, u64 floor_key,
                       Value value, Reached reached) {
  const int t = threadIdx.x;
  const int slots = row.slots();
  auto bin_of = [&](float x) {
    const float d = x == max ? 0.f : max - x;
    return (int)fminf(d * bin_scale, (float)(BINS - 1));
  };
  for (int i = t; i < BINS; i += THREADS) s.hist[i] = 0;
  if (t == 0) s.cand_n = 0;
  __syncthreads();
  for (int q = t; q < slots; q += THREADS) {
    float x[8];
    row.load(q, x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (x[e] > -INFINITY && rank_key(x[e], row.index(q, e)) >= floor_key)
        atomicAdd(&s.hist[bin_of(x[e])], value(x[e]));
  }
  __syncthreads();
  find_bin(s, reached);
  const int bin = s.found_bin;
  u64 before = s.found_before;
  // the bin's elements, if they fit
  for (int q = t; q < slots; q += THREADS) {
    float x[8];
    row.load(q, x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (x[e] > -INFINITY && bin_of(x[e]) == bin) {
        const u64 k = rank_key(x[e], row.index(q, e));
        if (k >= floor_key) {
          const int at = atomicAdd(&s.cand_n, 1);
          if (at < CAP) { s.cand_k[at] = k; s.cand_w[at] = value(x[e]); }
        }
      }
  }
  __syncthreads();
  const int n = s.cand_n;
  if (n <= CAP) {
    if (t < n) {
      const u64 mine = s.cand_k[t];
      u64 sum = before;
      for (int j = 0; j < n; ++j) sum += s.cand_k[j] > mine ? s.cand_w[j] : 0;
      if (!reached(sum) && reached(sum + s.cand_w[t])) s.border = mine;
    }
    __syncthreads();
    return s.border;
  }
  // Too many share the bin (a flat row, or masks of a finite value stretched
  // it): narrow the border down by 11 bits of the order's key at a time.
  u64 prefix = 0;
  int shift = 64;
  while (shift > 0) {
    const int bits = min(11, shift);
    const int up = shift;
    shift -= bits;
    __syncthreads();
    for (int i = t; i < BINS; i += THREADS) s.hist[i] = 0;
    __syncthreads();
    for (int q = t; q < slots; q += THREADS) {
      float x[8];
      row.load(q, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!(x[e] > -INFINITY) || bin_of(x[e]) != bin) continue;
        const u64 k = rank_key(x[e], row.index(q, e));
        if (k < floor_key || (up < 64 && (k >> up) != prefix)) continue;
        // bin 0 holds the largest
        const int b = (1 << bits) - 1 - (int)(k >> shift & ((1u << bits) - 1));
        atomicAdd(&s.hist[b], value(x[e]));
      }
    }
    __syncthreads();
    const u64 outer = before;
    find_bin(s, [&](u64 sum) { return reached(outer + sum); });
    before = outer + s.found_before;
    prefix = prefix << bits | (u64)((1 << bits) - 1 - s.found_bin);
  }
  return prefix;
}

template <typename T, typename U>
__global__ void __launch_bounds__(THREADS)
sample_kernel(const T* __restrict__ logits, long ld, int V, const U* __restrict__ uniform,
              Opt temperature, Opt top_k, Opt top_p, Opt min_p, long empty_token,
              long* __restrict__ out) {
  __shared__ Shared s;
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  Row<T> row;
  row.p = logits + r * ld;
  row.V = V;
  row.off = (int)(reinterpret_cast<uintptr_t>(row.p) % 16 / sizeof(T));
  const int slots = row.slots();
  if (t < 64) s.table[t] = EXP2_64[t];

  // extremes of what is there
  float mx = -INFINITY, mn = INFINITY, there = 0.f;
  for (int q = t; q < slots; q += THREADS) {
    float x[8];
    row.load(q, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mx = fmaxf(mx, x[e]);
      mn = fminf(mn, x[e] > -INFINITY ? x[e] : INFINITY);
      there += x[e] > -INFINITY ? 1.f : 0.f;
    }
  }
  mx = block_reduce_max(mx, s.red);
  mn = -block_reduce_max(-mn, s.red);
  there = block_reduce_sum(there, s.red);          // exact: under 2^24
  if (mx == -INFINITY) {
    if (t == 0) out[r] = empty_token;
    return;
  }

  double temp = temperature.f(r);
  int k = top_k.i(r);
  const double p = top_p.f(r);
  double floor_w = min_p.f(r);
  if (!(temp > 0.0)) { temp = 1.0; k = 1; }
  floor_w = floor_w < 1.0 ? floor_w : 1.0;       // the maximum always stays
  const Weights w{mx, 1.0 / temp, s.table};
  const u64 min_w = floor_w > 0.0 ? (u64)ceil(floor_w * 17592186044416.0 - 0.5) : 0;

  // bins over the distance from the maximum that matters; what is further
  // shares the last one
  const float range = fminf(mx - mn, 64.f * fmaxf(1.f, (float)temp));
  const float bin_scale = range > 0.f ? fminf((float)(BINS - 1) / range, 1e30f) : 0.f;

  u64 border = NO_BORDER;
  if (k > 0 && k < V) {
    // fewer than k may be there: then all stay
    const u64 need = k;
    if (there > (float)k)
      border = find_border(s, row, mx, bin_scale, NO_BORDER, [](float) { return (u64)1; },
                           [&](u64 sum) { return sum >= need; });
  }
  __syncthreads();
  if (p < 1.0 && k != 1) {
    // the sum over K first
    u64 mine = 0;
    for (int q = t; q < slots; q += THREADS) {
      float x[8];
      row.load(q, x);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (x[e] > -INFINITY && rank_key(x[e], row.index(q, e)) >= border) mine += w.of(x[e]);
    }
    mine = wave_sum64(mine);
    if (lane == 0) s.wave_tot[wave] = mine;
    __syncthreads();
    u64 total = 0;
    for (int v = 0; v < WAVES; ++v) total += s.wave_tot[v];
    __syncthreads();
    const double need = p * (double)total;
    // sum > 0: at least the first stays
    border = find_border(s, row, mx, bin_scale, border, [&](float x) { return w.of(x); },
                         [&](u64 sum) { return sum > 0 && (double)sum >= need; });
  }
  __syncthreads();

  // kept weights in index order: a sum for each wave's 512 logits
  auto kept = [&](float x, int idx) -> u64 {
    if (!(x > -INFINITY) || rank_key(x, idx) < border) return 0;
    const u64 v = w.of(x);
    return v >= min_w ? v : 0;
  };
  const int nseg = (slots + 63) / 64;
  for (int q = t; q < nseg * 64; q += THREADS) {
    u64 mine = 0;
    if (q < slots) {
      float x[8];
      row.load(q, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) mine += kept(x[e], row.index(q, e));
    }
    mine = wave_sum64(mine);
    if (lane == 0) s.seg[q >> 6] = mine;
  }
  __syncthreads();
  if (wave != 0) return;
  u64 own = 0;                               // lane's run of segments
  const int per = (nseg + 63) / 64;
  for (int i = 0; i < per; ++i)
    if (lane * per + i < nseg) own += s.seg[lane * per + i];
  const u64 inc = wave_scan64(own);
  const u64 total = __shfl(inc, 63, 64);
  const double target = (double)uniform[r] * (double)total;
  u64 want = target > 0.0 ? (u64)target : 0;  // running sum > u*total, in integers
  if (want >= total) want = total - 1;
  const u64 hits = __ballot(inc > want);
  const int owner = __ffsll(hits) - 1;
  int seg = 0;
  u64 before = inc - own;
  if (lane == owner)
    for (int i = 0; i < per; ++i) {
      const u64 v = lane * per + i < nseg ? s.seg[lane * per + i] : 0;
      seg = lane * per + i;
      if (before + v > want) break;
      before += v;
    }
  seg = __shfl(seg, owner, 64);
  before = __shfl(before, owner, 64);
  const int q = seg * 64 + lane;
  float x[8];
  u64 kw[8], sum = 0;
  if (q < slots) row.load(q, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    kw[e] = q < slots ? kept(x[e], row.index(q, e)) : 0;
    sum += kw[e];
  }
  const u64 upto = wave_scan64(sum) + before;
  const int who = __ffsll(__ballot(upto > want)) - 1;
  if (lane == who) {
    u64 c = upto - sum;
    int id = 0;
    bool done = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c += kw[e];
      if (!done && c > want) { id = row.index(q, e); done = true; }
    }
    out[r] = id;
  }
}

}  // namespace

torch::Tensor sample_tokens(torch::Tensor logits, torch::Tensor u,
                            c10::optional<torch::Tensor> temperatures, double temperature,
                            c10::optional<torch::Tensor> top_ks, long top_k,
                            c10::optional<torch::Tensor> top_ps, double top_p,
                            c10::optional<torch::Tensor> min_ps, double min_p, long empty_token) {
  TORCH_CHECK(logits.dim() == 2 && logits.is_cuda(), "sample_tokens: logits must be (B,V) on a GPU");
  const long B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V > 0 && V <= MAX_V, "sample_tokens: 1 to ", MAX_V, " logits a row, got ", V);
  TORCH_CHECK(B < (1L << 31), "sample_tokens: too many rows");
  TORCH_CHECK(u.dim() == 1 && u.size(0) == B && u.is_contiguous() &&
                  u.device() == logits.device() &&
                  (u.scalar_type() == torch::kFloat || u.scalar_type() == torch::kDouble),
              "sample_tokens: u must be fp32 or fp64 (B,) on the logits' device");
  auto opt = [&](const c10::optional<torch::Tensor>& each, double all, torch::ScalarType type,
                 const char* what) -> Opt {
    if (!each.has_value() || !each->defined()) return {nullptr, all};
    TORCH_CHECK(each->dim() == 1 && each->size(0) == B && each->is_contiguous() &&
                    each->scalar_type() == type && each->device() == logits.device(),
                "sample_tokens: ", what, " must be a number or a ", type,
                " (B,) tensor on the logits' device");
    return {each->data_ptr(), all};
  };
  const Opt ot = opt(temperatures, temperature, torch::kFloat, "temperature");
  const Opt ok = opt(top_ks, (double)top_k, torch::kInt, "top_k");
  const Opt op = opt(top_ps, top_p, torch::kFloat, "top_p");
  const Opt om = opt(min_ps, min_p, torch::kFloat, "min_p");
  c10::DeviceGuard guard(logits.device());
  auto out = torch::empty({B}, logits.options().dtype(torch::kLong));
  if (B == 0) return out;
  if (logits.stride(1) != 1) logits = logits.contiguous();
  auto stream = at::hip::getCurrentHIPStream().stream();
#define SAMPLE(T, U)                                                                               \
  hipLaunchKernelGGL((sample_kernel<T, U>), dim3(B), dim3(THREADS), 0, stream,                     \
                     (const T*)logits.data_ptr(), (long)logits.stride(0), (int)V,                  \
                     (const U*)u.data_ptr(), ot, ok, op, om, empty_token, out.data_ptr<long>())
#define BY_U(T)                                                 \
  do {                                                          \
    if (u.scalar_type() == torch::kFloat) SAMPLE(T, float);     \
    else SAMPLE(T, double);                                     \
  } while (0)
  if (logits.scalar_type() == torch::kBFloat16) BY_U(__hip_bfloat16);
  else if (logits.scalar_type() == torch::kHalf) BY_U(__half);
  else if (logits.scalar_type() == torch::kFloat) BY_U(float);
  else TORCH_CHECK(false, "sample_tokens: bf16, fp16 or fp32 logits, got ", logits.scalar_type());
#undef BY_U
#undef SAMPLE
  HIP_CHECK_KERNEL();
  return out;
}
