// Drawing one token per row of logits under temperature, top-k, top-p and
// min-p, from given random numbers (sde_sample).  It stands where the
// reference's loops call softmax_sample_temperature_kernel, which knows the
// temperature alone (kernels.cu:285-317).
//
//   w_i = exp((x_i - max x) / T)
//   tokens in order of falling x (ties: rising index): the first k; of those
//   the shortest run whose weight reaches p of theirs; of those w >= min_p
//   token = first index i with  sum_{j <= i, kept} w_j > u * sum_{kept} w_j
//
// Every filter keeps a run of the same order, so what is kept is told by the
// last token of it: a value and, among its ties, an index.  No sort: a row is
// walked a few times by one workgroup --
//  1. the max (and the first index of it: T < 1e-6 takes that token);
//  2. where top-p acts alone, the total weight, and a histogram of
//     (max - x) / T over the tokens that may be its last one (a token below
//     (1 - p) / V never is: all those together weigh less than 1 - p);
//     top-k needs no such walk: the k-th largest of the threads' own maxima
//     bounds the k-th largest of all from below;
//  3. the tokens at or above that bound go to LDS, where each is compared with
//     each: rank and weight above it, exactly, decide what is kept, and one
//     scan in index order finds the token.
// Rows that keep more than kList tokens (flat ones, or a large k) narrow the
// last token down by further histograms over ranges of x, then walk the row
// once more for the total in index order and a 16th of it for the token.
//
// Weights and sums are 64-bit (an fp64 multiply-add issues at the rate of an
// fp32 one): which token is drawn hangs on a sum's side of u * total, and fp32
// sums over 128256 tokens would take the neighbour in some 2 % of rows.  The
// histogram's weights are 64-bit fixed-point sums: atomics in any order give
// the same bits.
#include <cfloat>
#include <cmath>

#include "batch_common.hpp"

namespace sde {
namespace smp {

using batch::bf16_elem;
using batch::f16_elem;
using batch::f32_elem;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;           // histogram bins, 1/32 of a factor 2 each
constexpr float kBinsPerLog2 = 32.f;  // so tokens below 2^-64 of the largest are left out
constexpr int kList = 512;            // tokens compared in LDS
constexpr float kMinTemperature = 1e-6f;
constexpr int kMaxVocab = 1 << 24;

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int V;
  const float* u;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  int32_t* tokens;
  float* probs;
};

// Order of the values as unsigned numbers (-0 as 0; no NaN comes here).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// 2^t for t <= 0, to 1e-14 of it: the integer part to the exponent, the rest
// f in [-1/2, 1/2] by the series of exp(f ln 2).
__device__ __forceinline__ double exp2_f64(double t) {
  if (t < -1000.0) return 0.0;
  const double n = rint(t);
  const double f = t - n;
  double y = 4.44553827187081e-10;  // ln(2)^11 / 11!
  y = fma(y, f, 7.054911620801121e-09);
  y = fma(y, f, 1.0178086009239696e-07);
  y = fma(y, f, 1.3215486790144305e-06);
  y = fma(y, f, 1.5252733804059838e-05);
  y = fma(y, f, 0.00015403530393381606);
  y = fma(y, f, 0.0013333558146428441);
  y = fma(y, f, 0.009618129107628477);
  y = fma(y, f, 0.055504108664821576);
  y = fma(y, f, 0.2402265069591007);
  y = fma(y, f, 0.6931471805599453);
  y = fma(y, f, 1.0);
  return ldexp(y, (int)n);
}

// A row's weights: 1 at the max (also an infinite one), 0 at -inf.
struct Weight {
  float top;      // the row's max
  double per;     // log2(e) / T
  float bins;     // histogram bins per unit of (max - x) / 2
  __device__ __forceinline__ double of(float x) const {
    if (x == top) return 1.0;
    if (x == -INFINITY) return 0.0;
    return exp2_f64(((double)x - (double)top) * per);
  }
  // 0 at the max, rising as x falls; kBins: left out
  __device__ __forceinline__ int bin(float x) const {
    if (x == top) return 0;
    if (x == -INFINITY) return kBins;
    return (int)fminf((0.5f * top - 0.5f * x) * bins, (float)kBins);  // (halves: no overflow)
  }
};

// What is kept: keys above `key`, and the key itself up to index `last`.
struct Kept {
  uint32_t key = 0;
  int last = INT32_MAX;
  __device__ __forceinline__ bool has(uint32_t k, int i) const {
    return k > key || (k == key && i <= last);
  }
};

// A row as 16-byte vectors: vector v holds indexes v*VEC - shift and up (the
// first and the last may hold fewer).
template <class E>
struct RowView {
  using T = typename E::type;
  static constexpr int VEC = 16 / sizeof(T);
  const T* p;
  int V, shift, vectors;
  __device__ __forceinline__ RowView(const void* base, int64_t at, int n)
      : p(static_cast<const T*>(base) + at), V(n) {
    shift = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
    vectors = (V + shift + VEC - 1) / VEC;
  }
  // Elements of vector v (none from `end` on); places outside the row and NaN
  // read as -inf.
  __device__ __forceinline__ void load(int v, int end, T (&e)[VEC]) const {
    const int i0 = v * VEC - shift;
    if (v < end && i0 >= 0 && i0 + VEC <= V) {
      const uint4 raw = *reinterpret_cast<const uint4*>(p + i0);
      __builtin_memcpy(e, &raw, 16);
    } else {
#pragma unroll
      for (int k = 0; k < VEC; k++)
        e[k] = v < end && i0 + k >= 0 && i0 + k < V ? p[i0 + k] : E::put(-INFINITY);
    }
  }
  static __device__ __forceinline__ float value(T e) {
    const float x = E::get(e);
    return x == x ? x : -INFINITY;
  }
  // f(value, index) over vectors [v0, v1), the wave's lanes side by side; a
  // lane's indexes rise.
  template <class F>
  __device__ __forceinline__ void walk(int v0, int v1, F f) const {
    constexpr int U = 16 / VEC;  // vectors in flight
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int v = v0; v < v1; v += 64 * U) {
      T e[U][VEC];
      if (v + 64 * U <= v1 && v * VEC >= shift && (v + 64 * U) * VEC - shift <= V) {
#pragma unroll
        for (int k = 0; k < U; k++) {
          const uint4 raw =
              *reinterpret_cast<const uint4*>(p + ((v + 64 * k + lane) * VEC - shift));
          __builtin_memcpy(e[k], &raw, 16);
        }
      } else {
#pragma unroll
        for (int k = 0; k < U; k++) load(v + 64 * k + lane, v1, e[k]);
      }
#pragma unroll
      for (int k = 0; k < U; k++) {
#pragma unroll
        for (int i = 0; i < VEC; i++) f(value(e[k][i]), (v + 64 * k + lane) * VEC - shift + i);
      }
    }
  }
};

struct Lds {
  uint32_t count[kBins];
  unsigned long long mass[kBins];
  uint32_t key[kList];
  int index[kList];
  double weight[kList];
  uint32_t key2[kList];
  int index2[kList];
  double wave_d[kWaves];
  double wave_d2[kWaves];
  uint32_t wave_u[kWaves];
  float wave_f[kWaves];
  int wave_i[kWaves];
  uint32_t n;
  int found;
  uint32_t lo, hi;
  double out_d[2];
  int out_i[2];
  uint32_t out_u[2];
};

__device__ __forceinline__ double shfl_up_d(double x, int d) { return __shfl_up(x, d, 64); }

// Inclusive sum over the workgroup in thread order; `total` to every thread.
__device__ __forceinline__ double block_scan(double x, double* wave_tot, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = shfl_up_d(x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // (the last use of wave_tot is over)
  if (lane == 63) wave_tot[wave] = x;
  __syncthreads();
  double before = 0.0, all = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const double t = wave_tot[w];
    if (w < wave) before += t;
    all += t;
  }
  total = all;
  return before + x;
}

__device__ __forceinline__ uint32_t block_scan_u(uint32_t x, uint32_t* wave_tot) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) wave_tot[wave] = x;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kWaves; w++)
    if (w < wave) before += wave_tot[w];
  return before + x;
}

__device__ __forceinline__ void clear_histogram(Lds& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  __syncthreads();
}

// First bin where the running count reaches `k` or the running mass `m`
// (whichever the caller asks for), and what lies in the bins before it.  Where
// none does, the last that holds anything with `force`.
struct BinAt {
  int bin;           // kBins: never reached
  uint32_t before;   // tokens before it
  uint32_t in;       // and in it
  double mass;       // weight before it
};

template <bool BY_COUNT>
__device__ __forceinline__ BinAt find_bin(Lds& s, uint32_t k, double m, double unit,
                                          bool force = false) {
  constexpr int PER = kBins / kThreads;
  uint32_t c[PER];
  double w[PER];
  uint32_t ct = 0;
  double wt = 0.0, total;
  const int b0 = threadIdx.x * PER;
  if (threadIdx.x == 0) {
    s.found = kBins;
    s.lo = 0;
  }
#pragma unroll
  for (int i = 0; i < PER; i++) {
    c[i] = s.count[b0 + i];
    w[i] = (double)s.mass[b0 + i] * unit;
    ct += c[i];
    wt += w[i];
  }
  uint32_t cc = block_scan_u(ct, s.wave_u) - ct;
  double ww = block_scan(wt, s.wave_d, total) - wt;
#pragma unroll
  for (int i = 0; i < PER; i++) {
    const bool hit = c[i] > 0 && (BY_COUNT ? cc + c[i] >= k : ww + w[i] >= m);
    if (hit) atomicMin(&s.found, b0 + i);
    if (force && c[i] > 0) atomicMax(&s.lo, (uint32_t)(b0 + i));
    c[i] += cc;
    cc = c[i];
    w[i] += ww;
    ww = w[i];
  }
  __syncthreads();
  BinAt at;
  at.bin = s.found == kBins && force ? (int)s.lo : s.found;
  if (at.bin < kBins && threadIdx.x == (uint32_t)at.bin / PER) {
    const int i = at.bin - b0;
    s.out_u[0] = c[i] - s.count[at.bin];
    s.out_u[1] = s.count[at.bin];
    s.out_d[0] = w[i] - (double)s.mass[at.bin] * unit;
  }
  __syncthreads();
  at.before = s.out_u[0];
  at.in = s.out_u[1];
  at.mass = s.out_d[0];
  __syncthreads();
  return at;
}

// The first index where the running sum of f(value, index) >= 0 in index order
// passes `share` of the total (SHARE) or `share` itself, by a walk of the row
// and one of the 16th that holds it.  Every thread gets the index (-1: the sum
// is zero), its f and the total.
struct Found {
  int index;
  double f, total;
};

template <bool SHARE, class E, class F>
__device__ __forceinline__ Found find_index(const RowView<E>& row, double share, Lds& s, F f) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int per = (row.vectors + kWaves - 1) / kWaves;
  double x = 0.0;
  row.walk(min(wave * per, row.vectors), min((wave + 1) * per, row.vectors),
           [&](float v, int i) { x += f(v, i); });
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d, 64);
  __syncthreads();
  if (lane == 0) s.wave_d2[wave] = x;
  if (threadIdx.x == 0) s.out_i[0] = -1;
  __syncthreads();
  Found r{-1, 0.0, 0.0};
#pragma unroll
  for (int w = 0; w < kWaves; w++) r.total += s.wave_d2[w];
  if (!(r.total > 0.0)) {
    __syncthreads();
    return r;
  }
  const double target = SHARE ? share * r.total : share;
  int ws = -1;
  double base = 0.0, run = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; w++) {
    const double t = s.wave_d2[w];
    // (the last wave with weight takes what rounding leaves over)
    if (t > 0.0 && (ws < 0 || !(base + s.wave_d2[ws] > target))) {
      ws = w;
      base = run;
    }
    run += t;
  }
  // the wave's vectors, in order, over all threads
  const int v0 = ws * per, v1 = min(v0 + per, row.vectors);
  const int each = (v1 - v0 + kThreads - 1) / kThreads;
  const int a = min(v0 + (int)threadIdx.x * each, v1), b = min(a + each, v1);
  double mine = 0.0;
  int tail = -1;
  double tail_f = 0.0;
  for (int v = a; v < b; v++) {
    typename E::type e[RowView<E>::VEC];
    row.load(v, v1, e);
#pragma unroll
    for (int i = 0; i < RowView<E>::VEC; i++) {
      const int idx = v * RowView<E>::VEC - row.shift + i;
      const double y = f(row.value(e[i]), idx);
      mine += y;
      if (y > 0.0) {
        tail = idx;
        tail_f = y;
      }
    }
  }
  double unused;
  const double upto = base + block_scan(mine, s.wave_d, unused);
  if (threadIdx.x == 0) s.found = kThreads;
  __syncthreads();
  if (mine > 0.0 && upto > target) atomicMin(&s.found, (int)threadIdx.x);
  __syncthreads();
  const int at = s.found;
  if (at < kThreads) {
    if ((int)threadIdx.x == at) {
      double sum = upto - mine;
      for (int v = a; v < b; v++) {
        typename E::type e[RowView<E>::VEC];
        row.load(v, v1, e);
#pragma unroll
        for (int i = 0; i < RowView<E>::VEC; i++) {
          const int idx = v * RowView<E>::VEC - row.shift + i;
          const double y = f(row.value(e[i]), idx);
          sum += y;
          if (y > 0.0 && sum > target && s.out_i[0] < 0) {
            s.out_i[0] = idx;
            s.out_d[0] = y;
          }
        }
      }
      if (s.out_i[0] < 0) {
        s.out_i[0] = tail;
        s.out_d[0] = tail_f;
      }
    }
  } else {
    // rounding: the last one with weight
    __syncthreads();
    if (threadIdx.x == 0) s.found = -1;
    __syncthreads();
    if (tail >= 0) atomicMax(&s.found, (int)threadIdx.x);
    __syncthreads();
    if ((int)threadIdx.x == s.found) {
      s.out_i[0] = tail;
      s.out_d[0] = tail_f;
    }
  }
  __syncthreads();
  r.index = s.out_i[0];
  r.f = s.out_d[0];
  __syncthreads();
  return r;
}

// Gathers the tokens for which `in` holds into s.key / s.index in index order;
// their number, or kList + 1 for more than fit.
template <class E, class P>
__device__ __forceinline__ int gather(const RowView<E>& row, Lds& s, P in) {
  const int wave = threadIdx.x >> 6;
  const int per = (row.vectors + kWaves - 1) / kWaves;
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  row.walk(min(wave * per, row.vectors), min((wave + 1) * per, row.vectors), [&](float v, int i) {
    if (in(v, i)) {
      const uint32_t n = atomicAdd(&s.n, 1u);
      if (n < kList) {
        s.key2[n] = key_of(v);
        s.index2[n] = i;
      }
    }
  });
  __syncthreads();
  const uint32_t n = s.n;
  if (n > kList) return kList + 1;
  if (threadIdx.x < n) {
    const int me = s.index2[threadIdx.x];
    int at = 0;
    for (uint32_t j = 0; j < n; j++) at += s.index2[j] < me ? 1 : 0;
    s.key[at] = s.key2[threadIdx.x];
    s.index[at] = me;
  }
  __syncthreads();
  return (int)n;
}

__device__ __forceinline__ float value_of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Rank of listed token i among the n listed (falling value, rising index) and
// the weight of those before it.
__device__ __forceinline__ void rank_of(const Lds& s, int n, int i, uint32_t& rank, double& above) {
  const uint32_t k = s.key[i];
  uint32_t r = 0;
  double a = 0.0;
  for (int j = 0; j < n; j++) {
    const uint32_t o = s.key[j];
    const bool first = o > k || (o == k && j < i);
    r += first ? 1u : 0u;
    a += first ? s.weight[j] : 0.0;
  }
  rank = r;
  above = a;
}

// Narrows the last kept token down to a key and an index, over the tokens of
// `kept`: the k-th of them (BY_COUNT), or the one whose weight, with all before
// it, reaches `m`.
template <bool BY_COUNT, class E>
__device__ __forceinline__ Kept last_kept(const RowView<E>& row, const Weight& weight, Kept kept,
                                          uint32_t k, double m, double fixed, Lds& s) {
  const int wave = threadIdx.x >> 6;
  const int per = (row.vectors + kWaves - 1) / kWaves;
  const int w0 = min(wave * per, row.vectors), w1 = min((wave + 1) * per, row.vectors);
  // the first histogram goes by (max - x) / T, further ones by equal ranges of
  // keys within [lo, hi]
  uint32_t lo = 0, hi = 0xFFFFFFFFu, width = 0;
  uint32_t before = 0;
  double mass = 0.0;
  auto bin_of = [&](float v) {
    if (width == 0) return weight.bin(v);
    const uint32_t key = key_of(v);
    return key < lo || key > hi ? kBins : (int)((hi - key) / width);
  };
  for (;;) {
    clear_histogram(s);
    row.walk(w0, w1, [&](float v, int i) {
      const int b = bin_of(v);
      if (b < kBins && weight.bin(v) < kBins && kept.has(key_of(v), i)) {
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], (unsigned long long)(weight.of(v) * fixed + 0.5));
      }
    });
    __syncthreads();
    const BinAt at = find_bin<BY_COUNT>(s, k - before, m - mass, 1.0 / fixed, width > 0);
    if (at.bin == kBins) return kept;  // everything there is
    before += at.before;
    mass += at.mass;
    auto inside = [&](float v, int i) {
      return bin_of(v) == at.bin && weight.bin(v) < kBins && kept.has(key_of(v), i);
    };
    if (at.in <= (uint32_t)kList) {
      const int n = gather(row, s, inside);
      const int i = threadIdx.x;
      if (i < n) s.weight[i] = weight.of(value_of_key(s.key[i]));
      if (i == 0) s.found = -1;
      __syncthreads();
      if (i < n) {
        uint32_t rank;
        double above;
        rank_of(s, n, i, rank, above);
        const bool in = BY_COUNT ? before + rank < k : mass + above < m;
        // the kept ones have the ranks from 0 on
        if (in) atomicMax(&s.found, (int)rank);
        s.index2[rank] = i;
      }
      __syncthreads();
      const int r = max(s.found, 0);
      const int e = s.index2[r];
      Kept out;
      out.key = s.key[e];
      out.last = s.index[e];
      __syncthreads();
      return out;
    }
    // the range of keys in the bin
    __syncthreads();
    if (threadIdx.x == 0) {
      s.lo = 0xFFFFFFFFu;
      s.hi = 0;
    }
    __syncthreads();
    uint32_t mn = 0xFFFFFFFFu, mx = 0;
    row.walk(w0, w1, [&](float v, int i) {
      if (inside(v, i)) {
        mn = min(mn, key_of(v));
        mx = max(mx, key_of(v));
      }
    });
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      mn = min(mn, (uint32_t)__shfl_xor(mn, d, 64));
      mx = max(mx, (uint32_t)__shfl_xor(mx, d, 64));
    }
    if ((threadIdx.x & 63) == 0) {
      atomicMin(&s.lo, mn);
      atomicMax(&s.hi, mx);
    }
    __syncthreads();
    lo = s.lo;
    hi = s.hi;
    if (lo == hi) {
      // ties: the first t of them by index
      const double w = weight.of(value_of_key(lo));
      double t = BY_COUNT ? (double)(k - before) : ceil((m - mass) / w);
      t = fmin(fmax(t, 1.0), (double)at.in);
      const uint32_t key = lo;
      const Found f = find_index<false>(row, t - 1.0, s, [&](float v, int i) {
        return key_of(v) == key && kept.has(key, i) ? 1.0 : 0.0;
      });
      Kept out;
      out.key = key;
      out.last = f.index;
      return out;
    }
    width = (hi - lo) / kBins + 1;
  }
}

template <class E>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Lds s;
  const int r = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowView<E> row(a.logits, r * a.row_stride, a.V);
  const int per = (row.vectors + kWaves - 1) / kWaves;
  const int w0 = min(wave * per, row.vectors), w1 = min((wave + 1) * per, row.vectors);
  const float T = a.temperature ? a.temperature[r] : 1.f;
  const double u = a.u[r];
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.f;
  const double min_p = a.min_p && a.min_p[r] > 0.f ? fmin((double)a.min_p[r], 1.0) : 0.0;

  // ---- the max, and its first index
  float mine = -INFINITY;
  int at = -1;
  row.walk(w0, w1, [&](float v, int i) {
    if (v > mine) {
      mine = v;
      at = i;
    }
  });
  {
    float x = mine;
    int i = at;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const float y = __shfl_xor(x, d, 64);
      const int j = __shfl_xor(i, d, 64);
      if (y > x || (y == x && (uint32_t)j < (uint32_t)i)) {
        x = y;
        i = j;
      }
    }
    if (lane == 0) {
      s.wave_f[wave] = x;
      s.wave_i[wave] = i;
    }
  }
  __syncthreads();
  Weight weight;
  weight.top = s.wave_f[0];
  int first = s.wave_i[0];
#pragma unroll
  for (int w = 1; w < kWaves; w++)
    if (s.wave_f[w] > weight.top) {
      weight.top = s.wave_f[w];
      first = s.wave_i[w];
    }
  const bool hot = T >= kMinTemperature;
  if (first < 0 || !hot) {  // nothing to draw from, or the max itself
    if (threadIdx.x == 0) {
      a.tokens[r] = first;
      if (a.probs) a.probs[r] = first < 0 ? 0.f : 1.f;
    }
    return;
  }
  weight.per = 1.4426950408889634 / (double)T;
  weight.bins = 2.f * kBinsPerLog2 * (float)weight.per;
  const bool has_k = k > 0 && k < a.V;
  const bool has_p = p < 1.f;
  // fixed point of the histogram's weights: V of them fit 63 bits
  const double fixed = ldexp(1.0, 30 + __clz(a.V));

  int token = -1;
  double w_token = 0.0, total = 0.0;
  int n = kList + 1;      // listed tokens
  double all = 0.0;       // the total that top-p is a share of (has_k: the list's)
  if (has_k && k <= kList) {
    // the k-th largest of the threads' maxima, to a bin
    clear_histogram(s);
    const int b = weight.bin(mine);
    if (b < kBins) atomicAdd(&s.count[b], 1u);
    __syncthreads();
    const int cut = find_bin<true>(s, (uint32_t)k, 0.0, 0.0).bin;
    // (kBins: fewer than k threads hold a token of weight)
    n = gather(row, s, [&](float v, int) { return weight.bin(v) <= min(cut, kBins - 1); });
  } else if (has_p && !has_k) {
    const double least = 0.5 * fmax(1.0 - (double)p, 0.0) / (double)a.V;
    clear_histogram(s);
    double x = 0.0;
    row.walk(w0, w1, [&](float v, int) {
      const double w = weight.of(v);
      x += w;
      const int b = weight.bin(v);
      if (w >= least && b < kBins) {
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], (unsigned long long)(w * fixed + 0.5));
      }
    });
    block_scan(x, s.wave_d, all);
    // (a little beyond p: the fixed-point sums are cut off)
    const BinAt b = find_bin<false>(s, 0, (double)p * all * (1.0 + 1e-9), 1.0 / fixed);
    if (b.bin < kBins && b.before + b.in <= (uint32_t)kList)
      n = gather(row, s, [&](float v, int) { return weight.bin(v) <= b.bin; });
  }
  if (n <= kList) {
    const int i = threadIdx.x;
    if (i < n) s.weight[i] = weight.of(value_of_key(s.key[i]));
    if (i == 0) s.found = kList;
    __syncthreads();
    uint32_t rank = 0;
    double above = 0.0, w = 0.0;
    bool in = i < n;
    if (in) {
      rank_of(s, n, i, rank, above);
      w = s.weight[i];
      if (has_k) in = rank < (uint32_t)k;
    }
    if (has_k && has_p) block_scan(in ? w : 0.0, s.wave_d, all);
    if (in && has_p) in = above < (double)p * all || rank == 0;
    if (in) in = w >= min_p;
    const double upto = block_scan(in ? w : 0.0, s.wave_d, total);
    const double target = u * total;
    if (in && upto > target) atomicMin(&s.found, i);
    __syncthreads();
    if (s.found == kList) {  // u at or above 1 (or rounding): the last kept
      __syncthreads();
      if (i == 0) s.found = -1;
      __syncthreads();
      if (in) atomicMax(&s.found, i);
      __syncthreads();
    }
    token = s.index[s.found];
    w_token = s.weight[s.found];
  } else {
    Kept kept;
    if (has_k) kept = last_kept<true>(row, weight, kept, (uint32_t)k, 0.0, fixed, s);
    if (has_p) {
      double x = 0.0;
      row.walk(w0, w1, [&](float v, int i) { x += kept.has(key_of(v), i) ? weight.of(v) : 0.0; });
      block_scan(x, s.wave_d, all);
      kept = last_kept<false>(row, weight, kept, 0u, (double)p * all, fixed, s);
    }
    const Found f = find_index<true>(row, u, s, [&](float v, int i) {
      if (!kept.has(key_of(v), i)) return 0.0;
      const double w = weight.of(v);
      return w >= min_p ? w : 0.0;
    });
    token = f.index;
    w_token = f.f;
    total = f.total;
  }
  if (threadIdx.x == 0) {
    a.tokens[r] = token;
    if (a.probs) a.probs[r] = (float)(w_token / total);
  }
}

}  // namespace smp
}  // namespace sde

extern "C" int sde_sample(const void* d_logits, int64_t row_stride, int dtype, int n_rows,
                          int vocab, const float* d_u, const float* d_temperature,
                          const int32_t* d_top_k, const float* d_top_p, const float* d_min_p,
                          int32_t* d_tokens, float* d_probs, sde_stream_t stream) {
  using namespace sde::smp;
  if (n_rows < 0 || vocab < 1 || !sde::batch::known_dtype(dtype)) return SDE_ERR_INVALID_ARGUMENT;
  if (vocab > kMaxVocab || n_rows > (1 << 21)) return SDE_ERR_UNSUPPORTED;
  if (n_rows == 0) return SDE_OK;
  if (!d_logits || !d_u || !d_tokens || (n_rows > 1 && row_stride < vocab))
    return SDE_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(d_logits) % (size_t)sde::batch::elem_bytes(dtype) != 0)
    return SDE_ERR_INVALID_ARGUMENT;
  const SampleArgs a{d_logits, row_stride, vocab,   d_u,      d_temperature,
                     d_top_k,  d_top_p,    d_min_p, d_tokens, d_probs};
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == SDE_F32)
    sample_kernel<sde::batch::f32_elem><<<dim3(n_rows), dim3(kThreads), 0, s>>>(a);
  else if (dtype == SDE_F16)
    sample_kernel<sde::batch::f16_elem><<<dim3(n_rows), dim3(kThreads), 0, s>>>(a);
  else
    sample_kernel<sde::batch::bf16_elem><<<dim3(n_rows), dim3(kThreads), 0, s>>>(a);
  return sde::launch_status();
}
