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
// Weights and sums are 64-bit: which token is drawn hangs on a sum's side of
// u * total, and fp32 sums over 128256 tokens would take the neighbour in some
// 2 % of rows.  The histogram's weights are 64-bit fixed-point sums: atomics in
// any order give the same bits.
//
// Long rows that do not fill the chip by themselves go in slices: maxima, weights
// and lists are made by kernels with a workgroup per slice, and the row's own
// workgroup starts at step 3.
//
// Measured on MI355X: one fp32 row of 32000 15.4 us, a chain of walks by one
// workgroup; 24 fp32 rows of 128256 under top-k and top-p 58 us (max 5.7, weights 21,
// list 8.7, row 23); 192 bf16 ones 117 us (12, 55, 15, 35 to 42): the 64-bit
// weights and their histogram, not the 49 MB, take the time.
#include <cfloat>
#include <cmath>

#include "batch_common.hpp"

namespace sde {
namespace smp {

using batch::bf16_elem;
using batch::f16_elem;
using batch::f32_elem;

constexpr int kThreads = 1024;        // of a row's workgroup
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;           // its histogram bins, 1/32 of a factor 2 each
constexpr float kBinsPerLog2 = 32.f;  // so tokens below 2^-64 of the largest are left out
constexpr int kList = 512;            // tokens compared in LDS
constexpr int kSliceThreads = 256;    // of a slice's workgroup
constexpr int kSliceWaves = kSliceThreads / 64;
constexpr int kSliceBins = 1024;
constexpr int kMaxSlices = 16;
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

__device__ __forceinline__ float value_of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

constexpr int kPowers = 256;

// 2^(i / 256), i < 256, by the series of exp(f ln 2): to 1e-14 (f < 1: the
// twelfth term is 2.5e-11 of it; f is halved and the result squared).
template <int THREADS>
__device__ __forceinline__ void fill_powers(double* power) {
  for (int i = threadIdx.x; i < kPowers; i += THREADS) {
    const double f = (double)i * (0.5 / kPowers);
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
  power[i] = y * y;
  }
}

// A row's weights: 1 at the max (also an infinite one), 0 at -inf and below
// 2^-1000.  2^t to 2e-13 of it: t to 1/256ths, whose powers lie in LDS, and a
// cubic for the rest, f in [-1/512, 1/512]: ten 64-bit operations, where a series
// alone takes seventeen.
struct Weight {
  float top;            // the row's max
  float least;          // weights from here down are 0
  double per;           // 256 log2(e) / T
  uint32_t bin_mul;     // histogram bins per 1/256 of a factor 2, 16 bits of fraction
  uint32_t bin_end;     // 1/256ths that reach the last bin
  int limit;            // number of bins
  const double* power;  // fill_powers'
  __device__ __forceinline__ Weight(float max_x, float T, const double* powers)
      : top(max_x), power(powers) {
    per = 1.4426950408889634 * kPowers / (double)T;
    least = top - (1000.f * kPowers) / (float)per;
  }
  // `n` bins of 1 / per_log2 of a factor 2
  __device__ __forceinline__ void set_bins(float per_log2, int n) {
    bin_mul = (uint32_t)fmaxf(per_log2 * (65536.f / kPowers), 1.f);
    bin_end = (uint32_t)(((uint64_t)n << 16) / bin_mul) + 1;
    limit = n;
  }
  // The weight, and `n`: its log2 to 1/256ths (meaningless where it is 0).
  // NaN weighs 0.
  __device__ __forceinline__ double of(float x, int& n) const {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the sum's low word is rint(t)
    const double t = ((double)x - (double)top) * per;
    const double shifted = t + kRound;
    const double f = t - (shifted - kRound);
    n = (int)(uint32_t)__builtin_bit_cast(uint64_t, shifted);
    double y = fma(f, 3.308302680541371e-09, 3.665565596910106e-06);
    y = fma(f, y, 0.0027076061740622863);
    y = fma(f, y, 1.0) * power[n & (kPowers - 1)];
    // (above 2^-1000: the exponent takes the sum)
    uint64_t bits = __builtin_bit_cast(uint64_t, y);
    bits += (uint64_t)(uint32_t)((n >> 8) << 20) << 32;
    const double w = x > least ? __builtin_bit_cast(double, bits) : 0.0;
    n = x == top ? 0 : n;
    return x == top ? 1.0 : w;
  }
  __device__ __forceinline__ double of(float x) const {
    int n;
    return of(x, n);
  }
  // 0 at the max, rising as x falls, of a weight that is not 0; `limit` and
  // beyond: left out
  __device__ __forceinline__ int bin_of(int n) const {
    return (int)((min((uint32_t)-n, bin_end) * (uint64_t)bin_mul) >> 16);
  }
  // `limit` also for weights of 0
  __device__ __forceinline__ int bin(float x) const {
    int n;
    return of(x, n) > 0.0 ? min(bin_of(n), limit) : limit;
  }
};

// Fixed point of the histograms' weights: V of them fit 63 bits, one fits 52.
__device__ __forceinline__ double fixed_point(int V) { return ldexp(1.0, min(30 + __clz(V), 51)); }
// w * fixed, rounded (the sum's low bits).
__device__ __forceinline__ unsigned long long to_fixed(double w, double fixed) {
  constexpr double k2p52 = 4503599627370496.0;
  return __builtin_bit_cast(unsigned long long, fma(w, fixed, k2p52)) -
         __builtin_bit_cast(unsigned long long, k2p52);
}

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
  // Vector v (nothing from `end` on); places outside the row read as -inf.
  __device__ __forceinline__ uint4 load(int v, int end) const {
    const int i0 = v * VEC - shift;
    uint4 raw;
    if (v < end && i0 >= 0 && i0 + VEC <= V) {
      raw = *reinterpret_cast<const uint4*>(p + i0);
    } else {
      T e[VEC];
#pragma unroll
      for (int k = 0; k < VEC; k++)
        e[k] = v < end && i0 + k >= 0 && i0 + k < V ? p[i0 + k] : E::put(-INFINITY);
      __builtin_memcpy(&raw, e, 16);
    }
    return raw;
  }
  // (NaN passes no compare and weighs nothing)
  static __device__ __forceinline__ float value(T e) { return E::get(e); }
  // f(value, index) over a vector's elements, in pairs: the loop is rolled, since
  // f unrolled eight times over spilled registers (the time is the same).
  template <class F>
  static __device__ __forceinline__ void each(uint4 c, int index, F f) {
#pragma unroll 1
    for (int i = 0; i < VEC; i += 2) {
      if constexpr (sizeof(T) == 4) {
        f(value(__builtin_bit_cast(float, c.x)), index + i);
        f(value(__builtin_bit_cast(float, c.y)), index + i + 1);
        c.x = c.z;
        c.y = c.w;
      } else {
        f(value((T)(c.x & 0xFFFFu)), index + i);
        f(value((T)(c.x >> 16)), index + i + 1);
        c.x = c.y;
        c.y = c.z;
        c.z = c.w;
      }
    }
  }
  // f(value, index) over vectors [v0, v1), the wave's lanes side by side; a
  // lane's indexes rise.  LIGHT: a few instructions, unrolled.
  template <bool LIGHT = false, class F>
  __device__ __forceinline__ void walk(int v0, int v1, F f) const {
    constexpr int U = 4;  // vectors in flight
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int v = v0; v < v1; v += 64 * U) {
      uint4 raw[U];
      if (v + 64 * U <= v1 && v * VEC >= shift && (v + 64 * U) * VEC - shift <= V) {
#pragma unroll
        for (int k = 0; k < U; k++)
          raw[k] = *reinterpret_cast<const uint4*>(p + ((v + 64 * k + lane) * VEC - shift));
      } else {
#pragma unroll
        for (int k = 0; k < U; k++) raw[k] = load(v + 64 * k + lane, v1);
      }
      if constexpr (LIGHT) {
#pragma unroll
        for (int k = 0; k < U; k++) {
          T e[VEC];
          __builtin_memcpy(e, &raw[k], 16);
#pragma unroll
          for (int i = 0; i < VEC; i++) f(value(e[i]), (v + 64 * k + lane) * VEC - shift + i);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < U; k++) {
          each(raw[0], (v + 64 * k + lane) * VEC - shift, f);
#pragma unroll
          for (int j = 0; j + 1 < U; j++) raw[j] = raw[j + 1];
        }
      }
    }
  }
};

struct Lds {
  double power[kPowers];
  __attribute__((aligned(16))) uint32_t count[kBins];
  unsigned long long mass[kBins];
  __attribute__((aligned(16))) uint32_t key[kList];
  int index[kList];
  __attribute__((aligned(16))) double weight[kList];
  uint32_t key2[kList];
  __attribute__((aligned(16))) int index2[kList];
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
  uint32_t upto[64];
  double slice_w[kMaxSlices];
};

__device__ __forceinline__ double shfl_up_d(double x, int d) { return __shfl_up(x, d, 64); }

// Inclusive sum over the workgroup in thread order; `total` to every thread.
template <int W = kWaves>
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
  for (int w = 0; w < W; w++) {
    const double t = wave_tot[w];
    if (w < wave) before += t;
    all += t;
  }
  total = all;
  return before + x;
}

template <int W = kWaves>
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
  for (int w = 0; w < W; w++)
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

struct Found {
  int index;
  double f, total;
};

// The first index within vectors [v0, v1) where `base` and the running sum of f
// pass `target` (the last with f > 0 where rounding leaves none): the vectors
// in order over all threads, then one thread's.
template <class E, class F>
__device__ __forceinline__ Found find_within(const RowView<E>& row, int v0, int v1, double base,
                                             double target, Lds& s, F f) {
  __syncthreads();
  if (threadIdx.x == 0) s.out_i[0] = -1;
  const int each = (v1 - v0 + kThreads - 1) / kThreads;
  const int a = min(v0 + (int)threadIdx.x * each, v1), b = min(a + each, v1);
  double mine = 0.0;
  int tail = -1;
  double tail_f = 0.0;
  for (int v = a; v < b; v++) {
    row.each(row.load(v, v1), v * RowView<E>::VEC - row.shift, [&](float x, int idx) {
      const double y = f(x, idx);
      mine += y;
      if (y > 0.0) {
        tail = idx;
        tail_f = y;
      }
    });
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
        row.each(row.load(v, v1), v * RowView<E>::VEC - row.shift, [&](float x, int idx) {
          const double y = f(x, idx);
          sum += y;
          if (y > 0.0 && sum > target && s.out_i[0] < 0) {
            s.out_i[0] = idx;
            s.out_d[0] = y;
          }
        });
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
  const Found r{s.out_i[0], s.out_d[0], 0.0};
  __syncthreads();
  return r;
}

// The first index where the running sum of f(value, index) >= 0 in index order
// passes `share` of the total (SHARE) or `share` itself, by a walk of the row
// and one of the 16th that holds it.  Every thread gets the index (-1: the sum
// is zero), its f and the total.
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
  const int v0 = ws * per;
  const Found in = find_within(row, v0, min(v0 + per, row.vectors), base, target, s, f);
  r.index = in.index;
  r.f = in.f;
  return r;
}

// s.key2 / s.index2 to s.key / s.index in index order.  (Four listed tokens a
// read here and below: the loops run at the LDS latency otherwise.)
__device__ __forceinline__ void sort_list(Lds& s, int n) {
  const int i = threadIdx.x;
  if (i >= n && i < (n + 3) / 4 * 4) s.index2[i] = INT32_MAX;
  __syncthreads();
  if (i < n) {
    const int me = s.index2[i];
    int at = 0;
#pragma unroll 4
    for (int j = 0; j < n; j += 4) {
      const int4 o = *reinterpret_cast<const int4*>(&s.index2[j]);
      at += (o.x < me) + (o.y < me) + (o.z < me) + (o.w < me);
    }
    s.key[at] = s.key2[i];
    s.index[at] = me;
  }
  __syncthreads();
}

// Gathers the tokens for which `in` holds into s.key2 / s.index2, in no order;
// their number, or kList + 1 for more than fit.
template <bool LIGHT, class E, class P>
__device__ __forceinline__ int collect(const RowView<E>& row, Lds& s, P in) {
  const int wave = threadIdx.x >> 6;
  const int per = (row.vectors + kWaves - 1) / kWaves;
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  row.template walk<LIGHT>(min(wave * per, row.vectors), min((wave + 1) * per, row.vectors),
                           [&](float v, int i) {
    if (in(v, i)) {
      const uint32_t n = atomicAdd(&s.n, 1u);
      if (n < kList) {
        s.key2[n] = key_of(v);
        s.index2[n] = i;
      }
    }
  });
  __syncthreads();
  return (int)min(s.n, (uint32_t)kList + 1);
}

// The same into s.key / s.index in index order.
template <class E, class P>
__device__ __forceinline__ int gather(const RowView<E>& row, Lds& s, P in) {
  const int n = collect<false>(row, s, in);
  if (n <= kList) sort_list(s, n);
  return n;
}

// The listed tokens' weights to s.weight, and the list filled up to a multiple
// of four with tokens before which every other comes.  Every thread calls it.
__device__ __forceinline__ void weigh_list(Lds& s, int n, const Weight& weight) {
  const int i = threadIdx.x;
  if (i < (n + 3) / 4 * 4) {
    if (i >= n) s.key[i] = 0;
    s.weight[i] = i < n ? weight.of(value_of_key(s.key[i])) : 0.0;
  }
  __syncthreads();
}

// Rank of listed token i among the n listed (falling value, rising index) and
// the weight of those before it.
__device__ __forceinline__ void rank_of(const Lds& s, int n, int i, uint32_t& rank, double& above) {
  const uint32_t k = s.key[i];
  uint32_t r = 0;
  double a = 0.0;
#pragma unroll 2
  for (int j = 0; j < n; j += 4) {
    const uint4 o = *reinterpret_cast<const uint4*>(&s.key[j]);
    const double2 w0 = *reinterpret_cast<const double2*>(&s.weight[j]);
    const double2 w1 = *reinterpret_cast<const double2*>(&s.weight[j + 2]);
    const bool b0 = o.x > k || (o.x == k && j < i), b1 = o.y > k || (o.y == k && j + 1 < i);
    const bool b2 = o.z > k || (o.z == k && j + 2 < i), b3 = o.w > k || (o.w == k && j + 3 < i);
    r += (uint32_t)b0 + b1 + b2 + b3;
    a += b0 ? w0.x : 0.0;
    a += b1 ? w0.y : 0.0;
    a += b2 ? w1.x : 0.0;
    a += b3 ? w1.y : 0.0;
  }
  rank = r;
  above = a;
}

// Narrows the last kept token down to a key and an index, over the tokens of
// `kept`: the k-th of them (BY_COUNT), or the one whose weight, with all before
// it, reaches `m`.  `ready`: the first histogram is there.
template <bool BY_COUNT, class E>
__device__ __forceinline__ Kept last_kept(const RowView<E>& row, const Weight& weight, Kept kept,
                                          uint32_t k, double m, double fixed, Lds& s,
                                          bool ready = false) {
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
    if (!ready) {
      clear_histogram(s);
      row.walk(w0, w1, [&](float v, int i) {
        const int b = bin_of(v);
        if (b < kBins && weight.bin(v) < kBins && kept.has(key_of(v), i)) {
          atomicAdd(&s.count[b], 1u);
          atomicAdd(&s.mass[b], to_fixed(weight.of(v), fixed));
        }
      });
      __syncthreads();
    }
    ready = false;
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
      if (i == 0) s.found = -1;
      weigh_list(s, n, weight);
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

// ---- few rows: a row in slices ---------------------------------------------
//
// One workgroup walks a row of 128256 at some 20 us a time where weights are
// needed.  With fewer rows than fill the chip, a row is cut into slices of
// vectors, a workgroup each, in three launches before the row's own:
//  max      the slice's max, and for top-k each thread's;
//  weights  top-k above kList, or top-p: the slice's histogram, of tokens or of
//           weight, and its total; the last workgroup of a row joins them and
//           finds the bin that holds the last kept token;
//           no filter, or min-p alone: the slice's total;
//  gather   the tokens in that bin into a list per slice, and the slice's weight
//           before it.
// The row's workgroup then has the lists to compare, and the slices' weights
// to find the one that holds the token, which alone it walks.
// Which way a row goes is told by its parameters.  Rows with k up to kList take
// the threads' maxima and one light walk by their own workgroup; one whose list would be too long (flat rows, ties), or with
// both a large k and top-p, is walked whole by its workgroup.

enum class Way { kTop, kTopK, kRank, kNucleus, kTotals, kWhole };

struct RowParams {
  float T, p;
  double u, min_p;
  int k;
  bool has_k, has_p;
  Way way;
  __device__ __forceinline__ RowParams(const SampleArgs& a, int r) {
    // (all five loads at once: a branch round each would wait for each)
    const float tv = (a.temperature ? a.temperature : a.u)[r], uv = a.u[r];
    const int32_t kv = (a.top_k ? a.top_k : reinterpret_cast<const int32_t*>(a.u))[r];
    const float pv = (a.top_p ? a.top_p : a.u)[r], mv = (a.min_p ? a.min_p : a.u)[r];
    T = a.temperature ? tv : 1.f;
    u = uv;
    k = a.top_k ? kv : 0;
    p = a.top_p ? pv : 1.f;
    min_p = a.min_p && mv > 0.f ? fmin((double)mv, 1.0) : 0.0;
    has_k = k > 0 && k < a.V;
    has_p = p < 1.f;
    if (!(T >= kMinTemperature))
      way = Way::kTop;
    else if (has_k)
      way = k <= kList ? Way::kTopK : has_p ? Way::kWhole : Way::kRank;
    else
      way = has_p ? Way::kNucleus : Way::kTotals;
  }
  // tokens of less weight are never the last of a nucleus (half of it: sums
  // are rounded)
  __device__ __forceinline__ double least(int V) const {
    return 0.5 * (1.0 - fmax((double)p, 0.0)) / (double)V;
  }
};

struct SliceInfo {  // of a row
  float low, high;  // the values listed
  int lo;           // their first bin
  double below;     // what lies before them: weight (tokens, where top-k acts)
  double all;       // the row's weight
};

struct SliceArgs {
  SampleArgs a;
  int S;                      // slices of a row
  float* top;                 // [rows][S]
  int* first;                 // [rows][S]
  float* thread_top;          // [rows][S][kSliceThreads], where top-k acts
  double* total;              // [rows][S]; after the gather: the weight before bin lo
  unsigned long long* mass;   // [rows][S][kSliceBins] (tokens, where top-k acts)
  uint32_t* listed;           // [rows][S]
  uint2* list;                // [rows][S][kList]: key, index
  SliceInfo* info;            // [rows]
  uint32_t* arrived;          // [rows]
};

struct SliceLds {
  double power[kPowers];
  __attribute__((aligned(16))) unsigned long long mass[kSliceBins];
  double wave_d[kSliceWaves];
  uint32_t wave_u[kSliceWaves];
  float wave_f[kSliceWaves];
  int wave_i[kSliceWaves];
  int bin;
  uint32_t n, key;
  bool last;
};

template <class E>
struct SliceView {
  RowView<E> row;
  int v0, v1;  // the slice's vectors
  int w0, w1;  // the wave's
  __device__ __forceinline__ SliceView(const SliceArgs& sa, int r, int s)
      : row(sa.a.logits, r * sa.a.row_stride, sa.a.V) {
    const int per = (row.vectors + sa.S - 1) / sa.S;
    v0 = min(s * per, row.vectors);
    v1 = min(v0 + per, row.vectors);
    const int wave = threadIdx.x >> 6;
    const int wp = (v1 - v0 + kSliceWaves - 1) / kSliceWaves;
    w0 = min(v0 + wave * wp, v1);
    w1 = min(w0 + wp, v1);
  }
};

// (max, first index of it) over the lanes.
__device__ __forceinline__ void wave_top(float& x, int& i) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const float y = __shfl_xor(x, d, 64);
    const int j = __shfl_xor(i, d, 64);
    if (y > x || (y == x && (uint32_t)j < (uint32_t)i)) {
      x = y;
      i = j;
    }
  }
}

// The row's, from its slices'.
__device__ __forceinline__ void row_top(const SliceArgs& sa, int r, float& x, int& i) {
  const int lane = threadIdx.x & 63;
  x = -INFINITY;
  i = -1;
  if (lane < sa.S) {
    x = sa.top[r * sa.S + lane];
    i = sa.first[r * sa.S + lane];
  }
  wave_top(x, i);
}

// The bins of a nucleus: from the max down to the least weight that can be its
// last.  Of a larger k's: 2^-64 of the max, below which nothing is drawn.
__device__ __forceinline__ Weight slice_weight(const RowParams& q, float top, int V,
                                               const double* power) {
  Weight w(top, q.T, power);
  const float range =
      q.way == Way::kNucleus ? log2f((float)V / (1.f - fmaxf(q.p, 0.f))) + 2.f : 64.f;
  w.set_bins((float)kSliceBins / range, kSliceBins);
  return w;
}

template <class E>
__global__ __launch_bounds__(kSliceThreads) void sample_max_kernel(SliceArgs sa) {
  __shared__ SliceLds s;
  const int r = blockIdx.y, sl = blockIdx.x, tid = threadIdx.x;
  const SliceView<E> view(sa, r, sl);
  float x = -INFINITY;
  int i = -1;
  view.row.template walk<true>(view.w0, view.w1, [&](float v, int at) {
    if (v > x) {
      x = v;
      i = at;
    }
  });
  const size_t rs = (size_t)r * sa.S + sl;
  if (RowParams(sa.a, r).way == Way::kTopK) sa.thread_top[rs * kSliceThreads + tid] = x;
  wave_top(x, i);
  if ((tid & 63) == 0) {
    s.wave_f[tid >> 6] = x;
    s.wave_i[tid >> 6] = i;
  }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kSliceWaves; w++)
      if (s.wave_f[w] > x) {
        x = s.wave_f[w];
        i = s.wave_i[w];
      }
    sa.top[rs] = x;
    sa.first[rs] = i;
    if (sl == 0) sa.arrived[r] = 0;
  }
}

// The lowest key (of a finite value) in bins up to b; the max's is in bin 0.  A
// whole wave calls it: 63 places of the range at a time.
__device__ __forceinline__ uint32_t lowest_key(const Weight& weight, int b) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = key_of(-FLT_MAX), hi = key_of(weight.top);
#pragma unroll 1
  while (lo < hi) {
    const uint32_t step = (hi - lo) / 63 + 1;
    const uint32_t at = lane * step < hi - lo ? lo + lane * step : hi;  // (hi is one)
    const uint64_t in = __builtin_amdgcn_ballot_w64(weight.bin(value_of_key(at)) <= b);
    const int first = __builtin_ctzll(in);
    hi = __builtin_amdgcn_readlane(at, first);
    if (first > 0) lo = __builtin_amdgcn_readlane(at, first - 1) + 1;
  }
  return lo;
}

template <class E>
__global__ __launch_bounds__(kSliceThreads) void sample_weights_kernel(SliceArgs sa) {
  __shared__ SliceLds s;
  const int r = blockIdx.y, sl = blockIdx.x, tid = threadIdx.x;
  const RowParams q(sa.a, r);
  if (q.way == Way::kTop || q.way == Way::kWhole || q.way == Way::kTopK) return;
  float top;
  int first;
  row_top(sa, r, top, first);
  if (first < 0) return;
  fill_powers<kSliceThreads>(s.power);
  const SliceView<E> view(sa, r, sl);
  const size_t rs = (size_t)r * sa.S + sl;
  const Weight weight = slice_weight(q, top, sa.a.V, s.power);
  __syncthreads();
  double x = 0.0, all;
  if (q.way == Way::kTotals) {
    view.row.walk(view.w0, view.w1, [&](float v, int) {
      const double w = weight.of(v);
      x += w >= q.min_p ? w : 0.0;
    });
    block_scan<kSliceWaves>(x, s.wave_d, all);
    if (tid == 0) sa.total[rs] = all;
    return;
  }
  for (int i = tid; i < kSliceBins; i += kSliceThreads) s.mass[i] = 0;
  __syncthreads();
  const bool by_count = q.way == Way::kRank;
  const double fixed = by_count ? 1.0 : fixed_point(sa.a.V), least = q.least(sa.a.V);
  if (by_count) {
    view.row.walk(view.w0, view.w1, [&](float v, int) {
      const int b = weight.bin(v);
      if (b < kSliceBins) atomicAdd(&s.mass[b], 1ull);
    });
  } else {
    view.row.walk(view.w0, view.w1, [&](float v, int) {
      int n;
      const double w = weight.of(v, n);
      x += w;
      const int b = weight.bin_of(n);
      if (w >= least && b < kSliceBins) atomicAdd(&s.mass[b], to_fixed(w, fixed));
    });
  }
  block_scan<kSliceWaves>(x, s.wave_d, all);
  // Published by agent-scope stores, which write through; every wave waits for
  // its own before the arrival is counted.
  for (int i = tid; i < kSliceBins; i += kSliceThreads)
    __hip_atomic_store(sa.mass + rs * kSliceBins + i, s.mass[i], __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  if (tid == 0)
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(sa.total + rs),
                       __builtin_bit_cast(unsigned long long, all), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
  __syncthreads();
  if (tid == 0)
    s.last = __hip_atomic_fetch_add(sa.arrived + r, 1u, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)sa.S - 1;
  __syncthreads();
  if (!s.last) return;

  // ---- the row's histogram, and the bin of the last kept token
  constexpr int PER = kSliceBins / kSliceThreads;
  const size_t r0 = (size_t)r * sa.S;
  unsigned long long m[PER] = {};
#pragma unroll
  for (int i = 0; i < kMaxSlices; i++) {
    if (i >= sa.S) break;
#pragma unroll
    for (int j = 0; j < PER; j++)
      m[j] += __hip_atomic_load(sa.mass + (r0 + i) * kSliceBins + tid * PER + j, __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_AGENT);
  }
  all = 0.0;
#pragma unroll
  for (int i = 0; i < kMaxSlices; i++)
    if (i < sa.S)
      all += __builtin_bit_cast(
          double, __hip_atomic_load(reinterpret_cast<unsigned long long*>(sa.total + r0 + i),
                                    __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
  const double unit = 1.0 / fixed, target = by_count ? (double)q.k : (double)q.p * all;
  double wt = 0.0, unused;
#pragma unroll
  for (int j = 0; j < PER; j++) wt += (double)m[j] * unit;
  const double before = block_scan<kSliceWaves>(wt, s.wave_d, unused) - wt;
  if (tid == 0) s.bin = kSliceBins;
  __syncthreads();
  {
    double run = before;
#pragma unroll
    for (int j = 0; j < PER; j++) {
      run += (double)m[j] * unit;
      if (m[j] > 0 && run >= target) {
        atomicMin(&s.bin, tid * PER + j);
        break;
      }
    }
  }
  __syncthreads();
  // (no bin: fewer than k tokens have a weight; all bins are before the list)
  int lo = s.bin, hi = s.bin;
  if (q.min_p > 0.0) {
    // where w = min_p, give or take the bins' rounding
    const double at = -log2(q.min_p) * kPowers * (double)weight.bin_mul * (1.0 / 65536.0);
    const int b = at < (double)kSliceBins ? (int)at : kSliceBins;
    if (b + 1 < lo) {
      lo = max(b - 1, 0);
      hi = b + 1;
    } else if (b - 1 <= hi) {
      lo = max(min(lo, b - 1), 0);
    }
  }
  if (tid == min(lo / PER, kSliceThreads - 1)) {
    double w = before;
#pragma unroll
    for (int j = 0; j < PER; j++)
      if (tid * PER + j < lo) w += (double)m[j] * unit;
    sa.info[r].below = w;
    sa.info[r].lo = lo;
    sa.info[r].all = all;
  }
  // The values in those bins (bins rise as values fall), by bisection: two
  // compares tell in what follows.
  if (tid < 64) {
    const float low = value_of_key(lowest_key(weight, min(hi, kSliceBins - 1)));
    if (tid == 0) sa.info[r].low = low;
  } else if (tid < 128) {
    const float high =
        lo == 0 ? INFINITY : value_of_key(lowest_key(weight, min(lo, kSliceBins) - 1) - 1);
    if (tid == 64) sa.info[r].high = high;
  }
}

template <class E>
__global__ __launch_bounds__(kSliceThreads) void sample_gather_kernel(SliceArgs sa) {
  __shared__ SliceLds s;
  const int r = blockIdx.y, sl = blockIdx.x, tid = threadIdx.x;
  const RowParams q(sa.a, r);
  if (q.way != Way::kRank && q.way != Way::kNucleus) return;
  float top;
  int first;
  row_top(sa, r, top, first);
  if (first < 0) return;
  const SliceInfo info = sa.info[r];
  const SliceView<E> view(sa, r, sl);
  const size_t rs = (size_t)r * sa.S + sl;
  const Weight weight = slice_weight(q, top, sa.a.V, s.power);
  if (q.way == Way::kRank) fill_powers<kSliceThreads>(s.power);
  if (tid == 0) s.n = 0;
  __syncthreads();
  auto keep = [&](float v, int i) {
    const uint32_t n = atomicAdd(&s.n, 1u);
    if (n < kList) sa.list[rs * kList + n] = make_uint2(key_of(v), (uint32_t)i);
  };
  view.row.template walk<true>(view.w0, view.w1, [&](float v, int i) {
    if (v >= info.low && v <= info.high) keep(v, i);
  });
  // the slice's weight before the listed values
  double x = 0.0, below;
  if (q.way == Way::kRank) {
    view.row.walk(view.w0, view.w1, [&](float v, int) {
      if (v > info.high) x += weight.of(v);
    });
  } else {
    const double unit = 1.0 / fixed_point(sa.a.V);
#pragma unroll
    for (int j = 0; j < kSliceBins / kSliceThreads; j++) {
      const int i = tid + j * kSliceThreads;
      if (i < info.lo) x += (double)sa.mass[rs * kSliceBins + i] * unit;
    }
  }
  block_scan<kSliceWaves>(x, s.wave_d, below);
  if (tid == 0) sa.total[rs] = below;
  __syncthreads();
  if (tid == 0) sa.listed[rs] = s.n;
}

// The row's lists into s.key2 / s.index2; their number, or kList + 1 for more than
// fit.  s.upto[i]: tokens of slices 0 .. i.
__device__ __forceinline__ int join_lists(const SliceArgs& sa, int r, Lds& s) {
  const int lane = threadIdx.x & 63;
  const size_t r0 = (size_t)r * sa.S;
  uint32_t n = lane < sa.S ? sa.listed[r0 + lane] : 0;
  const bool over = __builtin_amdgcn_ballot_w64(n > (uint32_t)kList) != 0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t y = __shfl_up(n, d, 64);
    if (lane >= d) n += y;
  }
  const uint32_t total = __shfl(n, 63, 64);
  __syncthreads();
  if (threadIdx.x < 64) s.upto[lane] = n;
  __syncthreads();
  if (over || total > (uint32_t)kList) return kList + 1;
  const uint32_t i = threadIdx.x;
  if (i < total) {
    int sl = 0;
#pragma unroll
    for (int d = kMaxSlices / 2; d > 0; d >>= 1)
      if (s.upto[sl + d - 1] <= i) sl += d;
    const uint2 e = sa.list[(r0 + sl) * kList + (i - (sl > 0 ? s.upto[sl - 1] : 0))];
    s.key2[i] = e.x;
    s.index2[i] = (int)e.y;
  }
  __syncthreads();
  return (int)total;
}

// The token of a row whose whole kept weight is among n <= 64 listed tokens, by
// one wave without a barrier: s.key2 / s.index2 in any order.
__device__ __forceinline__ void finish_few(const SampleArgs& a, int r, const RowParams& q,
                                           const Weight& weight, int n, double all, Lds& s) {
  const int i = threadIdx.x;
  {
    const int me = i < n ? s.index2[i] : INT32_MAX;
    int at = 0;
    for (int j = 0; j < n; j++) at += __builtin_amdgcn_readlane(me, j) < me ? 1 : 0;
    if (i < n) {
      s.key[at] = s.key2[i];
      s.index[at] = me;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const uint32_t key = i < n ? s.key[i] : 0;
  double w = i < n ? weight.of(value_of_key(key)) : 0.0;
  const uint64_t wb = __builtin_bit_cast(uint64_t, w);
  uint32_t rank = 0;
  double above = 0.0;
  for (int j = 0; j < n; j++) {
    const uint32_t o = __builtin_amdgcn_readlane(key, j);
    const uint64_t b = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)wb, j) |
                       ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(wb >> 32), j)
                        << 32);
    const bool first = o > key || (o == key && j < i);
    rank += first ? 1u : 0u;
    above += first ? __builtin_bit_cast(double, b) : 0.0;
  }
  bool in = i < n && (!q.has_k || rank < (uint32_t)q.k);
  if (q.has_k && q.has_p) {
    all = in ? w : 0.0;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d, 64);
  }
  if (in && q.has_p) in = above < (double)q.p * all || rank == 0;
  if (in) in = w >= q.min_p && w > 0.0;
  double upto = in ? w : 0.0;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(upto, d, 64);
    if (i >= d) upto += y;
  }
  const double total = __shfl(upto, 63, 64);
  const uint64_t passed = __builtin_amdgcn_ballot_w64(in && upto > q.u * total);
  const uint64_t live = __builtin_amdgcn_ballot_w64(in);
  // (u at or above 1, or rounding: the last kept)
  const int at = passed ? __builtin_ctzll(passed) : 63 - __builtin_clzll(live);
  if (i == at) {
    a.tokens[r] = s.index[i];
    if (a.probs) a.probs[r] = (float)(w / total);
  }
}

// The lowest of the given maxima of parts of the row, kTops per thread, that at
// least k of them reach (to 8 bins): at least k tokens do.
constexpr int kTops = kMaxSlices * kSliceThreads / kThreads;

__device__ __forceinline__ float top_k_low(Lds& s, const Weight& weight, const float (&x)[kTops],
                                           int k) {
  constexpr int N = kBins / 8;
  const int tid = threadIdx.x;
  if (tid < N) s.count[tid] = 0;
  __syncthreads();
  int b[kTops];
#pragma unroll
  for (int i = 0; i < kTops; i++) {
    b[i] = weight.bin(x[i]);
    if (b[i] < kBins) atomicAdd(&s.count[b[i] / 8], 1u);
  }
  __syncthreads();
  if (tid < 64) {
    const uint4 c = *reinterpret_cast<const uint4*>(&s.count[4 * tid]);
    uint32_t x = c.x + c.y + c.z + c.w;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(x, d, 64);
      if (tid >= d) x += y;
    }
    const uint64_t m = __builtin_amdgcn_ballot_w64(x >= (uint32_t)k);
    if (tid == 0) {
      s.found = kBins;
      s.lo = 0xFFFFFFFFu;
    }
    if (m && tid == __builtin_ctzll(m)) {
      uint32_t run = x - c.w - c.z - c.y;  // with the first of the four
      int at = 0;
      if (run < (uint32_t)k) { run += c.y; at = 1; }
      if (at == 1 && run < (uint32_t)k) { run += c.z; at = 2; }
      if (at == 2 && run < (uint32_t)k) at = 3;
      s.found = 8 * (4 * tid + at) + 7;
    }
  }
  __syncthreads();
  const int cut = s.found;
  if (cut == kBins) return -FLT_MAX;  // fewer hold a token of weight: every one
  uint32_t low = 0xFFFFFFFFu;
#pragma unroll
  for (int i = 0; i < kTops; i++)
    if (b[i] <= cut) low = min(low, key_of(x[i]));
  if (low != 0xFFFFFFFFu) atomicMin(&s.lo, low);
  __syncthreads();
  return value_of_key(s.lo);
}

// A row's own workgroup: the whole row, or with SLICED what its slices leave.
template <class E, bool SLICED>
__global__ __launch_bounds__(kThreads) void sample_kernel(SliceArgs sa) {
  __shared__ Lds s;
  const SampleArgs& a = sa.a;
  const int r = blockIdx.x;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const RowView<E> row(a.logits, r * a.row_stride, a.V);
  const int per = (row.vectors + kWaves - 1) / kWaves;
  const int w0 = min(wave * per, row.vectors), w1 = min((wave + 1) * per, row.vectors);
  const RowParams q(a, r);

  fill_powers<kThreads>(s.power);
  // ---- the max, and its first index
  float part_top[kTops];  // maxima of parts of the row, for top-k
#pragma unroll
  for (int i = 0; i < kTops; i++) part_top[i] = -INFINITY;
  float top;
  int first;
  if constexpr (SLICED) {
    if (q.way == Way::kTopK) {
      const float* t = sa.thread_top + (size_t)r * sa.S * kSliceThreads;
#pragma unroll
      for (int i = 0; i < kTops; i++) {
        const int j = i * kThreads + threadIdx.x;
        if (j < sa.S * kSliceThreads) part_top[i] = t[j];
      }
    }
    row_top(sa, r, top, first);
  } else {
    float mine = -INFINITY;
    int at = -1;
    row.template walk<true>(w0, w1, [&](float v, int i) {
      if (v > mine) {
        mine = v;
        at = i;
      }
    });
    part_top[0] = mine;
    float x = mine;
    wave_top(x, at);
    if (lane == 0) {
      s.wave_f[wave] = x;
      s.wave_i[wave] = at;
    }
    __syncthreads();
    top = s.wave_f[0];
    first = s.wave_i[0];
#pragma unroll
    for (int w = 1; w < kWaves; w++)
      if (s.wave_f[w] > top) {
        top = s.wave_f[w];
        first = s.wave_i[w];
      }
  }
  if (first < 0 || q.way == Way::kTop) {  // nothing to draw from, or the max itself
    if (threadIdx.x == 0) {
      a.tokens[r] = first;
      if (a.probs) a.probs[r] = first < 0 ? 0.f : 1.f;
    }
    return;
  }
  __syncthreads();
  Weight weight(top, q.T, s.power);
  weight.set_bins(kBinsPerLog2, kBins);
  const double fixed = fixed_point(a.V);

  int token = -1;
  double w_token = 0.0, total = 0.0;
  int n = kList + 1;      // listed tokens
  double all = 0.0;       // the total that top-p is a share of (top-k: the list's)
  double below = 0.0;     // weight (where top-k acts, number) of the tokens before the listed
  bool ready = false;     // the whole row's histogram is there
  bool slices = false;    // the row's weight is in its slices, the list only its last part
  if (q.way == Way::kTopK) {
    const float low = top_k_low(s, weight, part_top, q.k);
    n = collect<true>(row, s, [&](float v, int) { return v >= low; });
  } else if constexpr (SLICED) {
    if (q.way == Way::kNucleus || q.way == Way::kRank) {
      const SliceInfo info = sa.info[r];
      n = join_lists(sa, r, s);
      all = info.all;
      below = info.below;
      slices = n <= kList && below > 0.0;
    } else if (q.way == Way::kTotals) {
      n = 0;
      slices = true;
    }
  } else if (q.way == Way::kNucleus) {
    const double least = q.least(a.V);
    clear_histogram(s);
    double x = 0.0;
    row.walk(w0, w1, [&](float v, int) {
      int e;
      const double w = weight.of(v, e);
      x += w;
      const int b = weight.bin_of(e);
      if (w >= least && b < kBins) {
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], to_fixed(w, fixed));
      }
    });
    block_scan(x, s.wave_d, all);
    ready = true;
    // (a little beyond p: the fixed-point sums are rounded)
    const BinAt b = find_bin<false>(s, 0, (double)q.p * all * (1.0 + 1e-9), 1.0 / fixed);
    if (b.bin < kBins && b.before + b.in <= (uint32_t)kList) {
      const float low = value_of_key(lowest_key(weight, b.bin));
      n = collect<true>(row, s, [&](float v, int) { return v >= low; });
    }
  }
  if (n <= 64 && !slices) {
    if (wave == 0) finish_few(a, r, q, weight, n, all, s);
    return;
  }
  if (n <= kList) {
    const int i = threadIdx.x;
    sort_list(s, n);
    if (i == 0) {
      s.found = kList;
      s.lo = 0;
    }
    weigh_list(s, n, weight);
    uint32_t rank = 0;
    double above = 0.0, w = 0.0;
    bool in = i < n;
    if (in) {
      rank_of(s, n, i, rank, above);
      w = s.weight[i];
      if (q.has_k) in = below + (double)rank < (double)q.k;
    }
    if (q.has_k && q.has_p) block_scan(in ? w : 0.0, s.wave_d, all);
    if (in && q.has_p) in = below + above < (double)q.p * all || (rank == 0 && below == 0.0);
    if (in) in = w >= q.min_p && w > 0.0;
    if (!slices) {
      const double upto = block_scan(in ? w : 0.0, s.wave_d, total);
      const double target = q.u * total;
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
      // The last kept token of the list, and with it the slices' weights.
      if (in) {
        atomicMax(&s.lo, rank + 1);
        s.index2[rank] = i;
      }
      if (i < n) s.weight[i] = in ? w : 0.0;
      __syncthreads();
      Kept kept;  // (of the list; none of it, where none of it is kept)
      kept.key = 0xFFFFFFFFu;
      kept.last = -1;
      if (s.lo > 0) {
        const int e = s.index2[s.lo - 1];
        kept.key = s.key[e];
        kept.last = s.index[e];
      }
      const bool totals = q.way == Way::kTotals;
      if (i < sa.S) {
        double x = sa.total[(size_t)r * sa.S + i];
        if (!totals)
          for (uint32_t j = i > 0 ? s.upto[i - 1] : 0; j < s.upto[i]; j++) x += s.weight[j];
        s.slice_w[i] = x;
      }
      __syncthreads();
      for (int j = 0; j < sa.S; j++) total += s.slice_w[j];
      const double target = q.u * total;
      int at = -1;
      double base = 0.0, run = 0.0;
      for (int j = 0; j < sa.S; j++) {
        const double x = s.slice_w[j];
        // (the last slice with weight takes what rounding leaves over)
        if (x > 0.0 && (at < 0 || !(run > target))) {
          at = j;
          base = run;
        }
        run += x;
      }
      const int sp = (row.vectors + sa.S - 1) / sa.S;
      const int v0 = min(max(at, 0) * sp, row.vectors), v1 = min(v0 + sp, row.vectors);
      const float high = totals ? INFINITY : sa.info[r].high;
      const Found f = find_within(row, v0, v1, base, target, s, [&](float v, int idx) {
        const double y = weight.of(v);
        if (totals) return y >= q.min_p ? y : 0.0;
        return v > high || kept.has(key_of(v), idx) ? y : 0.0;
      });
      token = f.index;
      w_token = f.f;
    }
  } else {
    Kept kept;
    if (q.has_k) kept = last_kept<true>(row, weight, kept, (uint32_t)q.k, 0.0, fixed, s);
    if (q.has_p) {
      if (!ready) {
        double x = 0.0;
        row.walk(w0, w1, [&](float v, int i) { x += kept.has(key_of(v), i) ? weight.of(v) : 0.0; });
        block_scan(x, s.wave_d, all);
      }
      kept = last_kept<false>(row, weight, kept, 0u, (double)q.p * all, fixed, s, ready);
    }
    const Found f = find_index<true>(row, q.u, s, [&](float v, int i) {
      if (!kept.has(key_of(v), i)) return 0.0;
      const double w = weight.of(v);
      return w >= q.min_p ? w : 0.0;
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

// ---- launch ------------------------------------------------------------------

struct Layout {
  int S = 1;  // 1: no slices
  size_t first = 0, thread_top = 0, total = 0, mass = 0, listed = 0, list = 0, info = 0,
         arrived = 0, bytes = 0;
};

// Some 1024 slices over all rows, 16 of a row at most, from 32768 tokens on:
// below, four launches cost what they save.  Measured on MI355X, us whole / in
// slices, fp32: one row of 32000, no filter 22 / 25, k = 50 16 / 25, p = 0.9 51 / 43;
// of 128256 55 / 27, 24 / 26, 222 / 44; 192 rows of 128256 68 / 74, 42 / 51, 246 /
// 122.
Layout layout_of(int rows, int V) {
  Layout l;
  int64_t S = (1024 + (int64_t)rows - 1) / rows;
  S = S < kMaxSlices ? S : kMaxSlices;
  if (V < 32768 || S < 2) return l;
  l.S = (int)S;
  const size_t n = (size_t)rows * S;
  size_t at = 0;
  auto put = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  put(n * 4);  // top
  l.first = put(n * 4);
  l.thread_top = put(n * 4 * kSliceThreads);
  l.total = put(n * 8);
  l.mass = put(n * 8 * kSliceBins);
  l.listed = put(n * 4);
  l.list = put(n * 8 * kList);
  l.info = put((size_t)rows * sizeof(SliceInfo));
  l.arrived = put((size_t)rows * 4);
  l.bytes = at;
  return l;
}

template <class E>
int launch_sample(const SliceArgs& sa, int rows, hipStream_t st) {
  if (sa.S < 2) {
    sample_kernel<E, false><<<dim3(rows), dim3(kThreads), 0, st>>>(sa);
    return launch_status();
  }
  const dim3 grid(sa.S, rows), block(kSliceThreads);
  sample_max_kernel<E><<<grid, block, 0, st>>>(sa);
  int s = launch_status();
  if (s != SDE_OK) return s;
  sample_weights_kernel<E><<<grid, block, 0, st>>>(sa);
  s = launch_status();
  if (s != SDE_OK) return s;
  sample_gather_kernel<E><<<grid, block, 0, st>>>(sa);
  s = launch_status();
  if (s != SDE_OK) return s;
  sample_kernel<E, true><<<dim3(rows), dim3(kThreads), 0, st>>>(sa);
  return launch_status();
}

}  // namespace smp
}  // namespace sde

extern "C" {

size_t sde_sample_workspace_size(int n_rows, int vocab) {
  using namespace sde::smp;
  if (n_rows < 1 || vocab < 1 || vocab > kMaxVocab || n_rows > (1 << 21)) return 0;
  return layout_of(n_rows, vocab).bytes;
}

int sde_sample(const void* d_logits, int64_t row_stride, int dtype, int n_rows, int vocab,
               const float* d_u, const float* d_temperature, const int32_t* d_top_k,
               const float* d_top_p, const float* d_min_p, int32_t* d_tokens, float* d_probs,
               void* d_workspace, size_t workspace_bytes, sde_stream_t stream) {
  using namespace sde::smp;
  if (n_rows < 0 || vocab < 1 || !sde::batch::known_dtype(dtype)) return SDE_ERR_INVALID_ARGUMENT;
  if (vocab > kMaxVocab || n_rows > (1 << 21)) return SDE_ERR_UNSUPPORTED;
  if (n_rows == 0) return SDE_OK;
  if (!d_logits || !d_u || !d_tokens || (n_rows > 1 && row_stride < vocab))
    return SDE_ERR_INVALID_ARGUMENT;
  if (reinterpret_cast<uintptr_t>(d_logits) % (size_t)sde::batch::elem_bytes(dtype) != 0)
    return SDE_ERR_INVALID_ARGUMENT;
  const Layout l = layout_of(n_rows, vocab);
  if (l.bytes > 0 && (!d_workspace || workspace_bytes < l.bytes ||
                      reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0))
    return SDE_ERR_WORKSPACE;
  SliceArgs sa{};
  sa.a = SampleArgs{d_logits, row_stride, vocab,   d_u,      d_temperature,
                    d_top_k,  d_top_p,    d_min_p, d_tokens, d_probs};
  sa.S = l.S;
  if (l.S > 1) {
    char* w = static_cast<char*>(d_workspace);
    sa.top = reinterpret_cast<float*>(w);
    sa.first = reinterpret_cast<int*>(w + l.first);
    sa.thread_top = reinterpret_cast<float*>(w + l.thread_top);
    sa.total = reinterpret_cast<double*>(w + l.total);
    sa.mass = reinterpret_cast<unsigned long long*>(w + l.mass);
    sa.listed = reinterpret_cast<uint32_t*>(w + l.listed);
    sa.list = reinterpret_cast<uint2*>(w + l.list);
    sa.info = reinterpret_cast<SliceInfo*>(w + l.info);
    sa.arrived = reinterpret_cast<uint32_t*>(w + l.arrived);
  }
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == SDE_F32) return launch_sample<sde::batch::f32_elem>(sa, n_rows, s);
  if (dtype == SDE_F16) return launch_sample<sde::batch::f16_elem>(sa, n_rows, s);
  return launch_sample<sde::batch::bf16_elem>(sa, n_rows, s);
}

}  // extern "C"
