// Attention of several requests' newest tokens over their own paged caches
// (sde_batch_attention): what sde_paged_attention does for one request, for
// n_seqs of them in one call, their lengths read on the device.
//
//   out[b, i] = sum_p softmax_p(q[b, i] . K[b, p] / sqrt(dph)) V[b, p],
//   p < len[b] - m + 1 + i        (query i of m)
//
// What bounds it is the cache: each K and V byte is read once and serves the
// G = nh / nkv query heads of its KV head (times m queries), a few operations
// per byte.  So:
//  * a workgroup takes (request, KV head, group of 16 rows, partition of the
//    positions); a wave takes every kWaves-th tile of 32 positions of it on
//    its own -- own buffers, no barrier in the loop -- and the waves' sums meet
//    in LDS at the end;
//  * K and V go from memory straight into LDS, two tiles ahead; a buffer is
//    filled again as soon as its tile is in registers, so some 24 KiB per
//    wave are in flight at head size 128 while it computes;
//  * one load covers whole token rows of the head (256 B at head size 128).
//    The lane that fetches a 16-byte unit is chosen so that the units of a row
//    lie swizzled in LDS: the K operand (16 tokens, one unit) and the
//    transposed V operand (4 tokens, 32 bytes) then use all banks;
//  * products are 16x16x32 fp16 MFMA: S^T = K q^T leaves a lane with one row's
//    logits of 8 positions, which are, in that order, its operand of
//    O^T = V^T P^T: the softmax needs no exchange but the running max's.  q is
//    scaled per row by a power of two and split into fp16 hi + lo parts, and so
//    are the weights, which keeps 22 bits of them; sums are fp32.  (fp16 and
//    bf16 q are their hi parts.)
//  * the max is raised only when a logit is 2^8 above it.
#include <algorithm>
#include <cmath>

#include "batch_common.hpp"
#include "sde/attention_device.hpp"

namespace sde {
namespace batch {

using attn::f4_t;
using attn::h8_t;
using attn::lds_s4_t;
using attn::s4_t;

constexpr int kRows = 16;       // rows (query, head in group) of a workgroup
constexpr int kTok = 32;        // positions per tile
constexpr int kTable = 1024;    // block table entries of a partition in LDS
constexpr int kMaxQueries = 64;
constexpr float kLazyMax = 8.f;     // log2 growth of a logit above the max that raises it
constexpr float kWeightShift = 7.f; // weights up to 2^(8 + 7): see batch weights below

struct BatchArgs {
  const uint16_t* pool;
  const int32_t* tables;
  const int32_t* lens;
  const void* q;
  void* out;
  float* partials;  // [n_seqs][nkv][R][n_parts][dph], then (max, sum) likewise
  int64_t q_stride, out_stride;
  int pool_blocks, bs, kv_dim, max_blocks, table_stride, n_seqs, max_len;
  int m, nh, nkv, G, R, dph, row_groups, n_parts, part_tokens;
  int dtype, wide_q, wide_out;
  uint32_t bs_magic;  // ceil(2^32 / bs), 0 for bs = 1
  float scale;        // log2(e) / sqrt(dph)
};

template <int DP>
struct Shape {
  static constexpr int UNITS = DP / 8;     // 16-byte units per token row
  static constexpr int KS = DP / 32;       // k-steps of the logits product
  static constexpr int FB = DP / 16;       // 16-feature blocks of the output
  static constexpr int ROWB = 2 * DP;      // bytes per staged row
  static constexpr int TILEB = kTok * ROWB;
  static constexpr int NL = TILEB / 1024;  // loads per wave and tile of K (or V)
  static constexpr int RING = 4 * TILEB;   // two tiles of K and V
  static constexpr int WAVES = DP > 128 ? 2 : 4;
};

// Which unit of token t's row lies at place u: u ^ swizzle(t).  16 tokens read
// at one unit, and 16 tokens read at two neighbouring units in halves, fall on
// all 64 banks whatever the row's length is beside 256 bytes.
template <int DP>
__device__ __forceinline__ int swizzle(int t) {
  if constexpr (Shape<DP>::UNITS % 16 == 0) return ((t & 3) << 2) | ((t >> 2) & 3);
  if constexpr (Shape<DP>::UNITS % 8 == 0) return (t >> 1) & 7;
  return (t >> 2) & 3;
}

// 16 bytes per lane from p straight into LDS, lane l's to lds_off + 16 l
// (wave-uniform).  Asynchronous (vmcnt); the memory clobber and the waits below
// order it.  m0 is reserved, which a clobber list may not name: nothing else
// here needs it.
__device__ __forceinline__ void load_to_lds(const uint16_t* p, uint32_t lds_off) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(lds_off), "v"(p)
      : "memory");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "vmcnt counts to 63");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// A lane's q operand elements, features 32 ks + 8 grp .. + 7 of one row, all
// loads ahead of their first use; features beyond the head's are zero.
template <class E, int KS>
__device__ __forceinline__ void load_q(const void* base, int64_t at, int grp, int dph, bool wide,
                                       float (&x)[KS][8]) {
  using T = typename E::type;
  const T* p = static_cast<const T*>(base) + at;
  T raw[KS][8];
  if (wide) {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; i++) {
        const uint4 v =
            reinterpret_cast<const uint4*>(p + min(32 * ks + 8 * grp, dph - 8))[i];
        __builtin_memcpy(reinterpret_cast<char*>(raw[ks]) + 16 * i, &v, 16);
      }
  } else {
#pragma unroll
    for (int ks = 0; ks < KS; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) raw[ks][e] = p[min(32 * ks + 8 * grp, dph - 8) + e];
  }
#pragma unroll
  for (int ks = 0; ks < KS; ks++)
#pragma unroll
    for (int e = 0; e < 8; e++) x[ks][e] = 32 * ks + 8 * grp < dph ? E::get(raw[ks][e]) : 0.f;
}

// Four outputs; 16- or 8-byte stores where the rows allow.
__device__ __forceinline__ void store4(void* p, int64_t i, float4 x, int dtype, bool wide) {
  if (dtype == SDE_F32) {
    float* d = static_cast<float*>(p) + i;
    if (wide) {
      *reinterpret_cast<float4*>(d) = x;
    } else {
      d[0] = x.x;
      d[1] = x.y;
      d[2] = x.z;
      d[3] = x.w;
    }
    return;
  }
  uint16_t e[4];
  if (dtype == SDE_F16) {
    e[0] = f16_elem::put(x.x);
    e[1] = f16_elem::put(x.y);
    e[2] = f16_elem::put(x.z);
    e[3] = f16_elem::put(x.w);
  } else {
    e[0] = bf16_elem::put(x.x);
    e[1] = bf16_elem::put(x.y);
    e[2] = bf16_elem::put(x.z);
    e[3] = bf16_elem::put(x.w);
  }
  uint16_t* d = static_cast<uint16_t*>(p) + i;
  if (wide) {
    uint2 raw;
    __builtin_memcpy(&raw, e, 8);
    *reinterpret_cast<uint2*>(d) = raw;
  } else {
#pragma unroll
    for (int k = 0; k < 4; k++) d[k] = e[k];
  }
}

// Row `row` of KV head kvh of request b: its query and q head.
__device__ __forceinline__ int64_t row_at(const BatchArgs& a, int b, int kvh, int row,
                                          int64_t stride) {
  const int i = row / a.G;
  return (int64_t)(b * a.m + i) * stride + (int64_t)(kvh * a.G + row - i * a.G) * a.dph;
}

// FULL: the head has DP features (else fewer: the rest of each staged row is
// zero).
template <int DP, bool FULL>
__global__ __launch_bounds__(64 * Shape<DP>::WAVES) void batch_attention_kernel(BatchArgs a) {
  using Sh = Shape<DP>;
  constexpr int W = Sh::WAVES;
  __shared__ __attribute__((aligned(1024))) char ring[W * Sh::RING];
  __shared__ int32_t tab[kTable];
  __shared__ float2 sums[W][kRows];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int l16 = lane & 15, grp = lane >> 4;

  // KV heads fastest: neighbours read neighbouring slices of the same tokens.
  int n = blockIdx.x;
  int u = wave_uniform(n / a.nkv);
  const int kvh = n - u * a.nkv;
  n = u;
  u = wave_uniform(n / a.row_groups);
  const int r0 = (n - u * a.row_groups) * kRows;
  const int b = wave_uniform(u / a.n_parts);
  const int part = u - b * a.n_parts;
  const int rows = min(kRows, a.R - r0);

  // Length, table entries and q are all on their way before any is used.
  const int p0 = part * a.part_tokens;
  const int b0 = wave_uniform(p0 / a.bs);
  const int n_tab = min(wave_uniform((p0 + a.part_tokens - 1) / a.bs) + 1, a.max_blocks) - b0;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int32_t* const trow = a.tables + (int64_t)b * a.table_stride + b0;
  for (int i = tid; i < n_tab; i += 64 * W) tab[i] = trow[i];
  const bool real = l16 < rows;
  const int row = r0 + l16;
  float qx[Sh::KS][8];
  {
    // (rows beyond the group's read its first: their logits are masked)
    const int64_t at = row_at(a, b, kvh, real ? row : r0, a.q_stride);
    if (a.dtype == SDE_F32)
      load_q<f32_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
    else if (a.dtype == SDE_F16)
      load_q<f16_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
    else
      load_q<bf16_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
  }
  const int p1 = min(p0 + a.part_tokens, len);
  if (p0 >= p1) {  // nothing here (the combine leaves this partition out)
    if (a.n_parts == 1)
      for (int i = tid; i < rows * (a.dph / 4); i += 64 * W) {
        const int r = i / (a.dph / 4);
        store4(a.out, row_at(a, b, kvh, r0 + r, a.out_stride) + 4 * (i - r * (a.dph / 4)),
               make_float4(0.f, 0.f, 0.f, 0.f), a.dtype, a.wide_out);
      }
    return;
  }
  // q scaled by a power of two to a largest element in [1, 2): any finite q
  // fits fp16's range, and the hi + lo split keeps 22 bits of it.
  float mx = 0.f;
#pragma unroll
  for (int ks = 0; ks < Sh::KS; ks++)
#pragma unroll
    for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qx[ks][e]));
  mx = attn::groups_max(mx);
  // (a row of zeros or with an infinity keeps its scale)
  const int ex = mx > 0.f && mx < INFINITY ? ilogbf(mx) : 0;
  const float row_scale = ldexpf(a.scale, ex);
  h8_t qh[Sh::KS], ql[Sh::KS];
#pragma unroll
  for (int ks = 0; ks < Sh::KS; ks++) {
#pragma unroll
    for (int e = 0; e < 8; e++) qx[ks][e] = ldexpf(qx[ks][e], -ex);
    attn::split_h8(qx[ks], qh[ks], ql[ks]);
  }
  const bool lo_q = a.dtype == SDE_F32;   // fp16 and bf16 elements are their hi parts

  int bad = 0;  // pages outside the pool: their positions are left out
  for (int i = tid; i <= wave_uniform((p1 - 1) / a.bs) - b0; i += 64 * W)
    if ((uint32_t)tab[i] >= (uint32_t)a.pool_blocks) {
      tab[i] = -1;
      bad = 1;
    }
  bad = wave_uniform(__syncthreads_or(bad));

  // ---- this wave's tiles: p0 + 32 (wave + W i)
  const int tiles = (p1 - p0 + kTok - 1) / kTok;
  const int nt = wave_uniform(tiles > wave ? (tiles - wave + W - 1) / W : 0);
  char* const mine = ring + wave * Sh::RING;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)mine;
  const int base_rel = p0 - b0 * a.bs;  // position p0, counted from block b0
  const int units = a.dph / 8;
  if (!FULL) {
    // the features beyond the head's, which no load reaches
    const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < Sh::RING / 1024; i++)
      reinterpret_cast<uint4*>(mine)[64 * i + lane] = z;
    wait_lds();
  }
  auto page_of = [&](int rel, int& slot) {  // table entry and slot of p0's block + rel
    const int lb = a.bs_magic ? (int)__umulhi((uint32_t)rel, a.bs_magic) : rel;
    slot = rel - lb * a.bs;
    return tab[lb];
  };
  // Pool row (in tokens) of tile i's position lane % 32; positions past the
  // last take the last's, pages outside the pool its first row: addresses are
  // always in the pool, and such positions are masked.
  auto rows_of = [&](int i) {
    const int at = min(kTok * (wave + W * i) + (lane & 31), p1 - p0 - 1);
    int slot;
    const int page = page_of(base_rel + at, slot);
    return page < 0 ? 0u : (uint32_t)page * (2u * (uint32_t)a.bs) + (uint32_t)slot;
  };
  const uint16_t* const head = a.pool + (int64_t)kvh * a.dph;
  auto load_rows = [&](uint32_t row_of_lane, uint32_t skip, uint32_t lds_off) {
#pragma unroll
    for (int j = 0; j < Sh::NL; j++) {
      const int at = 64 * j + lane;
      const int t = at / Sh::UNITS;
      const int unit = (at - t * Sh::UNITS) ^ swizzle<DP>(t);
      const uint32_t r =
          (uint32_t)__builtin_amdgcn_ds_bpermute(4 * t, (int)row_of_lane) + skip;
      // (every load has a lane within the head: the counts below are exact)
      if (FULL || unit < units)
        load_to_lds(head + (uint64_t)r * (uint32_t)a.kv_dim + 8 * unit, lds_off + 1024 * j);
    }
  };
  uint32_t prow = 0;
  if (nt > 0) {
    prow = rows_of(0);
    load_rows(prow, 0, lds0);
    load_rows(prow, a.bs, lds0 + Sh::TILEB);
  }
  if (nt > 1) {
    prow = rows_of(1);
    load_rows(prow, 0, lds0 + 2 * Sh::TILEB);
    load_rows(prow, a.bs, lds0 + 3 * Sh::TILEB);
  }

  const int qi = row / a.G;                       // the row's query
  const int last = real ? len - a.m + qi : -1;    // and the last position it sees
  const int all_see = len - a.m;                  // the last that every query sees
  f4_t o[Sh::FB];
#pragma unroll
  for (int fb = 0; fb < Sh::FB; fb++) o[fb] = f4_t{0.f, 0.f, 0.f, 0.f};
  // Weights are 2^(logit - ref), ref = max - kWeightShift: below 2^15, and
  // fp16's quantum of their lo parts is 2^-32 of the largest.
  float ref = 0.f, raise = -INFINITY, l = 0.f;
  const int vt = 4 * grp + (l16 >> 2);  // transposed V reads: this lane's token
  const int vu = (l16 & 3) >> 1, vsub = 8 * (l16 & 1);

  for (int i = 0; i < nt; i++) {
    const char* kst = mine + (i & 1) * 2 * Sh::TILEB;
    const uint32_t dst = lds0 + (uint32_t)(i & 1) * 2 * Sh::TILEB;
    const int at0 = kTok * (wave + W * i);
    if (i + 1 < nt)
      wait_loads<3 * Sh::NL>();
    else
      wait_loads<Sh::NL>();
    // (a long head's operands are read in halves, within the registers)
    constexpr bool kHalves = Sh::KS > 4;
    h8_t k8[kHalves ? 1 : 2][Sh::KS];
    f4_t s[2], s2[2];
    auto read_k = [&](int h, h8_t(&k)[Sh::KS]) {
      const int t = 16 * h + l16;
#pragma unroll
      for (int ks = 0; ks < Sh::KS; ks++)
        k[ks] = *reinterpret_cast<const h8_t*>(
            kst + t * Sh::ROWB + 16 * ((4 * ks + grp) ^ swizzle<DP>(t)));
    };
    auto logits = [&](int h, const h8_t(&k)[Sh::KS]) {
      s[h] = s2[h] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < Sh::KS; ks++)
        s[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[ks], qh[ks], s[h], 0, 0, 0);
      if (lo_q) {
#pragma unroll
        for (int ks = 0; ks < Sh::KS; ks++)
          s2[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[ks], ql[ks], s2[h], 0, 0, 0);
      }
    };
    read_k(0, k8[0]);
    if constexpr (kHalves) logits(0, k8[0]);
    read_k(1, k8[kHalves ? 0 : 1]);
    if (i + 2 < nt) prow = rows_of(i + 2);
    wait_lds();
    if (i + 2 < nt) load_rows(prow, 0, dst);
    if constexpr (!kHalves) logits(0, k8[0]);
    logits(1, k8[kHalves ? 0 : 1]);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (s[e >> 2][e & 3] + s2[e >> 2][e & 3]) * row_scale;

    // positions some row does not see, or past the end, or in no page
    const bool edge = bad || p0 + at0 + kTok - 1 > all_see;
    uint32_t seen = 0xFF;  // bit e: position e of this lane exists
    if (edge) {
      seen = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int at = at0 + 16 * (e >> 2) + 4 * grp + (e & 3);
        bool in = at < p1 - p0;
        if (bad) {
          int slot;
          in = in && page_of(base_rel + min(at, p1 - p0 - 1), slot) >= 0;
        }
        seen |= in ? 1u << e : 0u;
        x[e] = in && p0 + at <= last ? x[e] : -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
    if (__builtin_amdgcn_ballot_w64(top > raise) != 0) {
      top = attn::groups_max(top);
      if (top > raise) {
        // (a row's first logits: its sums are zero, and the factor too)
        const float to = fmaxf(top - kWeightShift, raise == -INFINITY ? -INFINITY : ref);
        const float f = raise == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - to);
        ref = to;
        raise = to + kWeightShift + kLazyMax;
        l *= f;
#pragma unroll
        for (int fb = 0; fb < Sh::FB; fb++) o[fb] *= f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; e++) {
      x[e] = __builtin_amdgcn_exp2f(x[e] - ref);
      l += x[e];
    }
    h8_t ph, pl;
    attn::split_h8(x, ph, pl);

    // outstanding after this tile's V: tile i + 1, and K of i + 2
    if (i + 2 < nt)
      wait_loads<3 * Sh::NL>();
    else if (i + 1 < nt)
      wait_loads<2 * Sh::NL>();
    else
      wait_loads<0>();
    const char* vst = kst + Sh::TILEB;
    typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
    u4_t v8[Sh::FB];
#pragma unroll
    for (int fb = 0; fb < Sh::FB; fb++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int t = 16 * h + vt;
        const s4_t r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(
            vst + t * Sh::ROWB + 16 * ((2 * fb + vu) ^ swizzle<DP>(t)) + vsub));
        const uint2 d = __builtin_bit_cast(uint2, r);
        v8[fb][2 * h] = d.x;
        v8[fb][2 * h + 1] = d.y;
      }
    wait_lds();
    if (i + 2 < nt) load_rows(prow, a.bs, dst + Sh::TILEB);

    if (edge) {
      // What lies at positions that do not exist must not meet a weight of 0
      // (0 x Inf): it becomes 0.  A non-finite element that some rows see and
      // others do not takes a product per query.
      uint32_t some = 0;  // bit e: hidden from a row of the workgroup
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (p0 + at0 + 16 * (e >> 2) + 4 * grp + (e & 3) > all_see) some |= 1u << e;
      uint32_t hit = 0;
#pragma unroll
      for (int d = 0; d < 4; d++) {
        const uint32_t two = seen >> (2 * d);
        const uint32_t keep = (two & 1 ? 0xFFFFu : 0u) | (two & 2 ? 0xFFFF0000u : 0u);
        const uint32_t st = some >> (2 * d);
        const uint32_t sm = (st & 1 ? 0xFFFFu : 0u) | (st & 2 ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int fb = 0; fb < Sh::FB; fb++) {
          v8[fb][d] &= keep;
          hit |= attn::nonfinite_h2(v8[fb][d] & sm);
        }
      }
      if (__builtin_amdgcn_ballot_w64(hit != 0) != 0) {
        const int i0 = r0 / a.G, i1 = (r0 + rows - 1) / a.G;
#pragma unroll 1
        for (int w = i0; w <= i1; w++) {
          uint32_t keep[4];
#pragma unroll
          for (int d = 0; d < 4; d++) {
            const int at = p0 + at0 + 16 * (d >> 1) + 4 * grp + 2 * (d & 1);
            const int lim = len - a.m + w;
            keep[d] = (at <= lim ? 0xFFFFu : 0u) | (at + 1 <= lim ? 0xFFFF0000u : 0u);
          }
#pragma unroll
          for (int fb = 0; fb < Sh::FB; fb++) {
            u4_t v = v8[fb];
#pragma unroll
            for (int d = 0; d < 4; d++) v[d] &= keep[d];
            f4_t y = f4_t{0.f, 0.f, 0.f, 0.f};
            y = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v), ph, y, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v), pl, y, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) o[fb][e] += qi == w ? y[e] : 0.f;
          }
        }
        continue;
      }
    }
#pragma unroll
    for (int fb = 0; fb < Sh::FB; fb++)
      o[fb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v8[fb]), ph, o[fb], 0,
                                                     0, 0);
#pragma unroll
    for (int fb = 0; fb < Sh::FB; fb++)
      o[fb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v8[fb]), pl, o[fb], 0,
                                                     0, 0);
  }

  // ---- the waves' sums meet in LDS (every tile has been read)
  l = attn::groups_sum(l);
  constexpr int C = DP / 4;  // 16-byte units per row
  static_assert(kRows * DP * 4 <= Sh::RING, "a wave's sums fit its ring");
  float4* const mo = reinterpret_cast<float4*>(mine);
#pragma unroll
  for (int fb = 0; fb < Sh::FB; fb++)
    mo[l16 * C + ((4 * fb + grp) ^ (l16 & 7))] =
        make_float4(o[fb][0], o[fb][1], o[fb][2], o[fb][3]);
  if (grp == 0) sums[wave][l16] = make_float2(raise == -INFINITY ? -INFINITY : ref, l);
  __syncthreads();
  for (int i = tid; i < rows * C; i += 64 * W) {
    const int r = i / C, c = i - r * C;
    if (4 * c >= a.dph) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < W; w++) top = fmaxf(top, sums[w][r].x);
    float lt = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float2 s = sums[w][r];
      // (a wave that saw nothing of the row has zeros; a sum of NaN logits
      // alone, which raised no max, stays)
      const float f = s.x == -INFINITY ? (s.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(s.x - top);
      const float4 z =
          reinterpret_cast<const float4*>(ring + w * Sh::RING)[r * C + (c ^ (r & 7))];
      lt += s.y * f;
      y.x += z.x * f;
      y.y += z.y * f;
      y.z += z.z * f;
      y.w += z.w * f;
    }
    if (a.n_parts == 1) {
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      y.x *= inv;
      y.y *= inv;
      y.z *= inv;
      y.w *= inv;
      store4(a.out, row_at(a, b, kvh, r0 + r, a.out_stride) + 4 * c, y, a.dtype, a.wide_out);
    } else {
      const size_t pr = (((size_t)b * a.nkv + kvh) * a.R + r0 + r) * a.n_parts + part;
      *reinterpret_cast<float4*>(a.partials + pr * a.dph + 4 * c) = y;
      if (c == 0)
        reinterpret_cast<float2*>(a.partials + (size_t)a.n_seqs * a.nkv * a.R * a.n_parts *
                                                   a.dph)[pr] = make_float2(top, lt);
    }
  }
}

// Joins a row's partitions, in order: one thread per (row, 4 features).
__global__ __launch_bounds__(256) void batch_combine_kernel(BatchArgs a) {
  const int C = a.dph / 4;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t kr = i / C;
  if (kr >= (size_t)a.n_seqs * a.nkv * a.R) return;
  const int c = (int)(i - kr * C);
  const int bk = (int)(kr / a.R), row = (int)(kr - (size_t)bk * a.R);
  const int b = bk / a.nkv, kvh = bk - b * a.nkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int P = (len + a.part_tokens - 1) / a.part_tokens;
  const float* acc = a.partials + kr * a.n_parts * a.dph + 4 * c;
  const float2* ml = reinterpret_cast<const float2*>(
                         a.partials + (size_t)a.n_seqs * a.nkv * a.R * a.n_parts * a.dph) +
                     kr * a.n_parts;
  float top = -INFINITY, l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < P; p0 += 4) {
    float2 v[4];
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int p = min(p0 + k, P - 1);
      v[k] = ml[p];
      x[k] = *reinterpret_cast<const float4*>(acc + (size_t)p * a.dph);
    }
    float to = top;
#pragma unroll
    for (int k = 0; k < 4; k++) to = fmaxf(to, v[k].x);
    const float old = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(top - to);
    top = to;
    l *= old;
    y.x *= old;
    y.y *= old;
    y.z *= old;
    y.w *= old;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      if (p0 + k >= P) continue;
      const float f =
          v[k].x == -INFINITY ? (v[k].y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(v[k].x - top);
      l += v[k].y * f;
      y.x += x[k].x * f;
      y.y += x[k].y * f;
      y.z += x[k].z * f;
      y.w += x[k].w * f;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store4(a.out, row_at(a, b, kvh, row, a.out_stride) + 4 * c,
         make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv), a.dtype, a.wide_out);
}

struct BatchPlan {
  int row_groups = 1, n_parts = 1, part_tokens = kTok;
};

// Positions per partition: enough partitions for some kFill workgroups over
// all requests (each of which may be much shorter than max_len), none shorter
// than kMinPart positions, and none longer than its table entries in LDS.
constexpr int kFill = 2048;
constexpr int kMinPart = 256;

BatchPlan batch_plan(int n_seqs, int nkv, int R, int max_len, int bs) {
  BatchPlan p;
  p.row_groups = (R + kRows - 1) / kRows;
  const int64_t units = std::max<int64_t>(1, (int64_t)n_seqs * nkv * p.row_groups);
  int64_t tokens = ((int64_t)max_len + kFill / units) / std::max<int64_t>(1, kFill / units);
  tokens = std::max<int64_t>(tokens, kMinPart);
  tokens = std::min<int64_t>(tokens, (int64_t)(kTable - 2) * bs);
  tokens = std::min<int64_t>(tokens, 1 << 20);  // (page_of's division)
  tokens = std::max<int64_t>(tokens / kTok * kTok, kTok);
  p.n_parts = (int)std::max<int64_t>(1, ((int64_t)max_len + tokens - 1) / tokens);
  p.part_tokens = (int)tokens;
  return p;
}

size_t batch_partial_bytes(const BatchPlan& p, int n_seqs, int nkv, int R, int dph) {
  return p.n_parts > 1 ? (size_t)n_seqs * nkv * R * p.n_parts * (size_t)(dph + 2) * sizeof(float)
                       : 0;
}

template <int DP>
void launch(const BatchArgs& a, unsigned grid, hipStream_t s) {
  const dim3 block(64 * Shape<DP>::WAVES);
  if (a.dph == DP)
    batch_attention_kernel<DP, true><<<dim3(grid), block, 0, s>>>(a);
  else
    batch_attention_kernel<DP, false><<<dim3(grid), block, 0, s>>>(a);
}

bool batch_shape(int n_seqs, int nh, int nkv, int dph, int n_queries, int max_len, int bs) {
  return n_seqs >= 0 && nh >= 1 && nkv >= 1 && nh % nkv == 0 && dph >= 8 && dph % 8 == 0 &&
         dph <= 256 && n_queries >= 1 && n_queries <= kMaxQueries && max_len >= 0 && bs >= 1 &&
         bs <= kMaxBlockSize && nh <= (1 << 20) / dph;
}

}  // namespace batch
}  // namespace sde

extern "C" {

size_t sde_batch_attention_workspace_size(int n_seqs, int nh, int nkv, int dph, int n_queries,
                                          int max_len, int block_size) {
  using namespace sde::batch;
  if (!batch_shape(n_seqs, nh, nkv, dph, n_queries, max_len, block_size)) return 0;
  const int R = n_queries * (nh / nkv);
  return batch_partial_bytes(batch_plan(n_seqs, nkv, R, max_len, block_size), n_seqs, nkv, R, dph);
}

int sde_batch_attention(const sde_batch_pool* pool, const int32_t* d_lens, int n_queries,
                        int max_len, int dtype, const void* d_q, int64_t q_stride, void* d_out,
                        int64_t out_stride, int nh, int nkv, int dph, void* d_workspace,
                        size_t workspace_bytes, sde_stream_t stream) {
  using namespace sde::batch;
  const int st = check_pool(pool);
  if (st != SDE_OK) return st;
  if (nh < 1 || nkv < 1 || dph < 1 || nh % nkv != 0 || n_queries < 1 || max_len < 0 ||
      !known_dtype(dtype) || (int64_t)nkv * dph != pool->kv_dim)
    return SDE_ERR_INVALID_ARGUMENT;
  if (!batch_shape(pool->n_seqs, nh, nkv, dph, n_queries, max_len, pool->block_size))
    return SDE_ERR_UNSUPPORTED;
  if (max_len > (int64_t)pool->max_blocks * pool->block_size) return SDE_ERR_CAPACITY;
  // (K and V units are 16-byte loads)
  if (reinterpret_cast<uintptr_t>(pool->pool) % 16 != 0) return SDE_ERR_UNSUPPORTED;
  if (pool->n_seqs == 0) return SDE_OK;
  if (!d_lens || !d_q || !d_out) return SDE_ERR_INVALID_ARGUMENT;
  const int64_t width = (int64_t)nh * dph;
  if (q_stride < width || out_stride < width) return SDE_ERR_INVALID_ARGUMENT;
  const size_t e = elem_bytes(dtype);
  if (reinterpret_cast<uintptr_t>(d_q) % e != 0 || reinterpret_cast<uintptr_t>(d_out) % e != 0)
    return SDE_ERR_INVALID_ARGUMENT;
  if ((int64_t)pool->n_seqs * n_queries > INT32_MAX) return SDE_ERR_UNSUPPORTED;

  BatchArgs a;
  const int R = n_queries * (nh / nkv);
  const BatchPlan p = batch_plan(pool->n_seqs, nkv, R, max_len, pool->block_size);
  const size_t need = batch_partial_bytes(p, pool->n_seqs, nkv, R, dph);
  if (need > 0 && (!d_workspace || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0))
    return SDE_ERR_WORKSPACE;
  const int64_t grid = (int64_t)pool->n_seqs * nkv * p.row_groups * p.n_parts;
  if (grid > (1 << 23)) return SDE_ERR_UNSUPPORTED;  // (a launch counts its threads in 32 bits)
  a.pool = pool->pool;
  a.tables = pool->tables;
  a.lens = d_lens;
  a.q = d_q;
  a.out = d_out;
  a.partials = static_cast<float*>(d_workspace);
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.pool_blocks = pool->pool_blocks;
  a.bs = pool->block_size;
  a.kv_dim = pool->kv_dim;
  a.max_blocks = pool->max_blocks;
  a.table_stride = pool->table_stride;
  a.n_seqs = pool->n_seqs;
  a.max_len = max_len;
  a.m = n_queries;
  a.nh = nh;
  a.nkv = nkv;
  a.G = nh / nkv;
  a.R = R;
  a.dph = dph;
  a.row_groups = p.row_groups;
  a.n_parts = p.n_parts;
  a.part_tokens = p.part_tokens;
  a.dtype = dtype;
  a.wide_q = aligned(d_q, q_stride, dtype, 16) ? 1 : 0;
  a.wide_out = aligned(d_out, out_stride, dtype, 4 * e) ? 1 : 0;
  a.bs_magic = a.bs > 1 ? (uint32_t)((0x100000000ull + a.bs - 1) / a.bs) : 0;
  a.scale = (float)(1.4426950408889634 / std::sqrt((double)dph));
  const hipStream_t s = (hipStream_t)stream;
  const unsigned g = (unsigned)grid;
  if (dph <= 32)
    launch<32>(a, g, s);
  else if (dph <= 64)
    launch<64>(a, g, s);
  else if (dph <= 96)
    launch<96>(a, g, s);
  else if (dph <= 128)
    launch<128>(a, g, s);
  else if (dph <= 160)
    launch<160>(a, g, s);
  else if (dph <= 192)
    launch<192>(a, g, s);
  else
    launch<256>(a, g, s);
  const int ls = sde::launch_status();
  if (ls != SDE_OK || p.n_parts == 1) return ls;
  const int64_t threads = (int64_t)pool->n_seqs * nkv * R * (dph / 4);
  if ((threads + 255) / 256 > (1 << 23)) return SDE_ERR_UNSUPPORTED;
  batch_combine_kernel<<<dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s>>>(a);
  return sde::launch_status();
}

}  // extern "C"
