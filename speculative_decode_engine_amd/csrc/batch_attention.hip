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
//  * a workgroup takes (request, KV head, up to 48 rows, partition of the
//    positions); each of its waves takes every W-th tile of 32 positions of it
//    on its own -- own buffers, no barrier in the loop -- and the waves' sums
//    meet in LDS at the end;
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
//
// Measured on MI355X (graph replays over three inputs), 32/8 heads of 128 where
// not said: 96 requests up to 8K, bf16, 1.64 GB: 318 us, 5.2 TB/s (a copy of 4 GiB
// runs at 4.7); 16 up to 4K, 149 MB: 38 us, 3.9 TB/s; one of 32K: 35 us, 3.9; the
// 5-query verify of 3 up to 32K, 28/4 heads, 144 MB: 47 us, 3.1 TB/s, the combine's
// 5 in it.
// Short of the bandwidth there: some 4 us pass before a workgroup's first tile is
// there (length and table, then K), and partitions end unevenly.
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

constexpr int kRows = 16;       // rows (query, head in group) of a group: one MFMA's
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
// zero).  W waves, RG row groups, whose rows share every tile's operands.
template <int DP, bool FULL, int W, int RG>
__global__ __launch_bounds__(64 * W) void batch_attention_kernel(BatchArgs a) {
  using Sh = Shape<DP>;
  __shared__ __attribute__((aligned(1024))) char ring[W * Sh::RING];
  __shared__ int32_t tab[kTable];
  __shared__ float2 sums[W][RG * kRows];
  __shared__ int first_bad[DP], any_bad;
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
  const int r0 = (n - u * a.row_groups) * (RG * kRows);
  const int b = wave_uniform(u / a.n_parts);
  const int part = u - b * a.n_parts;
  const int rows = min(RG * kRows, a.R - r0);
  const int groups = (rows + kRows - 1) / kRows;

  // Length, table entries and q are all on their way before any is used.
  const int p0 = part * a.part_tokens;
  const int b0 = wave_uniform(p0 / a.bs);
  const int n_tab = min(wave_uniform((p0 + a.part_tokens - 1) / a.bs) + 1, a.max_blocks) - b0;
  const int len = min(max(a.lens[b], 0), a.max_len);
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
  const int32_t* const trow = a.tables + (int64_t)b * a.table_stride + b0;
  for (int i = tid; i < n_tab; i += 64 * W) tab[i] = trow[i];
  for (int i = tid; i < DP; i += 64 * W) first_bad[i] = INT32_MAX;
  if (tid == 0) any_bad = 0;

  // q scaled by a power of two to a largest element in [1, 2): any finite q
  // fits fp16's range, and the hi + lo split keeps 22 bits of it.
  h8_t qh[RG][Sh::KS], ql[RG][Sh::KS];
  float row_scale[RG];
  int last[RG];  // the last position that this lane's row sees
#pragma unroll
  for (int g = 0; g < RG; g++) {
    const int row = r0 + kRows * g + l16;
    const bool real = kRows * g + l16 < rows;
    last[g] = real ? len - a.m + row / a.G : -1;
    // (rows beyond the group's read its first: their logits are masked)
    float qx[Sh::KS][8];
    const int64_t at = row_at(a, b, kvh, real ? row : r0, a.q_stride);
    if (a.dtype == SDE_F32)
      load_q<f32_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
    else if (a.dtype == SDE_F16)
      load_q<f16_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
    else
      load_q<bf16_elem>(a.q, at, grp, a.dph, a.wide_q, qx);
    float mx = 0.f;
#pragma unroll
    for (int ks = 0; ks < Sh::KS; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qx[ks][e]));
    mx = attn::groups_max(mx);
    // (a row of zeros or with an infinity keeps its scale)
    const int ex = mx > 0.f && mx < INFINITY ? ilogbf(mx) : 0;
    row_scale[g] = ldexpf(a.scale, ex);
#pragma unroll
    for (int ks = 0; ks < Sh::KS; ks++) {
#pragma unroll
      for (int e = 0; e < 8; e++) qx[ks][e] = ldexpf(qx[ks][e], -ex);
      attn::split_h8(qx[ks], qh[g][ks], ql[g][ks]);
    }
  }
  const bool lo_q = a.dtype == SDE_F32;  // fp16 and bf16 elements are their hi parts

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

  const int all_see = len - a.m;  // the last position that every query sees
  f4_t o[RG][Sh::FB];
#pragma unroll
  for (int g = 0; g < RG; g++)
#pragma unroll
    for (int fb = 0; fb < Sh::FB; fb++) o[g][fb] = f4_t{0.f, 0.f, 0.f, 0.f};
  // Weights are 2^(logit - ref), ref = max - kWeightShift: below 2^15, and
  // fp16's quantum of their lo parts is 2^-32 of the largest.
  float ref[RG], raise[RG], l[RG];
#pragma unroll
  for (int g = 0; g < RG; g++) {
    ref[g] = l[g] = 0.f;
    raise[g] = -INFINITY;
  }
  const int vt = 4 * grp + (l16 >> 2);  // transposed V reads: this lane's token
  const int vu = (l16 & 3) >> 1, vsub = 8 * (l16 & 1);

  for (int i = 0; i < nt; i++) {
    char* const kst = mine + (i & 1) * 2 * Sh::TILEB;
    char* const vst = kst + Sh::TILEB;
    const uint32_t dst = lds0 + (uint32_t)(i & 1) * 2 * Sh::TILEB;
    const int at0 = kTok * (wave + W * i);
    if (i + 1 < nt)
      wait_loads<3 * Sh::NL>();
    else
      wait_loads<Sh::NL>();
    // (a long head's operands are read in halves, within the registers)
    constexpr bool kHalves = Sh::KS > 4;
    h8_t k8[kHalves ? 1 : 2][Sh::KS];
    f4_t s[RG][2];
    auto read_k = [&](int h, h8_t(&k)[Sh::KS]) {
      const int t = 16 * h + l16;
#pragma unroll
      for (int ks = 0; ks < Sh::KS; ks++)
        k[ks] = *reinterpret_cast<const h8_t*>(
            kst + t * Sh::ROWB + 16 * ((4 * ks + grp) ^ swizzle<DP>(t)));
    };
    auto logits = [&](int h, const h8_t(&k)[Sh::KS]) {
#pragma unroll
      for (int g = 0; g < RG; g++) {
        if (g > 0 && g >= groups) break;
        f4_t x = f4_t{0.f, 0.f, 0.f, 0.f}, y = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < Sh::KS; ks++)
          x = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[ks], qh[g][ks], x, 0, 0, 0);
        if (lo_q) {
#pragma unroll
          for (int ks = 0; ks < Sh::KS; ks++)
            y = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[ks], ql[g][ks], y, 0, 0, 0);
        }
        s[g][h] = x + y;
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

    // positions some row does not see, or past the end, or in no page
    const bool edge = bad || p0 + at0 + kTok - 1 > all_see;
    uint32_t there = 0xFF;  // bit e: position e of this lane exists
    if (edge) {
      there = 0;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int at = at0 + 16 * (e >> 2) + 4 * grp + (e & 3);
        bool in = at < p1 - p0;
        if (bad) {
          int slot;
          in = in && page_of(base_rel + min(at, p1 - p0 - 1), slot) >= 0;
        }
        there |= in ? 1u << e : 0u;
      }
    }
    h8_t ph[RG], pl[RG];
#pragma unroll
    for (int g = 0; g < RG; g++) {
      if (g > 0 && g >= groups) break;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = s[g][e >> 2][e & 3] * row_scale[g];
      if (edge) {
#pragma unroll
        for (int e = 0; e < 8; e++)
          x[e] = (there >> e & 1) && p0 + at0 + 16 * (e >> 2) + 4 * grp + (e & 3) <= last[g]
                     ? x[e]
                     : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; e++) top = fmaxf(top, x[e]);
      if (__builtin_amdgcn_ballot_w64(top > raise[g]) != 0) {
        top = attn::groups_max(top);
        if (top > raise[g]) {
          // (a row's first logits: its sums are zero, and the factor too)
          const float to = top - kWeightShift;
          const float f = raise[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref[g] - to);
          ref[g] = to;
          raise[g] = to + kWeightShift + kLazyMax;
          l[g] *= f;
#pragma unroll
          for (int fb = 0; fb < Sh::FB; fb++) o[g][fb] *= f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; e++) {
        x[e] = __builtin_amdgcn_exp2f(x[e] - ref[g]);
        l[g] += x[e];
      }
      attn::split_h8(x, ph[g], pl[g]);
    }

    // outstanding after this tile's V: tile i + 1, and K of i + 2
    if (i + 2 < nt)
      wait_loads<3 * Sh::NL>();
    else if (i + 1 < nt)
      wait_loads<2 * Sh::NL>();
    else
      wait_loads<0>();
    if (edge) {
      // What lies at positions that do not exist must not meet a weight of 0
      // (0 x Inf): it becomes 0.  So does an element that is not finite at a
      // position hidden from some row, and the rows that do see it are marked:
      // by feature, the first such position.
#pragma unroll 1
      for (int j = 0; j < Sh::NL; j++) {
        const int place = 64 * j + lane;
        const int t = place / Sh::UNITS;
        const int at = at0 + t;
        bool in = at < p1 - p0;
        if (bad && in) {
          int slot;
          in = page_of(base_rel + at, slot) >= 0;
        }
        uint4* const v = reinterpret_cast<uint4*>(vst + 16 * place);
        const uint4 x = *v;
        if (!in) {
          *v = make_uint4(0, 0, 0, 0);
        } else if (p0 + at > all_see && (attn::nonfinite_h2(x.x) | attn::nonfinite_h2(x.y) |
                                         attn::nonfinite_h2(x.z) | attn::nonfinite_h2(x.w)) != 0) {
          const int unit = (place - t * Sh::UNITS) ^ swizzle<DP>(t);
          uint16_t* const e = reinterpret_cast<uint16_t*>(v);
#pragma unroll 1
          for (int k = 0; k < 8; k++)
            if (attn::nonfinite_h2(e[k]) != 0) {
              e[k] = 0;
              atomicMin(&first_bad[8 * unit + k], p0 + at);
              any_bad = 1;
            }
        }
      }
      wait_lds();
    }
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
#pragma unroll
    for (int g = 0; g < RG; g++) {
      if (g > 0 && g >= groups) break;
#pragma unroll
      for (int fb = 0; fb < Sh::FB; fb++)
        o[g][fb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v8[fb]), ph[g],
                                                          o[g][fb], 0, 0, 0);
#pragma unroll
      for (int fb = 0; fb < Sh::FB; fb++)
        o[g][fb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, v8[fb]), pl[g],
                                                          o[g][fb], 0, 0, 0);
    }
  }

  // ---- the waves' sums meet in LDS (every tile has been read)
  constexpr int C = DP / 4;  // 16-byte units per row
  static_assert(RG * kRows * DP * 4 <= Sh::RING, "a wave's sums fit its ring");
  float4* const mo = reinterpret_cast<float4*>(mine);
#pragma unroll
  for (int g = 0; g < RG; g++) {
    const float lt = attn::groups_sum(l[g]);
#pragma unroll
    for (int fb = 0; fb < Sh::FB; fb++)
      mo[(kRows * g + l16) * C + ((4 * fb + grp) ^ (l16 & 7))] =
          make_float4(o[g][fb][0], o[g][fb][1], o[g][fb][2], o[g][fb][3]);
    if (grp == 0)
      sums[wave][kRows * g + l16] = make_float2(raise[g] == -INFINITY ? -INFINITY : ref[g], lt);
  }
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
    if (any_bad) {
      const int see = len - a.m + (r0 + r) / a.G;
      const int* fb = &first_bad[4 * c];
      y.x = fb[0] <= see ? NAN : y.x;
      y.y = fb[1] <= see ? NAN : y.y;
      y.z = fb[2] <= see ? NAN : y.z;
      y.w = fb[3] <= see ? NAN : y.w;
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

// Joins a row's partitions: a workgroup per row, kJoin of its threads side by
// side over a 16-byte unit's partitions, whose sums meet in LDS in order.  Eight
// for more than eight partitions (43 each of 420 rows: 15.6 us by one, 5.2 by
// eight; 5 each of 96 x 32 rows: 5.7 and 9.1).
template <int kJoin>
__global__ __launch_bounds__(64 * kJoin) void batch_combine_kernel(BatchArgs a) {
  __shared__ float4 part_y[kJoin][64];
  __shared__ float2 part_ml[kJoin];
  const int kr = blockIdx.x;
  const int c = threadIdx.x & 63, j = threadIdx.x >> 6;
  const int bk = kr / a.R, row = kr - bk * a.R;
  const int b = bk / a.nkv, kvh = bk - b * a.nkv;
  const int len = min(max(a.lens[b], 0), a.max_len);
  const int P = (len + a.part_tokens - 1) / a.part_tokens;
  const bool in = 4 * c < a.dph;
  const float* acc = a.partials + (size_t)kr * a.n_parts * a.dph + (in ? 4 * c : 0);
  const float2* ml = reinterpret_cast<const float2*>(
                         a.partials + (size_t)a.n_seqs * a.nkv * a.R * a.n_parts * a.dph) +
                     (size_t)kr * a.n_parts;
  float top = -INFINITY, l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = j; p0 < P; p0 += 4 * kJoin) {
    float2 v[4];
    float4 x[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int p = min(p0 + k * kJoin, P - 1);
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
      if (p0 + k * kJoin >= P) continue;
      const float f =
          v[k].x == -INFINITY ? (v[k].y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(v[k].x - top);
      l += v[k].y * f;
      y.x += x[k].x * f;
      y.y += x[k].y * f;
      y.z += x[k].z * f;
      y.w += x[k].w * f;
    }
  }
  part_y[j][c] = y;
  if (c == 0) part_ml[j] = make_float2(top, l);
  __syncthreads();
  if (j > 0 || !in) return;
  top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kJoin; k++) top = fmaxf(top, part_ml[k].x);
  l = 0.f;
  y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kJoin; k++) {
    const float2 v = part_ml[k];
    const float4 x = part_y[k][c];
    const float f = v.x == -INFINITY ? (v.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(v.x - top);
    l += v.y * f;
    y.x += x.x * f;
    y.y += x.y * f;
    y.z += x.z * f;
    y.w += x.w * f;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  store4(a.out, row_at(a, b, kvh, row, a.out_stride) + 4 * c,
         make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv), a.dtype, a.wide_out);
}

struct BatchPlan {
  int per_group = 1;  // row groups of a workgroup
  int row_groups = 1, n_parts = 1, part_tokens = kTok;
};

// Row groups of a workgroup: rows up to 48 together, so that K and V are read
// once; as many as the registers hold without scratch, whose loads would wait
// for the tiles' (two above head size 128, one above 192).
int groups_per(int R, int dph) {
  const int g = (R + kRows - 1) / kRows;
  const int most = dph > 192 ? 1 : dph > 128 ? 2 : 3;
  const int n = (g + most - 1) / most;
  return (g + n - 1) / n;
}

// Partitions.  With few (request, KV head, row group) units, some 640 workgroups
// over max_len: at the requests' own lengths that is about the two per CU that
// run at once.  Positions: 256 or more.  From a unit per CU on a partition only
// evens out the requests' lengths: up to 4096 workgroups, over 512 positions or
// more, from two units per CU on over 1024.  Measured on MI355X, us per call by
// the number of workgroups aimed at (512 / 768 / 4096), 32/8 heads of 128: 16
// requests up to 4K 41.1 / 39.1 / 45 (640: 38.4), one of 32K 35.6 / 36 / 45, the
// 5-query verify of 3 up to 32K 55 / 66 / 90 (640, with a faster combine: 47), 40 up
// to 2K 61.9 / 61 / 56.5, 96 up to 8K 367 / 367 / 323 (318 with the faster combine);
// 128 up to 1K with 1024 positions at least 67, with 256 98.  No partition has more
// table entries than fit LDS.
BatchPlan batch_plan(int n_seqs, int nkv, int R, int dph, int max_len, int bs) {
  BatchPlan p;
  p.per_group = groups_per(R, dph);
  p.row_groups = (R + kRows * p.per_group - 1) / (kRows * p.per_group);
  const int64_t units = std::max<int64_t>(1, (int64_t)n_seqs * nkv * p.row_groups);
  const int64_t parts = std::max<int64_t>(1, (units < 256 ? 640 : 4096) / units);
  int64_t tokens = ((int64_t)max_len + parts - 1) / parts;
  tokens = std::max<int64_t>(tokens, units < 256 ? 256 : units < 512 ? 512 : 1024);
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

template <int DP, int W, int RG>
void launch_groups(const BatchArgs& a, unsigned grid, hipStream_t s) {
  if (a.dph == DP)
    batch_attention_kernel<DP, true, W, RG><<<dim3(grid), dim3(64 * W), 0, s>>>(a);
  else
    batch_attention_kernel<DP, false, W, RG><<<dim3(grid), dim3(64 * W), 0, s>>>(a);
}
template <int DP, int W>
void launch_w(const BatchArgs& a, int per_group, unsigned grid, hipStream_t s) {
  if constexpr (DP <= 128)
    if (per_group == 3) return launch_groups<DP, W, 3>(a, grid, s);
  if constexpr (DP <= 192)
    if (per_group == 2) return launch_groups<DP, W, 2>(a, grid, s);
  launch_groups<DP, W, 1>(a, grid, s);
}
template <int DP>
void launch(const BatchArgs& a, int per_group, unsigned grid, hipStream_t s) {
  // Waves by what lies in LDS (16, 32, 64 KiB per wave at 64, 128, 256), two
  // workgroups or more to a CU: one starts or ends while the other streams.  (16
  // requests up to 4K, 32/8 heads of 128: 4 / 2 / 1 waves 45.7 / 39.1 / 42.6 us; 8
  // up to 2K, 32/4 of 64: 11.5 / 13.0 / 13.9; 8 up to 4K, 16/8 of 256: 2 / 1 waves
  // 45.8 / 38.9.)
  launch_w<DP, (DP <= 64 ? 4 : DP <= 128 ? 2 : 1)>(a, per_group, grid, s);
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
  return batch_partial_bytes(batch_plan(n_seqs, nkv, R, dph, max_len, block_size), n_seqs, nkv, R, dph);
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
  const BatchPlan p = batch_plan(pool->n_seqs, nkv, R, dph, max_len, pool->block_size);
  const size_t need = batch_partial_bytes(p, pool->n_seqs, nkv, R, dph);
  if (need > 0 && (!d_workspace || workspace_bytes < need ||
                   reinterpret_cast<uintptr_t>(d_workspace) % 16 != 0))
    return SDE_ERR_WORKSPACE;
  const int64_t grid = (int64_t)pool->n_seqs * nkv * p.row_groups * p.n_parts;
  // (a launch counts its threads in 32 bits)
  if (grid > (1 << 23) || (int64_t)pool->n_seqs * nkv * R > (1 << 22)) return SDE_ERR_UNSUPPORTED;
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
    launch<32>(a, p.per_group, g, s);
  else if (dph <= 64)
    launch<64>(a, p.per_group, g, s);
  else if (dph <= 96)
    launch<96>(a, p.per_group, g, s);
  else if (dph <= 128)
    launch<128>(a, p.per_group, g, s);
  else if (dph <= 160)
    launch<160>(a, p.per_group, g, s);
  else if (dph <= 192)
    launch<192>(a, p.per_group, g, s);
  else
    launch<256>(a, p.per_group, g, s);
  const int ls = sde::launch_status();
  if (ls != SDE_OK || p.n_parts == 1) return ls;
  const dim3 joins((unsigned)(pool->n_seqs * nkv * R));
  if (p.n_parts > 8)
    batch_combine_kernel<8><<<joins, dim3(512), 0, s>>>(a);
  else
    batch_combine_kernel<1><<<joins, dim3(64), 0, s>>>(a);
  return sde::launch_status();
}

}  // extern "C"
