// Causal attention of packed prompts (sde_prompt_attention): sequence b's rows
// are starts[b] .. starts[b+1]-1 of q, k, v and out, and query i of it sees keys
// 0 .. i of it.  q head h reads KV head h * nkv / nh.
//
//   out[i] = sum_{j <= i} softmax_j(q_i . k_j / sqrt(dph)) v_j
//
// What bounds it is arithmetic, 4 dph multiply-adds per visible (row, key) on
// the matrix cores and, beside them, one exponential, so:
//  * a workgroup takes 128 rows -- (query, head in group) pairs of one KV head,
//    so that the heads of a group share every key tile and short prompts still
//    fill their tiles -- or 256 of long prompts, and each of its waves 32;
//  * tiles of 64 keys go from memory straight into LDS, one or three ahead of the
//    one multiplied (one barrier a tile), K and V rows swizzled so that operand
//    reads use all banks;
//  * S^T = K q^T by 32x32x16 MFMA leaves a lane with one row's logits; in that
//    order they are its operand of O^T = V^T P^T, so the softmax exchanges
//    nothing but the row's max and sum, between two lanes;
//  * logits, weights and sums are fp32; a weight is rounded once to the inputs'
//    type to enter its product (half a step of it, as the output's rounding).
//    The scale enters with the max in one multiply-add ahead of exp2.  The max
//    is raised only when a logit is 2^8 above it.
//  * row tiles start from the end of the packed rows, where they are longest;
//    the KV head is the fastest index: with 8 of them each XCD's L2 holds one's.
//
// Measured on MI355X: one prompt of 8192 tokens, 32/8 heads of 128: 526 to 556 us
// in fp16 by the card, 988 to 1045 TFLOP/s, 504 us in bf16, 1091 (a square product
// of 8192 reaches 1184 and 1238 in the library), the matrix cores busy for half of
// the SIMDs' cycles and the vector unit for 44 %, no bank conflicts; of 4096 147
// us, 934 TFLOP/s; six uneven prompts of 4093 tokens in all 47 us, 580 TFLOP/s:
// some 3000 cycles pass from a tile's logits to its output in one wave, and short
// prompts have too few waves to hide them.
#include <cmath>

#include "batch_common.hpp"
#include "sde/attention_device.hpp"

namespace sde {
namespace prompt {

using attn::lds_s4_t;
using attn::s4_t;
using batch::bf16_elem;
using batch::f16_elem;

typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

constexpr int kTok = 64;            // keys per tile
constexpr int kBatch = 2;             // k-steps whose operands are read together
constexpr float kLazyMax = 8.f;

struct PromptArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* out;
  const int32_t* starts;
  int64_t q_stride, k_stride, v_stride, out_stride;
  int n_tokens, n_seqs, nkv, G, dph;
  int rows, tiles;  // rows of a workgroup, row tiles
  float scale;  // log2(e) / sqrt(dph)
};

// WAVES of 32 rows.  Eight: one workgroup to a CU, four tiles of keys in LDS, three
// on their way.  Four: two workgroups to a CU (head sizes up to 128), two tiles
// each.
template <int DP, int WAVES>
struct Shape {
  static constexpr int THREADS = 64 * WAVES;
  static constexpr int ROWS = 32 * WAVES;
  static constexpr int STAGES = WAVES == 8 ? 4 : 2;
  static constexpr int UNITS = DP / 8;      // 16-byte units per staged row
  static constexpr int KS = DP / 16;        // k-steps of the logits product
  static constexpr int DB = DP / 32;        // 32-feature blocks of the output
  static constexpr int ROWB = 2 * DP;
  static constexpr int TILEB = kTok * ROWB;
  static_assert(TILEB % (16 * THREADS) == 0, "a tile is whole loads of every thread");
  static constexpr int NU = TILEB / (16 * THREADS);  // loads per thread, K or V
};

// Place of unit u of token t's row: u ^ swizzle(t).  Any 16 tokens read at one
// unit, and 8 tokens read over 64 bytes, use all 64 banks evenly.
template <int DP>
__device__ __forceinline__ int swizzle(int t) {
  if constexpr (DP % 128 == 0) return ((t & 3) << 2) | ((t >> 2) & 3);
  if constexpr (DP % 64 == 0) return (((t >> 1) & 1) << 2) | ((t >> 2) & 3);
  return (t >> 2) & 3;
}

// 16 bytes per lane from p + off straight into LDS, lane l's to lds_off + 16 l.
// Asynchronous (vmcnt); m0 is reserved: nothing else here needs it.
__device__ __forceinline__ void load_to_lds(const uint16_t* p, uint32_t off, uint32_t lds_off) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "s"(lds_off), "v"(off), "s"(p)
      : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N < 64, "vmcnt counts to 63");
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

template <bool BF16>
__device__ __forceinline__ f16v mfma(u4v a, u4v b, f16v c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8v, a),
                                                   __builtin_bit_cast(b8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8v, a),
                                                  __builtin_bit_cast(h8v, b), c, 0, 0, 0);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (BF16) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), b2));
  } else {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{x, y}), h2));
  }
}

// Whether either half of a pair of elements is not finite.
template <bool BF16>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t x) {
  if constexpr (BF16) return ((x & 0x7F807F80u) + 0x00800080u) & 0x80008000u;
  return attn::nonfinite_h2(x);
}

__device__ __forceinline__ float half_max(float x) {
  const int v = __builtin_bit_cast(int, x);
  const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__builtin_bit_cast(float, (int)h[0]), __builtin_bit_cast(float, (int)h[1]));
}

// Row tiles are numbered so that sequence b's begin at
// first_tile(b) = starts[b] * G / rows + b: at least as many numbers as it has
// tiles, without a sum over the sequences before it.
__device__ __forceinline__ int64_t first_tile(const PromptArgs& a, int b) {
  const int s = min(max(a.starts[b], 0), a.n_tokens);
  return (int64_t)s * a.G / a.rows + b;
}

// The last sequence whose tiles begin at or before t (starts[0]'s at worst).
__device__ __forceinline__ int sequence_of(const PromptArgs& a, int64_t t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.n_seqs;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lo + lane * step;
    const bool in = lane * step < n && first_tile(a, i) <= t;
    const uint64_t m = __builtin_amdgcn_ballot_w64(in);
    const int last = m ? 63 - __builtin_clzll(m) : 0;
    const int next = lo + last * step;
    n = min(step, n - last * step);
    lo = next;
  }
  return wave_uniform(lo);
}

template <int DP, bool FULL, bool BF16, int WAVES>
__global__ __launch_bounds__(64 * WAVES, WAVES == 8 || DP <= 128 ? 2 : 1) void prompt_kernel(PromptArgs a) {
  using Sh = Shape<DP, WAVES>;
  constexpr int kThreads = Sh::THREADS, kRows = Sh::ROWS, S = Sh::STAGES;
  __shared__ __attribute__((aligned(1024))) char lds[S][2 * Sh::TILEB];  // [buffer][K, V]
  __shared__ int first_bad[DP], any_bad;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int l32 = lane & 31, hf = lane >> 5;

  const int tile = wave_uniform((int)blockIdx.x / a.nkv);
  const int kvh = blockIdx.x - tile * a.nkv;
  const int t = a.tiles - 1 - tile;
  const int b = sequence_of(a, t);
  const int s0 = min(max(a.starts[b], 0), a.n_tokens);
  const int n = min(max(a.starts[b + 1], 0), a.n_tokens) - s0;  // its length
  const int64_t r0 = (t - first_tile(a, b)) * kRows;            // the workgroup's first row
  const int64_t R = (int64_t)n * a.G;
  if (r0 < 0 || r0 >= R) return;
  const int rows = (int)(R - r0 < kRows ? R - r0 : kRows);
  const int units = a.dph / 8;

  // row -> query, head
  const int row = 32 * wave + l32;
  const bool real = row < rows;
  const int q0 = wave_uniform((int)(r0 / a.G)), g0 = wave_uniform((int)(r0 - (int64_t)q0 * a.G));
  const int off = g0 + (real ? row : 0);
  const int qi = q0 + off / a.G;  // the row's query
  const int head = kvh * a.G + off - off / a.G * a.G;
  const int last = real ? qi : -1;  // and the last key it sees
  const int wg_last = wave_uniform(q0 + (g0 + rows - 1) / a.G);
  const int w_first = wave_uniform(q0 + (g0 + min(32 * wave, rows - 1)) / a.G);
  const int w_last = wave_uniform(
      32 * wave < rows ? q0 + (g0 + min(32 * wave + 31, rows - 1)) / a.G : -1);
  const int tiles = wg_last / kTok + 1;

  // ---- tile loads: place i of the staged tile is unit i % UNITS of token
  // i / UNITS; keys past the sequence's last take the last's
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0] + 1024u * wave;
  const uint16_t* const kb = wave_uniform(a.k + (int64_t)s0 * a.k_stride + (int64_t)kvh * a.dph);
  const uint16_t* const vb = wave_uniform(a.v + (int64_t)s0 * a.v_stride + (int64_t)kvh * a.dph);
  if (!FULL) {
    // the features beyond the head's, which no load reaches
    const uint4 z = make_uint4(0, 0, 0, 0);
    for (int i = tid; i < S * 2 * Sh::TILEB / 16; i += kThreads)
      reinterpret_cast<uint4*>(&lds[0][0])[i] = z;
    __syncthreads();
  }
  const uint32_t k_row = 2u * (uint32_t)a.k_stride, v_row = 2u * (uint32_t)a.v_stride;
  auto load_tile = [&](int kt) {
    const uint32_t dst = lds0 + (uint32_t)(kt % S) * (2 * Sh::TILEB);
    const uint16_t* const kp = kb + (int64_t)kt * kTok * a.k_stride;
    const uint16_t* const vp = vb + (int64_t)kt * kTok * a.v_stride;
    const int left = n - 1 - kt * kTok;  // (the clamp's only use: a sequence's end)
#pragma unroll
    for (int j = 0; j < Sh::NU; j++) {
      const int i = j * kThreads + tid;
      const int tk = i / Sh::UNITS;
      const int u = (i - tk * Sh::UNITS) ^ swizzle<DP>(tk);
      const uint32_t key = (uint32_t)min(tk, left);
      if (FULL || u < units) {
        load_to_lds(kp, key * k_row + 16 * u, dst + j * (16 * kThreads));
        load_to_lds(vp, key * v_row + 16 * u, dst + Sh::TILEB + j * (16 * kThreads));
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S - 1; i++)
    if (i < tiles) load_tile(i);
  for (int i = tid; i < DP; i += kThreads) first_bad[i] = INT32_MAX;
  if (tid == 0) any_bad = 0;
  __syncthreads();

  // ---- q operand: this lane's row, features 16 ks + 8 hf .. + 7
  u4v qf[Sh::KS];
  {
    const uint16_t* qp = a.q + (int64_t)(s0 + qi) * a.q_stride + (int64_t)head * a.dph;
#pragma unroll
    for (int ks = 0; ks < Sh::KS; ks++) {
      const int f = 16 * ks + 8 * hf;
      qf[ks] = u4v{0, 0, 0, 0};
      if (FULL || f < a.dph) qf[ks] = *reinterpret_cast<const u4v*>(qp + f);
    }
    // (waited for here: left to their first use, in the loop, the waits would
    // count the next tile's loads too, which the compiler does not know)
#pragma unroll
    for (int ks = 0; ks < Sh::KS; ks++) asm volatile("" : "+v"(qf[ks]));
  }

  float ref = 0.f, raise = -INFINITY, l = 0.f;
  f16v o[Sh::DB];
#pragma unroll
  for (int d = 0; d < Sh::DB; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) o[d][e] = 0.f;
  // Operand reads.  K: token l32 (+ 32 h), unit 2 ks + hf.  V, transposed: token
  // vt (+ 16 k2 + 8 g), unit 4 d + vu, 8 bytes.  The swizzle is bitwise and goes
  // by the token mod 16, 8 tokens on flipping its second bit, so the constants
  // enter by xor.
  const int vt = 4 * hf + ((lane & 15) >> 2);
  const int vu = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int k_at = l32 * Sh::ROWB, v_at = vt * Sh::ROWB + 8 * (lane & 1);
  int kx = 16 * (hf ^ swizzle<DP>(l32)), vx = 16 * (vu ^ swizzle<DP>(vt));

  for (int kt = 0; kt < tiles; kt++) {
    char* const kst = &lds[kt % S][0];
    char* const vst = kst + Sh::TILEB;
    const int ts = kt * kTok;
    // (opaque here: kept across the loop, the addresses of all reads take more
    // registers than there are)
    asm volatile("" : "+v"(kx), "+v"(vx));
    // tile kt is here; those behind it may be on their way
    if constexpr (S == 4) {
      if (kt + 2 < tiles)
        wait_loads<4 * Sh::NU>();
      else if (kt + 1 < tiles)
        wait_loads<2 * Sh::NU>();
      else
        wait_loads<0>();
    } else {
      wait_loads<0>();
    }
    if (ts + kTok - 1 > q0) {
      // Keys that some row of the workgroup does not see: a V element there
      // that is not finite must not meet a weight of 0.  It becomes 0, and the
      // rows that do see it are marked: by feature, the first such key.
#pragma unroll
      for (int j = 0; j < Sh::NU; j++) {
        const int i = j * kThreads + tid;
        const int tk = i / Sh::UNITS, key = ts + tk;
        uint16_t* const at = reinterpret_cast<uint16_t*>(vst + 16 * i);
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        if (key > q0 && (nonfinite2<BF16>(x.x) | nonfinite2<BF16>(x.y) | nonfinite2<BF16>(x.z) |
                         nonfinite2<BF16>(x.w)) != 0) {
          const int u = (i - tk * Sh::UNITS) ^ swizzle<DP>(tk);
#pragma unroll 1
          for (int e = 0; e < 8; e++)
            if (nonfinite2<BF16>(at[e]) != 0) {
              at[e] = 0;
              atomicMin(&first_bad[8 * u + e], key);
              any_bad = 1;
            }
        }
      }
    }
    __syncthreads();
    // (every wave is past tile kt - 1, whose buffer this is)
    if (kt + S - 1 < tiles) load_tile(kt + S - 1);
    if (ts > w_last) continue;  // (wave-uniform)

    f16v s[2];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 16; e++) s[h][e] = 0.f;
    // operand reads a batch ahead of their products (the scheduling barriers
    // keep them there, and the batches in flight to two)
    u4v kf[2][kBatch][2];
    auto read_k = [&](int k0, u4v(&x)[kBatch][2]) {
#pragma unroll
      for (int i = 0; i < kBatch; i++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          x[i][h] = *reinterpret_cast<const u4v*>(kst + 32 * h * Sh::ROWB + k_at +
                                                  (kx ^ (32 * (k0 + i))));
        }
    };
    read_k(0, kf[0]);
#pragma unroll
    for (int k0 = 0; k0 < Sh::KS; k0 += kBatch) {
      if (k0 + kBatch < Sh::KS) read_k(k0 + kBatch, kf[(k0 / kBatch + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kBatch; i++)
#pragma unroll
        for (int h = 0; h < 2; h++)
          s[h] = mfma<BF16>(kf[(k0 / kBatch) & 1][i][h], qf[k0 + i], s[h]);
    }
    // this lane: row l32, keys ts + 32 h + 8 (e / 4) + 4 hf + e % 4
    if (ts + kTok - 1 > w_first) {
      const int left = last - ts - 4 * hf;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 16; e++)
          s[h][e] = 32 * h + 8 * (e / 4) + (e & 3) <= left ? s[h][e] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 16; e++) top = fmaxf(top, s[h][e]);
    top *= a.scale;
    if (__builtin_amdgcn_ballot_w64(top > raise) != 0) {
      top = half_max(top);
      if (top > raise) {
        const float f = raise == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - top);
        ref = top;
        raise = top + kLazyMax;
        l *= f;
#pragma unroll
        for (int d = 0; d < Sh::DB; d++) o[d] *= f;
      }
    }
    auto read_v = [&](int k2, int d) {
      u4v v;
#pragma unroll
      for (int g = 0; g < 2; g++) {
        const uint2 x = __builtin_bit_cast(
            uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4_t*)(
                       vst + (16 * k2 + 8 * g) * Sh::ROWB + v_at + (vx ^ (64 * d + 32 * g)))));
        v[2 * g] = x.x;
        v[2 * g + 1] = x.y;
      }
      return v;
    };
    u4v vf[2][Sh::DB];
#pragma unroll
    for (int d = 0; d < Sh::DB; d++) vf[0][d] = read_v(0, d);
    __builtin_amdgcn_sched_barrier(0);
    float sum[2] = {0.f, 0.f};
    u4v p[4];
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[h][e], a.scale, -ref));
        const float y = __builtin_amdgcn_exp2f(fmaf(s[h][e + 1], a.scale, -ref));
        sum[0] += x;
        sum[1] += y;
        p[2 * h + e / 8][(e & 7) / 2] = pack2<BF16>(x, y);
      }
    l += sum[0] + sum[1];
#pragma unroll
    for (int k2 = 0; k2 < 4; k2++) {
      if (k2 < 3) {
#pragma unroll
        for (int d = 0; d < Sh::DB; d++) vf[(k2 + 1) & 1][d] = read_v(k2 + 1, d);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < Sh::DB; d++) o[d] = mfma<BF16>(vf[k2 & 1][d], p[k2], o[d]);
    }
  }

  l = attn::half_pair_total(l, l);
  __syncthreads();
  if (any_bad) {
#pragma unroll
    for (int d = 0; d < Sh::DB; d++)
#pragma unroll
      for (int e = 0; e < 16; e++)
        if (first_bad[32 * d + 8 * (e / 4) + 4 * hf + (e & 3)] <= qi) o[d][e] = NAN;
  }
  if (!real) return;
  const float inv = 1.f / l;
  uint16_t* op = a.out + (int64_t)(s0 + qi) * a.out_stride + (int64_t)head * a.dph + 4 * hf;
#pragma unroll
  for (int d = 0; d < Sh::DB; d++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int f = 32 * d + 8 * j;
      if (FULL || f < a.dph)
        *reinterpret_cast<uint2*>(op + f) =
            make_uint2(pack2<BF16>(o[d][4 * j] * inv, o[d][4 * j + 1] * inv),
                       pack2<BF16>(o[d][4 * j + 2] * inv, o[d][4 * j + 3] * inv));
    }
}

template <int DP, bool BF16, int WAVES>
void launch_waves(const PromptArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)(a.tiles * a.nkv)), block(64 * WAVES);
  if (a.dph == DP)
    prompt_kernel<DP, true, BF16, WAVES><<<grid, block, 0, s>>>(a);
  else
    prompt_kernel<DP, false, BF16, WAVES><<<grid, block, 0, s>>>(a);
}

template <int DP, bool BF16>
void launch(const PromptArgs& a, hipStream_t s) {
  if (a.rows == 256) {
    if constexpr (DP % 64 == 0 && DP <= 128) launch_waves<DP, BF16, 8>(a, s);
  } else {
    launch_waves<DP, BF16, 4>(a, s);
  }
}

template <bool BF16>
void launch_type(const PromptArgs& a, hipStream_t s) {
  if (a.dph <= 32)
    launch<32, BF16>(a, s);
  else if (a.dph <= 64)
    launch<64, BF16>(a, s);
  else if (a.dph <= 96)
    launch<96, BF16>(a, s);
  else if (a.dph <= 128)
    launch<128, BF16>(a, s);
  else if (a.dph <= 160)
    launch<160, BF16>(a, s);
  else if (a.dph <= 192)
    launch<192, BF16>(a, s);
  else
    launch<256, BF16>(a, s);
}

}  // namespace prompt
}  // namespace sde

extern "C" int sde_prompt_attention(const int32_t* d_starts, int n_seqs, int n_tokens, int dtype,
                                    const void* d_q, int64_t q_stride, const void* d_k,
                                    int64_t k_stride, const void* d_v, int64_t v_stride,
                                    void* d_out, int64_t out_stride, int nh, int nkv, int dph,
                                    sde_stream_t stream) {
  using namespace sde::prompt;
  if (n_seqs < 0 || n_tokens < 0 || nh < 1 || nkv < 1 || dph < 1 || nh % nkv != 0 ||
      !sde::batch::known_dtype(dtype))
    return SDE_ERR_INVALID_ARGUMENT;
  if (dtype == SDE_F32 || dph % 8 != 0 || dph > 256 || nh > (1 << 20) / dph)
    return SDE_ERR_UNSUPPORTED;
  // (a tile's rows are addressed with 32-bit byte offsets)
  if (k_stride > (1 << 24) || v_stride > (1 << 24)) return SDE_ERR_UNSUPPORTED;
  if (n_seqs == 0 || n_tokens == 0) return SDE_OK;
  if (!d_starts || !d_q || !d_k || !d_v || !d_out) return SDE_ERR_INVALID_ARGUMENT;
  const int64_t qw = (int64_t)nh * dph, kw = (int64_t)nkv * dph;
  if (q_stride < qw || k_stride < kw || v_stride < kw || out_stride < qw)
    return SDE_ERR_INVALID_ARGUMENT;
  using sde::batch::aligned;
  if (!aligned(d_q, q_stride, dtype, 16) || !aligned(d_k, k_stride, dtype, 16) ||
      !aligned(d_v, v_stride, dtype, 16) || !aligned(d_out, out_stride, dtype, 16))
    return SDE_ERR_UNSUPPORTED;
  PromptArgs a;
  a.q = static_cast<const uint16_t*>(d_q);
  a.k = static_cast<const uint16_t*>(d_k);
  a.v = static_cast<const uint16_t*>(d_v);
  a.out = static_cast<uint16_t*>(d_out);
  a.starts = d_starts;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.out_stride = out_stride;
  a.n_tokens = n_tokens;
  a.n_seqs = n_seqs;
  a.nkv = nkv;
  a.G = nh / nkv;
  a.dph = dph;
  // 256 rows of long prompts: each key tile is brought in once for twice the
  // rows, if that still makes two workgroups per CU.  Measured on MI355X, 128 / 256
  // rows, us: one prompt of 8192 tokens, 32/8 heads of 128, fp16 629 / 534, bf16 598
  // / 504, of 4096 184 / 147; four of 1024 72 / 68, six of 680 on average, uneven,
  // 54 / 62; 8/8 heads, 4096 tokens (128 workgroups) 89 / 106; 32/4 heads of 64,
  // 4096 99.7 / 99.3.
  const bool whole = (dph > 32 && dph <= 64) || (dph > 96 && dph <= 128);  // (Shape's NU)
  a.rows = whole && (int64_t)n_tokens * nh >= 512 * 256 && n_tokens / n_seqs >= 1024 ? 256 : 128;
  const int64_t tiles = (int64_t)n_tokens * a.G / a.rows + n_seqs;
  if (tiles * nkv > (1 << 22)) return SDE_ERR_UNSUPPORTED;  // (threads of a launch: 32 bits)
  a.tiles = (int)tiles;
  a.scale = (float)(1.4426950408889634 / std::sqrt((double)dph));
  if (dtype == SDE_F16)
    launch_type<false>(a, (hipStream_t)stream);
  else
    launch_type<true>(a, (hipStream_t)stream);
  return sde::launch_status();
}
