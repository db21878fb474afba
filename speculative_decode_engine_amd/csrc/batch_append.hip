// Appending the new tokens of several requests to one paged pool, with the
// position rotation of q and k on the way (sde_batch_append): the work of
// cublas_rope_kernel (kernels.cu:797-817) and cublas_kv_append_kernel
// (kernels.cu:826-844) for tokens that each name their request and position.
//
//   a_j = pos / div * theta^(-2j/dph),  j < dph/2
//   (x_j, x_{j+dph/2}) -> (x_j cos a_j - x_{j+dph/2} sin a_j,
//                          x_{j+dph/2} cos a_j + x_j sin a_j)
//
// A copy with a little arithmetic: every row is read once and written once
// (k once into the pool and, where asked, once more).  A thread takes one
// 16-byte vector of each half of a head (or two of v), so all loads and
// stores of a half-precision row are 16 bytes wide; a workgroup's token is
// the same for all its threads, so its request, position and page are scalar
// loads.
//
// Angles: a frequency is held as the fraction of a turn it advances per
// position, in 64-bit fixed point, so the product with the position wraps by
// itself into [0, 1) turn without losing the fraction: fp32 angles, as the
// one-sequence call has them, are off by pos * 2^-24 turns at far positions.
// The top 32 bits, read as signed, go to sincospi.
//
// Measured on MI355X: 8191 prompt tokens, 218 MB read and written: 48.6 us, 4.5 TB/s
// (a copy of 4 GiB runs at 4.7); one token of each of 8 requests: 4.1 us, the chain
// of request, position, page and rows.
#include <cmath>
#include <cstring>

#include "batch_common.hpp"

namespace sde {
namespace batch {

constexpr int kAppendThreads = 256;
constexpr int kMaxPairs = 256;  // dph up to 512

struct AppendArgs {
  uint16_t* pool;
  const int32_t* tables;
  const int32_t* seq;
  const int32_t* pos;
  const void* k;
  const void* v;
  const void* q;
  void* k_out;
  void* q_out;
  int64_t k_stride, v_stride, q_stride, k_out_stride, q_out_stride;
  int pool_blocks, bs, kv_dim, n_seqs, max_blocks, table_stride;
  int nkv, dph;
  int q_items, k_items;  // vector pairs of a token's q and of its k (and v)
  int rotate;
  uint64_t turn[kMaxPairs];  // turns per position, 2^-64 units
};

template <class E, int VEC>
struct Vec {
  float x[VEC];
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    const typename E::type* p = static_cast<const typename E::type*>(base) + at;
    if constexpr (VEC == 1) {
      x[0] = E::get(*p);
    } else {
      const uint4 raw = *reinterpret_cast<const uint4*>(p);
      typename E::type e[VEC];
      static_assert(sizeof(e) == 16, "one 16-byte vector");
      __builtin_memcpy(e, &raw, 16);
#pragma unroll
      for (int i = 0; i < VEC; i++) x[i] = E::get(e[i]);
    }
  }
  __device__ __forceinline__ void store(void* base, int64_t at) const {
    typename E::type* p = static_cast<typename E::type*>(base) + at;
    if constexpr (VEC == 1) {
      *p = E::put(x[0]);
    } else {
      typename E::type e[VEC];
#pragma unroll
      for (int i = 0; i < VEC; i++) e[i] = E::put(x[i]);
      uint4 raw;
      __builtin_memcpy(&raw, e, 16);
      *reinterpret_cast<uint4*>(p) = raw;
    }
  }
  // fp16 (round to nearest even) into the pool
  __device__ __forceinline__ void store_half(uint16_t* p) const {
    uint16_t e[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) e[i] = f16_elem::put(x[i]);
    if constexpr (VEC == 1) {
      *p = e[0];
    } else if constexpr (VEC == 4) {
      uint2 raw;
      __builtin_memcpy(&raw, e, 8);
      *reinterpret_cast<uint2*>(p) = raw;
    } else {
      uint4 raw;
      __builtin_memcpy(&raw, e, 16);
      *reinterpret_cast<uint4*>(p) = raw;
    }
  }
};

// Workgroup (token, part of its items).  Items: the q pairs, the k pairs, the
// v vectors (two neighbours each).
template <class E, int VEC>
__global__ __launch_bounds__(kAppendThreads) void batch_append_kernel(AppendArgs a) {
  const int t = blockIdx.x;
  const int s = a.seq[t], pos = a.pos[t];
  if (s < 0 || s >= a.n_seqs || pos < 0) return;
  const int lb = pos / a.bs;
  if (lb >= a.max_blocks) return;
  const int page = a.tables[(int64_t)s * a.table_stride + lb];
  if (page < 0 || page >= a.pool_blocks) return;
  int item = blockIdx.y * kAppendThreads + threadIdx.x;
  const int half = a.dph >> 1;
  const int chunks = half / VEC;  // per head
  uint16_t* const krow =
      a.pool + ((uint64_t)(uint32_t)page * 2u * a.bs + (uint32_t)(pos - lb * a.bs)) * a.kv_dim;
  if (item >= a.q_items + a.k_items) {
    item -= a.q_items + a.k_items;
    if (item >= a.k_items) return;
    uint16_t* const vrow = krow + (int64_t)a.bs * a.kv_dim;
    const int at = 2 * VEC * item;
    Vec<E, VEC> x, y;
    x.load(a.v, t * a.v_stride + at);
    y.load(a.v, t * a.v_stride + at + VEC);
    x.store_half(vrow + at);
    y.store_half(vrow + at + VEC);
    return;
  }
  const bool is_k = item >= a.q_items;
  if (is_k) item -= a.q_items;
  const int head = item / chunks;
  const int j = (item - head * chunks) * VEC;
  const int at = head * a.dph + j;
  const void* src = is_k ? a.k : a.q;
  const int64_t row = t * (is_k ? a.k_stride : a.q_stride);
  Vec<E, VEC> x, y;
  x.load(src, row + at);
  y.load(src, row + at + half);
  if (a.rotate) {
#pragma unroll
    for (int i = 0; i < VEC; i++) {
      const uint64_t turns = a.turn[j + i] * (uint64_t)(uint32_t)pos;
      // half turns in [-1, 1)
      const float h = (float)(int32_t)(uint32_t)(turns >> 32) * 0x1p-31f;
      float sn, cs;
      sincospif(h, &sn, &cs);
      const float u = x.x[i], w = y.x[i];
      x.x[i] = u * cs - w * sn;
      y.x[i] = w * cs + u * sn;
    }
  }
  if (!is_k) {
    const int64_t o = t * a.q_out_stride + at;
    x.store(a.q_out, o);
    y.store(a.q_out, o + half);
    return;
  }
  x.store_half(krow + at);
  y.store_half(krow + at + half);
  if (a.k_out) {
    const int64_t o = t * a.k_out_stride + at;
    x.store(a.k_out, o);
    y.store(a.k_out, o + half);
  }
}

// Turns per position of each rotation pair, in units of 2^-64.  Every layer of
// a model asks for the same ones: a thread keeps the last it formed.
const uint64_t* rope_turns(double theta, double divisor, int dph) {
  struct Table {
    double theta = 0.0, divisor = 0.0;
    int dph = 0;
    uint64_t turn[kMaxPairs];
  };
  thread_local Table t;
  if (t.dph != dph || t.theta != theta || t.divisor != divisor) {
    const double log_theta = std::log(theta);
    for (int j = 0; j < kMaxPairs; j++) {
      // (below 0.16 turns, or as much more as a theta under 1 gives: the
      // whole turns drop out)
      double f = 0.0;
      if (j < dph / 2)
        f = std::exp(-log_theta * (2.0 * j) / dph) / divisor * 0.15915494309189533577;
      f -= std::floor(f);
      t.turn[j] = f < 1.0 ? (uint64_t)std::ldexp(f, 64) : 0;
    }
    t.theta = theta;
    t.divisor = divisor;
    t.dph = dph;
  }
  return t.turn;
}

template <class E, int VEC>
void launch_append(const AppendArgs& a, int n_tokens, hipStream_t stream) {
  const int items = a.q_items + 2 * a.k_items;
  const dim3 grid(n_tokens, (items + kAppendThreads - 1) / kAppendThreads);
  batch_append_kernel<E, VEC><<<grid, dim3(kAppendThreads), 0, stream>>>(a);
}

}  // namespace batch
}  // namespace sde

extern "C" int sde_batch_append(const sde_batch_pool* pool, const int32_t* d_seq,
                                const int32_t* d_pos, int n_tokens, int dtype, const void* d_k,
                                int64_t k_stride, const void* d_v, int64_t v_stride, void* d_k_out,
                                int64_t k_out_stride, const void* d_q, int64_t q_stride,
                                void* d_q_out, int64_t q_out_stride, int nh, int nkv, int dph,
                                const sde_rope_config* rope, sde_stream_t stream) {
  using namespace sde::batch;
  const int st = check_pool(pool);
  if (st != SDE_OK) return st;
  if (n_tokens < 0 || nkv < 1 || dph < 1 || !known_dtype(dtype)) return SDE_ERR_INVALID_ARGUMENT;
  if ((int64_t)nkv * dph != pool->kv_dim) return SDE_ERR_INVALID_ARGUMENT;
  if (dph % 2 != 0 || dph > 2 * kMaxPairs) return SDE_ERR_UNSUPPORTED;
  if ((d_q == nullptr) != (d_q_out == nullptr)) return SDE_ERR_INVALID_ARGUMENT;
  if (d_q && (nh < 1 || nh > (1 << 20) / dph)) return SDE_ERR_INVALID_ARGUMENT;
  // (a launch counts its threads in 32 bits)
  if (pool->kv_dim > (1 << 20) || n_tokens > (1 << 23)) return SDE_ERR_UNSUPPORTED;
  if (rope && (rope->scaling_type < SDE_ROPE_NONE || rope->scaling_type > SDE_ROPE_YARN ||
               !std::isfinite(rope->theta) || !std::isfinite(rope->scaling_factor)))
    return SDE_ERR_INVALID_ARGUMENT;
  if (n_tokens == 0 || pool->n_seqs == 0) return SDE_OK;
  if (!d_seq || !d_pos || !d_k || !d_v) return SDE_ERR_INVALID_ARGUMENT;
  const int64_t kvd = pool->kv_dim, qd = (int64_t)(d_q ? nh : 0) * dph;
  if (k_stride < kvd || v_stride < kvd || (d_k_out && k_out_stride < kvd) ||
      (d_q && (q_stride < qd || q_out_stride < qd)))
    return SDE_ERR_INVALID_ARGUMENT;
  const size_t e = elem_bytes(dtype);
  for (const void* p : {d_k, d_v, d_q, (const void*)d_k_out, (const void*)d_q_out})
    if ((reinterpret_cast<uintptr_t>(p) % e) != 0) return SDE_ERR_INVALID_ARGUMENT;

  AppendArgs a;
  a.pool = pool->pool;
  a.tables = pool->tables;
  a.seq = d_seq;
  a.pos = d_pos;
  a.k = d_k;
  a.v = d_v;
  a.q = d_q;
  a.k_out = d_k_out;
  a.q_out = d_q_out;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_stride = q_stride;
  a.k_out_stride = k_out_stride;
  a.q_out_stride = q_out_stride;
  a.pool_blocks = pool->pool_blocks;
  a.bs = pool->block_size;
  a.kv_dim = pool->kv_dim;
  a.n_seqs = pool->n_seqs;
  a.max_blocks = pool->max_blocks;
  a.table_stride = pool->table_stride;
  a.nkv = nkv;
  a.dph = dph;
  a.rotate = rope ? 1 : 0;
  if (rope) {
    // theta defaults to 10000; NTK scales theta by factor^(dph/(dph-2)); linear
    // and YaRN divide the position; each applies only for a factor above 1
    // (rope_apply_inplace, model.cu:281-323).
    const double factor = rope->scaling_factor;
    double theta = rope->theta > 1e-6f ? (double)rope->theta : 10000.0;
    if (rope->scaling_type == SDE_ROPE_NTK && factor > 1.0 && dph > 2)
      theta *= std::pow(factor, (double)dph / ((double)dph - 2.0));
    const bool div =
        (rope->scaling_type == SDE_ROPE_LINEAR || rope->scaling_type == SDE_ROPE_YARN) &&
        factor > 1.0;
    std::memcpy(a.turn, rope_turns(theta, div ? factor : 1.0, dph), sizeof(a.turn));
  }
  // Wide vectors where every row's halves start on 16 bytes (8 in the pool for
  // fp32 rows).
  const int vec = dtype == SDE_F32 ? 4 : 8;
  const bool wide = (dph / 2) % vec == 0 &&
                    (reinterpret_cast<uintptr_t>(a.pool) % (2 * (size_t)vec)) == 0 &&
                    aligned(d_k, k_stride, dtype, 16) && aligned(d_v, v_stride, dtype, 16) &&
                    (!d_k_out || aligned(d_k_out, k_out_stride, dtype, 16)) &&
                    (!d_q || (aligned(d_q, q_stride, dtype, 16) &&
                              aligned(d_q_out, q_out_stride, dtype, 16)));
  const int n = wide ? vec : 1;
  a.q_items = (int)(qd / 2 / n);
  a.k_items = (int)(kvd / 2 / n);
  const hipStream_t s = (hipStream_t)stream;
  if (dtype == SDE_F32)
    wide ? launch_append<f32_elem, 4>(a, n_tokens, s) : launch_append<f32_elem, 1>(a, n_tokens, s);
  else if (dtype == SDE_F16)
    wide ? launch_append<f16_elem, 8>(a, n_tokens, s) : launch_append<f16_elem, 1>(a, n_tokens, s);
  else
    wide ? launch_append<bf16_elem, 8>(a, n_tokens, s)
         : launch_append<bf16_elem, 1>(a, n_tokens, s);
  return sde::launch_status();
}
