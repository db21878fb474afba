// Element types, strided rows and page lookups shared by the operators over
// several requests (batch_append.hip, batch_attention.hip,
// prompt_attention.hip, sample.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sde_internal.hpp"

namespace sde {
namespace batch {

constexpr int kMaxBlockSize = 1024;

struct f32_elem {
  using type = float;
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
struct f16_elem {
  using type = uint16_t;
  static __device__ __forceinline__ float get(uint16_t x) {
    return (float)__builtin_bit_cast(_Float16, x);
  }
  static __device__ __forceinline__ uint16_t put(float x) {
    return __builtin_bit_cast(uint16_t, (_Float16)x);
  }
};
struct bf16_elem {
  using type = uint16_t;
  static __device__ __forceinline__ float get(uint16_t x) {
    return __builtin_bit_cast(float, (uint32_t)x << 16);
  }
  // round-to-nearest-even (the hardware's conversion)
  static __device__ __forceinline__ uint16_t put(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  }
};

__host__ __device__ inline int elem_bytes(int dtype) { return dtype == SDE_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) {
  return dtype == SDE_F32 || dtype == SDE_F16 || dtype == SDE_BF16;
}

// Whether rows of `n`-byte vectors can be read there: base and row stride.
inline bool aligned(const void* p, int64_t stride_elems, int dtype, size_t n) {
  return (reinterpret_cast<uintptr_t>(p) % n) == 0 &&
         ((uint64_t)stride_elems * (uint64_t)elem_bytes(dtype)) % n == 0;
}

// Checks the pool and its tables; the pool's rows ([block][K, V][slot]) are
// numbered in 32 bits.
inline int check_pool(const sde_batch_pool* p) {
  if (!p || !p->pool || (!p->tables && p->n_seqs > 0)) return SDE_ERR_INVALID_ARGUMENT;
  if (p->pool_blocks < 1 || p->block_size < 1 || p->kv_dim < 1 || p->n_seqs < 0 ||
      p->max_blocks < 1 || p->table_stride < p->max_blocks)
    return SDE_ERR_INVALID_ARGUMENT;
  if (p->block_size > kMaxBlockSize) return SDE_ERR_UNSUPPORTED;
  if ((int64_t)p->max_blocks * p->block_size > INT32_MAX) return SDE_ERR_UNSUPPORTED;
  if ((uint64_t)p->pool_blocks * 2u * (uint64_t)p->block_size > 0xFFFFFFFFull)
    return SDE_ERR_UNSUPPORTED;
  return SDE_OK;
}

}  // namespace batch
}  // namespace sde
