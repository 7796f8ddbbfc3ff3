// What the kernels over a paged KV cache share.
#pragma once

#include "kernels.hpp"

namespace nml {

typedef float f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void tell(int* err) {
  if (err) __hip_atomic_fetch_or(err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// New tokens of row b.
__device__ __forceinline__ int row_count(const int32_t* counts, int b, int S, int* err) {
  if (!counts) return S;
  const int n = counts[b], c = n < 0 ? 0 : (n > S ? S : n);
  if (c != n) tell(err);
  return c;
}

// The pages of one row and KV head.
struct RowPages {
  const int32_t* table;
  int shift, num_pages, Hkv, hk;
  // Number of the page of a key, as it stands in the table.
  __device__ __forceinline__ int number(int key) const { return table[key >> shift]; }
  // Where that key's vector starts, in vectors. `bad`: the page is out of range (page 0 is read).
  __device__ __forceinline__ size_t place(int key, int page, bool& bad) const {
    const bool out = static_cast<unsigned>(page) >= static_cast<unsigned>(num_pages);
    bad |= out;
    return ((static_cast<size_t>(out ? 0 : page) * Hkv + hk) << shift) + (key & ((1 << shift) - 1));
  }
};

// Partial results pass between workgroups of any XCD: stores and loads at agent scope (past the
// L2s) and a count that each workgroup adds to once its stores have arrived.
__device__ __forceinline__ void put2(float* p, f2 v) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 get2(const float* p) {
  return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT));
}

// ws of the attention: counters of tiles whose keys are in pieces (zero before and after every launch,
// in the same place for calls of any size), then the pieces' parts.
constexpr int kCounters = 4096, kCounterStep = 16;  // a line for each
constexpr size_t kCounterBytes = sizeof(unsigned) * kCounters * kCounterStep;

// Attention of many new tokens (ops_paged_prefill.hip), for the calls that it takes; the buffers are
// 16-byte aligned.
bool paged_prefill_applies(int dt, int H, int Hkv, int S, int dk);
size_t paged_prefill_workspace(int dt, int B, int H, int Hkv, int S, int P, int dk);
int launch_paged_prefill(int dt, PagedAttnArgs a, hipStream_t st);

}  // namespace nml
