// Rows of logits read in 16-byte pieces wherever they start, for the kernels that go over whole
// rows of a vocabulary.
#pragma once

#include "common.hpp"

namespace nml {

__device__ __forceinline__ float exp_of(float t) { return __builtin_amdgcn_exp2f(t * 1.44269504088896341f); }

constexpr float kNone = -3.402823466e38f;  // a reference below every finite logit

// The 16-byte pieces of a row: piece c holds elements c·E − off … c·E − off + E − 1.
template <typename T>
struct RowPieces {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  typedef T vec __attribute__((ext_vector_type(E)));
  const T* row;
  int V, off, n;
  __device__ RowPieces(const T* r, int v) : row(r), V(v) {
    off = static_cast<int>((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    n = (V + off + E - 1) / E;
  }
  __device__ int first(int c) const { return c * E - off; }
  __device__ vec load(int c) const {
    const int i = first(c);
    if (i >= 0 && i + E <= V) return *reinterpret_cast<const vec*>(row + i);
    return edge(i);
  }
  // (word by word: as a vector its values would take a register each beside the whole pieces)
  __device__ vec edge(int i) const {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    u4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (E == 4) {
        r[w] = i + w >= 0 && i + w < V ? __builtin_bit_cast(unsigned, row[i + w]) : 0xff800000u;
      } else {
        unsigned half[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = i + 2 * w + e;
          half[e] = at >= 0 && at < V ? __builtin_bit_cast(unsigned short, row[at]) : 0xfc00u;
        }
        r[w] = half[0] | half[1] << 16;
      }
    }
    return __builtin_bit_cast(vec, r);
  }
};

template <typename T>
__device__ __forceinline__ float piece_max(const typename RowPieces<T>::vec& v);
template <>
__device__ __forceinline__ float piece_max<float>(const typename RowPieces<float>::vec& v) {
  return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
}
template <>
__device__ __forceinline__ float piece_max<half_t>(const typename RowPieces<half_t>::vec& v) {
  typedef half_t h2 __attribute__((ext_vector_type(2)));
  const h2 a = __builtin_elementwise_max(h2{v[0], v[1]}, h2{v[2], v[3]});
  const h2 b = __builtin_elementwise_max(h2{v[4], v[5]}, h2{v[6], v[7]});
  const h2 c = __builtin_elementwise_max(a, b);
  return fmaxf(static_cast<float>(c.x), static_cast<float>(c.y));
}

}  // namespace nml
