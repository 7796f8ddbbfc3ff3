// A KV cache in pages: written, and attended to by a row's newest tokens.
//
// The cache is two pools, (pages, kv_heads, page, dk): a page holds `page` (a power of two) positions
// of one row, a head's positions in a run. Row b's position p is position p % page of page
// table[b·max_pages + p / page].
#include "kernels.hpp"

namespace nml {

namespace {

typedef unsigned u4 __attribute__((ext_vector_type(4)));

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

// ------------------------------------------------------------------------- write

// n / d for n < 2^31 by a product and a shift.
struct Div {
  unsigned mul, shift;
};
inline Div div_by(unsigned d) {
  unsigned s = 0;
  while ((1ull << s) < d) ++s;
  return Div{static_cast<unsigned>(((1ull << 32) * ((1ull << s) - d)) / d + 1), s};
}
__device__ __forceinline__ unsigned quotient(unsigned n, Div d) { return (__umulhi(d.mul, n) + n) >> d.shift; }

// A writing workgroup, and the units that a lane of it takes (their loads in flight together).
constexpr int kWriters = 256, kEach = 4;

// Units of one row: (head, token, unit of its vector), the unit fastest: the order of the pages, so
// that a workgroup writes runs of them.
struct Units {
  Div by_units, by_tokens;
  int units, tokens, count;
};

// U: what is copied at once, 16 bytes where everything is aligned so, else a value.
template <typename U>
__global__ __launch_bounds__(kWriters) void paged_write_kernel(PagedWriteArgs a, Units n) {
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const U* src = static_cast<const U*>(is_v ? a.v : a.k) + b * a.stride_b;
  U* pages = static_cast<U*>(is_v ? a.v_pages : a.k_pages);
  const int32_t* table = a.table + static_cast<size_t>(b) * a.max_pages;
  const int count = row_count(a.counts, b, a.S, a.err), pos = a.pos ? a.pos[b] : 0;
  const long long room = static_cast<long long>(a.max_pages) << a.shift;
  U x[kEach];
  size_t to[kEach];
  bool here[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const unsigned i = (blockIdx.x * kEach + k) * kWriters + threadIdx.x;
    const unsigned t = quotient(i, n.by_units), h = quotient(t, n.by_tokens);
    const int s = static_cast<int>(t - h * n.tokens), unit = static_cast<int>(i - t * n.units);
    const long long p = static_cast<long long>(pos) + s;
    here[k] = i < static_cast<unsigned>(n.count) && s < count;
    if (here[k]) {
      const int page = p >= 0 && p < room ? table[p >> a.shift] : -1;
      if (page < 0 || page >= a.num_pages) {
        here[k] = false;
        tell(a.err);
      } else {
        const int in = static_cast<int>(p & ((1 << a.shift) - 1));
        to[k] = (((static_cast<size_t>(page) * a.H + h) << a.shift) + in) * n.units + unit;
        x[k] = src[h * a.stride_h + s * a.stride_s + unit];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (here[k]) pages[to[k]] = x[k];
}

template <typename U>
int write_launch(PagedWriteArgs a, size_t es, hipStream_t st) {
  const int per = static_cast<int>(sizeof(U) / es);
  Units n;
  n.units = a.dk / per;
  n.tokens = a.S;
  n.count = a.S * a.H * n.units;
  n.by_units = div_by(n.units);
  n.by_tokens = div_by(a.S);
  a.stride_b /= per;
  a.stride_h /= per;
  a.stride_s /= per;
  const dim3 grid((n.count + kEach * kWriters - 1) / (kEach * kWriters), a.B, 2);
  paged_write_kernel<U><<<grid, kWriters, 0, st>>>(a, n);
  NML_LAUNCHED();
  return 0;
}

// --------------------------------------------------------------------- attention

// One query of a head a workgroup: a wave takes 64 keys at a time, one a lane.
template <typename T>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedAttnArgs a) {
  __shared__ float q[kMaxHeadDim], o_w[4][kMaxHeadDim], m_w[4], l_w[4];
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int n = row_count(a.counts, b, a.S, a.err);
  const int room = a.max_pages << a.shift, len0 = a.lens[b], len = min(max(len0, 0), room);
  if (len != len0 && tid == 0) tell(a.err);
  if (s >= n) return;
  const int keys = max(len - n + s + 1, 0), hk = h / a.group;
  for (int d = tid; d < a.dk; d += 256)
    q[d] = static_cast<float>(static_cast<const T*>(a.q)[((static_cast<size_t>(b) * a.H + h) * a.S + s) * a.dk + d]);
  __syncthreads();
  const int32_t* table = a.table + static_cast<size_t>(b) * a.max_pages;
  auto at = [&](int key) {
    int page = table[key >> a.shift];
    if (page < 0 || page >= a.num_pages) {
      tell(a.err);
      page = 0;
    }
    return (((static_cast<size_t>(page) * a.Hkv + hk) << a.shift) + (key & ((1 << a.shift) - 1))) * a.dk;
  };
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 64 * w; k0 < keys; k0 += 256) {
    const int key = k0 + lane;
    float x = -INFINITY;
    if (key < keys) {
      const T* k = static_cast<const T*>(a.k_pages) + at(key);
      x = 0.f;
      for (int d = 0; d < a.dk; ++d) x = __builtin_fmaf(q[d], static_cast<float>(k[d]), x);
      x /= a.scale;
    }
    const float mn = fmaxf(m, wave_max(x)), ref = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - ref), p = expf(x - ref);
    m = mn;
    l = l * f + wave_sum(p);
    for (int i = 0; i < 4; ++i) o[i] *= f;
    for (int j = 0; j < min(64, keys - k0); ++j) {
      const float pj = __shfl(p, j, 64);
      const T* v = static_cast<const T*>(a.v_pages) + at(k0 + j);
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < a.dk) o[i] = __builtin_fmaf(pj, static_cast<float>(v[lane + 64 * i]), o[i]);
    }
  }
  for (int i = 0; i < 4; ++i) o_w[w][lane + 64 * i] = o[i];
  if (lane == 0) m_w[w] = m, l_w[w] = l;
  __syncthreads();
  for (int d = tid; d < a.dk; d += 256) {
    float mn = m_w[0], lt = 0.f, ot = 0.f;
    for (int i = 1; i < 4; ++i) mn = fmaxf(mn, m_w[i]);
    for (int i = 0; i < 4; ++i) {
      const float f = mn == -INFINITY ? 0.f : expf(m_w[i] - mn);
      lt += l_w[i] * f;
      ot += o_w[i][d] * f;
    }
    static_cast<T*>(a.out)[((static_cast<size_t>(b) * a.S + s) * a.H + h) * a.dk + d] = static_cast<T>(keys == 0 ? 0.f : ot / lt);
  }
}

}  // namespace

int launch_paged_write(int dt, const PagedWriteArgs& a, hipStream_t st) {
  const size_t es = dtype_size(dt);
  const long long per = static_cast<long long>(16 / es);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.k_pages) | reinterpret_cast<uintptr_t>(a.v_pages);
  if ((bits & 15) == 0 && ((a.dk | a.stride_b | a.stride_h | a.stride_s) & (per - 1)) == 0)
    return write_launch<u4>(a, es, st);
  return es == 2 ? write_launch<unsigned short>(a, es, st) : write_launch<unsigned>(a, es, st);
}

size_t paged_attention_workspace(int dt, int B, int H, int Hkv, int S, int P, int dk) { return 0; }

int launch_paged_attention(int dt, const PagedAttnArgs& a, hipStream_t st) {
  const dim3 grid(a.S, a.H, a.B);
  if (dt == F16) paged_attention_kernel<half_t><<<grid, 256, 0, st>>>(a);
  else paged_attention_kernel<float><<<grid, 256, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

}  // namespace nml
