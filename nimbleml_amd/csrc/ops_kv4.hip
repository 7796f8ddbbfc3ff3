// A KV cache in 4 bits: written, read back and attended to.
//
// Format (one head's vector of dk values, ⌈dk/32⌉ blocks of 32, the last padded with zeros):
// 32 E2M1 codes (0 ½ 1 1½ 2 3 4 6 with a sign; the first of two in a byte's low half) and one
// scale byte e that stands for 2^(e − 127), 255 for NaN: 17 bytes a block, 4.25 bits a value,
// 3.76 times fewer bytes than fp16. gfx950 converts two codes to two values, scale included, in
// one instruction, and rounds two values to two codes in another.
//
// With 2^k ≤ max|x| < 2^(k+1) the scale is 2^(k−2), or 2^(k−1) where max|x| ≥ 1.75·2^k: there
// saturating the largest value at 6 would cost more than the coarser step (signal to error on
// normal values 19.02 dB with the change at 1.75, 18.75 at 1.5, 18.79 without it; 16.33, 15.41
// and 16.30 with one channel of 32 six times as large).
#include "kernels.hpp"

namespace nml {

namespace {

constexpr int kBlock = 32;            // values of one scale
constexpr int kBlockBytes = 16;       // and their codes
constexpr int kMinExp = -120;         // ½·2^-120 is a normal float32 and bf16
constexpr unsigned kScaleNaN = 255u;

// New tokens of row b, and whether the count had to be clamped.
__device__ __forceinline__ int row_count(const int32_t* counts, int b, int S, int* err) {
  if (!counts) return S;
  const int n = counts[b], c = n < 0 ? 0 : (n > S ? S : n);
  if (c != n && err) __hip_atomic_fetch_or(err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return c;
}

__device__ __forceinline__ unsigned quad_umax(unsigned v) {
  const unsigned a = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppXor1, 0xF, 0xF, false);
  v = v > a ? v : a;
  const unsigned c = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kDppXor2, 0xF, 0xF, false);
  return v > c ? v : c;
}

// The scale of a block from the bits of max|x| (finite): exponent as described above, at most
// `top`, at least kMinExp.
__device__ __forceinline__ int block_exponent(unsigned amax_bits, int top) {
  const int e = static_cast<int>(amax_bits >> 23) - 127 - 2 + ((amax_bits & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return e < kMinExp ? kMinExp : (e > top ? top : e);
}

// fp16 values: every code has to be finite in fp16 (6·2^13 = 49152, 4·2^14 is not).
template <typename T>
constexpr int top_exponent() {
  return sizeof(T) == 2 ? 13 : 125;
}

// 2^(e − 127) of a scale byte (0: 2^-127, a denormal).
__device__ __forceinline__ float scale_value(unsigned e) {
  return __builtin_bit_cast(float, e ? e << 23 : 0x00400000u);
}

// Items of one row b: (s, h, block) with the block fastest, then the head (HEAD_INNER) or the
// token. Four lanes share a block, eight values each.
struct Item {
  int s, h, blk;
};
template <bool HEAD_INNER>
__device__ __forceinline__ Item item_of(unsigned i, int S, int H, int nb) {
  const unsigned t = i / static_cast<unsigned>(nb), blk = i - t * nb;
  const unsigned in = HEAD_INNER ? H : S;
  const unsigned o = t / in, r = t - o * in;
  return HEAD_INNER ? Item{static_cast<int>(o), static_cast<int>(r), static_cast<int>(blk)}
                    : Item{static_cast<int>(r), static_cast<int>(o), static_cast<int>(blk)};
}

// Eight values from d0 on of a vector of dk, zeros past its end. VEC: 16-byte loads (dk and
// the row's place are multiples of eight values there, so a lane's values are all in or out).
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int d0, int dk, float* x) {
  if (VEC) {
    typedef T v8 __attribute__((ext_vector_type(8), aligned(16)));
    if (d0 < dk) {
      const v8 r = *reinterpret_cast<const v8*>(p + d0);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = 0.f;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = d0 + i < dk ? static_cast<float>(p[d0 + i]) : 0.f;
  }
}

template <typename T, bool VEC, bool HEAD_INNER>
__global__ __launch_bounds__(256) void kv4_write_kernel(Kv4WriteArgs a) {
  const int b = blockIdx.y, nb = (a.dk + kBlock - 1) / kBlock;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const unsigned item = idx >> 2, part = idx & 3u;
  if (item >= static_cast<unsigned>(a.S) * a.H * nb) return;  // (a block's four lanes together)
  const Item it = item_of<HEAD_INNER>(item, a.S, a.H, nb);
  if (it.s >= row_count(a.counts, b, a.S, a.err)) return;
  const long long p = static_cast<long long>(a.pos ? a.pos[b] : 0) + it.s;
  if (p < 0 || p >= a.P) {
    if (a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return;
  }
  const bool is_v = blockIdx.z != 0;
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + b * a.stride_b + it.h * a.stride_h + it.s * a.stride_s;
  float x[8];
  load8<T, VEC>(src, it.blk * kBlock + part * 8, a.dk, x);
  // max|x| on the bits: infinity and NaN are the largest
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned u = __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu;
    top = top > u ? top : u;
  }
  top = quad_umax(top);
  unsigned codes = 0, scale = kScaleNaN;
  if (top < 0x7f800000u) {
    const int e = block_exponent(top, top_exponent<T>());
    scale = static_cast<unsigned>(e + 127);
    const float s = scale_value(scale);
    // to the nearest code, ties to the even one, saturated at 6
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[0], x[1], s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[2], x[3], s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[4], x[5], s, 2);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[6], x[7], s, 3);
  }
  const size_t at = ((static_cast<size_t>(b) * a.H + it.h) * a.P + p) * nb + it.blk;
  *reinterpret_cast<unsigned*>((is_v ? a.v_codes : a.k_codes) + at * kBlockBytes + part * 4) = codes;
  if (part == 0) (is_v ? a.v_scales : a.k_scales)[at] = static_cast<uint8_t>(scale);
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4ReadArgs a) {
  typedef T v8 __attribute__((ext_vector_type(8), aligned(16)));
  const int b = blockIdx.y, nb = (a.dk + kBlock - 1) / kBlock;
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  const unsigned item = idx >> 2, part = idx & 3u;
  if (item >= static_cast<unsigned>(a.S) * a.H * nb) return;
  const Item it = item_of<false>(item, a.S, a.H, nb);
  if (it.s >= row_count(a.counts, b, a.S, a.err)) return;
  const int d0 = it.blk * kBlock + part * 8;
  if (d0 >= a.dk) return;
  const long long p = static_cast<long long>(a.pos ? a.pos[b] : 0) + it.s;
  const bool is_v = blockIdx.z != 0, inside = p >= 0 && p < a.P;
  unsigned codes = 0, scale = 127;
  if (inside) {
    const size_t at = ((static_cast<size_t>(b) * a.H + it.h) * a.P + p) * nb + it.blk;
    codes = *reinterpret_cast<const unsigned*>((is_v ? a.v_codes : a.k_codes) + at * kBlockBytes + part * 4);
    scale = (is_v ? a.v_scales : a.k_scales)[at];
  } else if (a.err) {
    __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  typedef float f2 __attribute__((ext_vector_type(2)));
  const float s = scale_value(scale);
  const f2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 0);
  const f2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 1);
  const f2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 2);
  const f2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, s, 3);
  float x[8] = {x0.x, x0.y, x1.x, x1.y, x2.x, x2.y, x3.x, x3.y};
  if (scale == kScaleNaN) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
  }
  T* out = static_cast<T*>(is_v ? a.v_out : a.k_out) +
           ((static_cast<size_t>(b) * a.H + it.h) * a.S + it.s) * a.dk + d0;
  if (VEC) {
    v8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<T>(x[i]);
    *reinterpret_cast<v8*>(out) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (d0 + i < a.dk) out[i] = static_cast<T>(x[i]);
  }
}

// One query per workgroup, a wave takes every fourth key, a lane four of the head's values;
// online softmax in float32.
template <typename T>
__global__ __launch_bounds__(256) void kv4_attention_kernel(Kv4AttnArgs a) {
  __shared__ float sm[4], sl[4], so[4][256];
  typedef float f2 __attribute__((ext_vector_type(2)));
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int nb = (a.dk + kBlock - 1) / kBlock, group = a.H / a.Hkv;
  const int n = row_count(a.counts, b, a.S, a.err);
  if (s >= n) return;
  int len = a.lens[b];
  if (len < 0 || len > a.P) {
    len = len < 0 ? 0 : a.P;
    if (a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const int keys = len - n + s + 1;
  const int d0 = lane * 4, blk = d0 / kBlock;
  const bool mine = d0 < nb * kBlock;
  float q[4] = {0.f, 0.f, 0.f, 0.f}, o[4] = {0.f, 0.f, 0.f, 0.f};
  const T* qp = static_cast<const T*>(a.q) + ((static_cast<size_t>(b) * a.H + h) * a.S + s) * a.dk;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d0 + i < a.dk) q[i] = static_cast<float>(qp[d0 + i]);
  float m = -INFINITY, l = 0.f;
  auto load = [&](const uint8_t* codes, const uint8_t* scales, int j, float* x) {
    unsigned c = 0, e = 127;
    if (mine) {
      const size_t at = ((static_cast<size_t>(b) * a.Hkv + h / group) * a.P + j) * nb + blk;
      c = *reinterpret_cast<const uint16_t*>(codes + at * kBlockBytes + (d0 % kBlock) / 2);
      e = scales[at];
    }
    const float sc = scale_value(e);
    const f2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 0);
    const f2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, sc, 1);
    x[0] = x0.x, x[1] = x0.y, x[2] = x1.x, x[3] = x1.y;
    if (e == kScaleNaN) x[0] = x[1] = x[2] = x[3] = __builtin_nanf("");
  };
  for (int j = w; j < keys; j += 4) {
    float x[4];
    load(a.k_codes, a.k_scales, j, x);
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) dot += q[i] * x[i];
    const float sc = wave_sum(dot) / a.scale;
    const float mn = fmaxf(m, sc), ref = mn == -INFINITY ? 0.f : mn;
    const float f = expf(m - ref), p = expf(sc - ref);
    load(a.v_codes, a.v_scales, j, x);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + p * x[i];
    m = mn;
  }
  if (lane == 0) sm[w] = m, sl[w] = l;
#pragma unroll
  for (int i = 0; i < 4; ++i) so[w][d0 + i] = o[i];
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), ref = mm == -INFINITY ? 0.f : mm;
  float f[4], lt = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = expf(sm[i] - ref);
    lt += sl[i] * f[i];
  }
  const int d = threadIdx.x;
  if (d < a.dk) {
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v += so[i][d] * f[i];
    T* out = static_cast<T*>(a.out) + (static_cast<size_t>(b) * a.S + s) * a.H * a.dk + static_cast<size_t>(h) * a.dk;
    out[d] = static_cast<T>(keys > 0 ? v / lt : 0.f);
  }
}

unsigned quads(int S, int H, int dk) {
  const long long lanes = 4LL * S * H * ((dk + kBlock - 1) / kBlock);
  return static_cast<unsigned>((lanes + 255) / 256);
}

template <typename T>
int write_launch(const Kv4WriteArgs& a, hipStream_t st) {
  const dim3 grid(quads(a.S, a.H, a.dk), a.B, 2);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  const bool vec = (bits & 15) == 0 && ((a.dk | a.stride_b | a.stride_h | a.stride_s) & 7) == 0;
  // the order in which the input lies in memory
  const bool heads = a.stride_h < a.stride_s;
  if (vec && heads) kv4_write_kernel<T, true, true><<<grid, 256, 0, st>>>(a);
  else if (vec) kv4_write_kernel<T, true, false><<<grid, 256, 0, st>>>(a);
  else if (heads) kv4_write_kernel<T, false, true><<<grid, 256, 0, st>>>(a);
  else kv4_write_kernel<T, false, false><<<grid, 256, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

template <typename T>
int read_launch(const Kv4ReadArgs& a, hipStream_t st) {
  const dim3 grid(quads(a.S, a.H, a.dk), a.B, 2);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out);
  if ((bits & 15) == 0 && (a.dk & 7) == 0) kv4_read_kernel<T, true><<<grid, 256, 0, st>>>(a);
  else kv4_read_kernel<T, false><<<grid, 256, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

}  // namespace

int launch_kv4_write(int dt, const Kv4WriteArgs& a, hipStream_t st) {
  return dt == F16 ? write_launch<half_t>(a, st) : write_launch<float>(a, st);
}

int launch_kv4_read(int dt, const Kv4ReadArgs& a, hipStream_t st) {
  return dt == F16 ? read_launch<half_t>(a, st) : read_launch<float>(a, st);
}

size_t kv4_attention_workspace(int B, int H, int Hkv, int S, int P, int dk) { return 0; }

int launch_kv4_attention(int dt, const Kv4AttnArgs& a, hipStream_t st) {
  const dim3 grid(a.S, a.H, a.B);
  if (dt == F16) kv4_attention_kernel<half_t><<<grid, 256, 0, st>>>(a);
  else kv4_attention_kernel<float><<<grid, 256, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

}  // namespace nml
