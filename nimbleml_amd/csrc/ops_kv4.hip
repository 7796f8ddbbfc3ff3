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

// ---------------------------------------------------------------------- attention
//
// The queries that share a KV head — its group's heads times the new tokens — are the columns of
// 16-wide MFMA tiles: S = K·Qᵀ takes 16 keys' blocks as its rows (a lane converts the codes it
// loaded and has its operand, no LDS), O = Vᵀ·Pᵀ takes the probabilities from the lanes where S
// left them, with the keys of the contraction in that order. Only V passes through LDS, for the
// transpose of its read. The codes' values are exact in bf16, a query is split in two (float16)
// or three (float32) bf16 parts without loss and a probability into as many, so every product
// is exact and scores, statistics and outputs are float32 sums.
//
// A wave goes through tiles of 32 keys on its own: its loads of the next tile are in flight
// during this one; the running maximum that the exponentials refer to moves only when a score
// passes it by 2^8 (probabilities are then at most 2^8, all the same to float32), which skips
// the rescaling of O on nearly every tile. Waves merge in LDS, the splits of a long row in a
// second launch.

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr int kKeys = 32;                  // keys of a wave's tile
constexpr int kSpan = kWaves * kKeys;      // a split takes a multiple of these
constexpr float kSlack = 8.f;              // in powers of two

// Keys of a split when a row's are dealt to `splits`.
__host__ __device__ __forceinline__ int split_keys(int len, int splits) {
  const int per = (len + splits - 1) / splits;
  return per < kSpan ? kSpan : (per + kSpan - 1) / kSpan * kSpan;
}

// One row of the batch: cached length and new tokens, in range.
struct RowInfo {
  int len, n;
};
__device__ __forceinline__ RowInfo row_info(const Kv4AttnArgs& a, int b, int* err) {
  RowInfo r;
  r.n = row_count(a.counts, b, a.S, err);
  const int len = a.lens[b];
  r.len = len < 0 ? 0 : (len > a.P ? a.P : len);
  if (r.len != len && err) __hip_atomic_fetch_or(err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return r;
}

// x = Σ of NP bf16 parts (the rest lost is below 2^-8·NP of x).
template <int NP>
__device__ __forceinline__ void split_bf16(float x, __bf16* part) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    part[p] = static_cast<__bf16>(x);
    x -= static_cast<float>(part[p]);
  }
}

// What a lane holds of one tile: of keys l % 16 and 16 + l % 16, values 8·NB·(l / 16) on.
template <int NB>
struct Kv4Tile {
  static constexpr int W = NB > 4 ? 2 : 1;  // blocks a lane's values touch
  unsigned c[2][NB];
  unsigned e[2][W];
};

template <int NB>
__device__ __forceinline__ void load_tile(Kv4Tile<NB>& t, const uint8_t* __restrict__ codes,
                                          const uint8_t* __restrict__ scales, int k0, int last, int nb, int lane) {
  constexpr int W = Kv4Tile<NB>::W;
  const int g = lane >> 4;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const int key = min(k0 + 16 * s + (lane & 15), last);  // (past the end: the last key again)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int blk = min(g * NB / 4 + w, nb - 1);  // (blocks that pad nb: the last one again)
      const size_t at = static_cast<size_t>(key) * nb + blk;
      const uint8_t* p = codes + at * kBlockBytes;
      if constexpr (NB >= 4) {
        const u4 v = *reinterpret_cast<const u4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.c[s][4 * w + i] = v[i];
      } else if constexpr (NB == 2) {
        const u2 v = *reinterpret_cast<const u2*>(p + (g & 1) * 8);
        t.c[s][0] = v[0];
        t.c[s][1] = v[1];
      } else {
        t.c[s][0] = *reinterpret_cast<const unsigned*>(p + g * 4);
      }
      t.e[s][w] = scales[at];
    }
  }
}

// Eight values as bf16.
__device__ __forceinline__ bf8 convert8(unsigned c, float s) {
  const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0);
  const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
  const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2);
  const bf2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
  return bf8{a.x, a.y, b.x, b.y, d.x, d.y, e.x, e.y};
}

// Keys of a 16-key subtile (bit i: key i) that hold a NaN block, from the lanes' scales; the
// NaN blocks themselves become zeros. `of`: per block, the keys; null: any block.
template <int NB>
__device__ __forceinline__ unsigned take_nan(Kv4Tile<NB>& t, int s, unsigned* of) {
  constexpr int W = Kv4Tile<NB>::W;
  unsigned any = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const bool bad = t.e[s][w] == kScaleNaN;
    const unsigned long long m = __ballot(bad);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const unsigned keys = static_cast<unsigned>(m >> (16 * g)) & 0xffffu;
      any |= keys;
      if (of) of[g * NB / 4 + w] |= keys;
    }
    if (bad) {
      t.e[s][w] = 127;
#pragma unroll
      for (int i = 0; i < NB / W; ++i) t.c[s][w * (NB / W) + i] = 0;
    }
  }
  return any;
}

template <typename T, int NB>
__global__ __launch_bounds__(256) void kv4_attention_kernel(Kv4AttnArgs a, int splits) {
  constexpr int NP = sizeof(T) == 2 ? 2 : 3;
  constexpr int W = Kv4Tile<NB>::W, DT = 2 * NB;  // DT: 16-wide tiles of the head dim
  constexpr int kRow = 64 * NB + 32;              // bytes of a key's values in LDS (+32: banks)
  constexpr int kWaveLds = kKeys * kRow;          // and 16 rows of 32·NB floats fit as well
  __shared__ __align__(16) char lds[kWaves * kWaveLds];
  __shared__ float sm[kWaves][16], sl[kWaves][16];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int split = blockIdx.x % splits, tile = blockIdx.x / splits, hk = blockIdx.y, b = blockIdx.z;
  const int nb = (a.dk + kBlock - 1) / kBlock, group = a.H / a.Hkv, R = group * a.S;
  const RowInfo row = row_info(a, b, split == 0 ? a.err : nullptr);
  const int per = split_keys(row.len, splits), active = max(1, (row.len + per - 1) / per);
  if (split >= active) return;
  const int k0 = split * per, k1 = min(row.len, k0 + per);

  // This lane's query: row r of the KV head's R, token s of head hk·group + r / S. It sees keys
  // up to lim; a column without a query (or of the padding) runs along with zeros.
  const int r = tile * 16 + col, s = r % a.S;
  const bool live = r < R && s < row.n;
  const int h = hk * group + r / a.S;
  const int lim = live ? row.len - row.n + s : 0x7fffffff;
  int least = lim;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) least = min(least, __shfl_xor(least, o, 64));

  bf8 q[NP][NB];
  {
    const T* qp = static_cast<const T*>(a.q) + ((static_cast<size_t>(b) * a.H + (live ? h : 0)) * a.S + (live ? s : 0)) * a.dk;
    const bool vec = (a.dk & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0;
#pragma unroll
    for (int t = 0; t < NB; ++t) {
      float x[8];
      const int d0 = 8 * (g * NB + t);
      if (vec) load8<T, true>(qp, d0, a.dk, x);
      else load8<T, false>(qp, d0, a.dk, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        __bf16 part[NP];
        split_bf16<NP>(live ? x[i] : 0.f, part);
#pragma unroll
        for (int p = 0; p < NP; ++p) q[p][t][i] = part[p];
      }
    }
  }
  const float scale = 1.44269504088896341f / a.scale;  // scores in powers of two
  floatx4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, ref = 0.f, l = 0.f;  // l: of this lane's keys
  unsigned nan_blocks = 0;                  // blocks of the output that a NaN block of V reached

  const size_t head = (static_cast<size_t>(b) * a.Hkv + hk) * a.P * nb;
  const uint8_t* kc = a.k_codes + head * kBlockBytes;
  const uint8_t* ks = a.k_scales + head;
  const uint8_t* vc = a.v_codes + head * kBlockBytes;
  const uint8_t* vs = a.v_scales + head;
  char* mine = lds + w * kWaveLds;
  Kv4Tile<NB> kt, vt;
  int j = k0 + w * kKeys;
  if (j < k1) {
    load_tile<NB>(kt, kc, ks, j, row.len - 1, nb, lane);
    load_tile<NB>(vt, vc, vs, j, row.len - 1, nb, lane);
  }
  for (; j < k1; j += kSpan) {
    Kv4Tile<NB> k = kt, v = vt;
    if (j + kSpan < k1) {
      load_tile<NB>(kt, kc, ks, j + kSpan, row.len - 1, nb, lane);
      load_tile<NB>(vt, vc, vs, j + kSpan, row.len - 1, nb, lane);
    }
    unsigned bad_e = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < W; ++i) bad_e = max(bad_e, max(k.e[t][i], v.e[t][i]));
    const bool nan = __ballot(bad_e == kScaleNaN) != 0;
    unsigned k_nan[2] = {0, 0};
    if (nan) {
      for (int t = 0; t < 2; ++t) {
        k_nan[t] = take_nan<NB>(k, t, nullptr);
        unsigned of[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        take_nan<NB>(v, t, of);
        const int seen = min(max(min(lim, k1 - 1) - (j + 16 * t) + 1, 0), 16);
        const unsigned vis = (1u << seen) - 1u;
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (of[i] & vis) nan_blocks |= 1u << i;
      }
    }
    // S = K·Qᵀ: this lane's are keys 4g … 4g+3 of both subtiles with its query
    float x[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const bf8 kk = convert8(k.c[t][i], scale_value(k.e[t][W == 2 ? i / 4 : 0]));
#pragma unroll
        for (int p = 0; p < NP; ++p) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kk, q[p][i], acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * t + i] = acc[i] * scale;
    }
    // V to LDS, a key a row
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < NB; ++i)
        *reinterpret_cast<bf8*>(mine + (16 * t + col) * kRow + 16 * (g * NB + i)) =
            convert8(v.c[t][i], scale_value(v.e[t][W == 2 ? i / 4 : 0]));
    if (nan) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (k_nan[i / 4] >> (4 * g + i % 4) & 1u) x[i] = __builtin_nanf("");
    }
    if (j + kKeys - 1 > least) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j + 16 * (i / 4) + 4 * g + i % 4 > lim) x[i] = -INFINITY;
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
    if (__ballot(top > m + kSlack)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m, top), rn = mn == -INFINITY ? 0.f : mn;
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - rn);
      m = mn;
      ref = rn;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    bf8 p[NP];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(x[i] - ref);
      l += e;
      __bf16 part[NP];
      split_bf16<NP>(e, part);
#pragma unroll
      for (int c = 0; c < NP; ++c) p[c][i] = part[c];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (LDS of this wave alone, in order)
    // O += Vᵀ·Pᵀ: four keys of either subtile and 16 dims a transposing read
    const char* at = mine + (4 * g + col / 4) * kRow + (col % 4) * 8;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 32 * d));
      const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * kRow + 32 * d));
      typedef short s8 __attribute__((ext_vector_type(8)));
      const bf8 vv = __builtin_bit_cast(bf8, s8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
#pragma unroll
      for (int c = 0; c < NP; ++c) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, p[c], o[d], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // The waves' parts: o[d] holds dims 16d + 4g … + 3 of this lane's query.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) sm[w][col] = m, sl[w][col] = l;
  float* part = reinterpret_cast<float*>(mine);
  constexpr int D = 32 * NB;
  if (live) {
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (nan_blocks >> (d / 2) & 1u) o[d] = floatx4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
      *reinterpret_cast<floatx4*>(part + col * D + 16 * d + 4 * g) = o[d];
    }
  }
  __syncthreads();
  const int rows = min(16, R - tile * 16);
  for (int i = threadIdx.x; i < rows * D; i += 256) {
    const int c = i / D, d = i % D, rr = tile * 16 + c, ss = rr % a.S;
    if (ss >= row.n || d >= a.dk) continue;
    float mm = sm[0][c];
#pragma unroll
    for (int y = 1; y < kWaves; ++y) mm = fmaxf(mm, sm[y][c]);
    const float rf = mm == -INFINITY ? 0.f : mm;
    float lt = 0.f, ot = 0.f;
#pragma unroll
    for (int y = 0; y < kWaves; ++y) {
      const float f = __builtin_amdgcn_exp2f(sm[y][c] - rf);  // (−inf: 0)
      lt += sl[y][c] * f;
      ot += reinterpret_cast<const float*>(lds + y * kWaveLds)[c * D + d] * f;
    }
    const int hh = hk * group + rr / a.S;
    if (active == 1) {
      T* out = static_cast<T*>(a.out) + (static_cast<size_t>(b) * a.S + ss) * a.H * a.dk + static_cast<size_t>(hh) * a.dk;
      out[d] = static_cast<T>(row.len - row.n + ss < 0 ? 0.f : ot / lt);
    } else {
      const size_t p = ((static_cast<size_t>(b) * a.H + hh) * a.S + ss) * splits + split;
      float* ws = static_cast<float*>(a.ws);
      const size_t parts = static_cast<size_t>(a.B) * a.H * a.S * splits;
      if (d == 0) ws[2 * p] = mm, ws[2 * p + 1] = lt;
      ws[2 * parts + p * a.dk + d] = ot;
    }
  }
}

// The splits of one query's row, in order.
template <typename T>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4AttnArgs a, int splits) {
  const int s = blockIdx.x, h = blockIdx.y, b = blockIdx.z, d = threadIdx.x;
  const RowInfo row = row_info(a, b, nullptr);
  const int per = split_keys(row.len, splits), active = max(1, (row.len + per - 1) / per);
  if (active == 1 || s >= row.n || d >= a.dk) return;
  const size_t p = ((static_cast<size_t>(b) * a.H + h) * a.S + s) * splits;
  const float* ml = static_cast<const float*>(a.ws) + 2 * p;
  const float* o = static_cast<const float*>(a.ws) + 2 * static_cast<size_t>(a.B) * a.H * a.S * splits + p * a.dk + d;
  float m = -INFINITY, l = 0.f, v = 0.f;
  for (int i = 0; i < active; ++i) m = fmaxf(m, ml[2 * i]);
  const float ref = m == -INFINITY ? 0.f : m;
  for (int i = 0; i < active; ++i) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * i] - ref);
    l += ml[2 * i + 1] * f;
    v += o[static_cast<size_t>(i) * a.dk] * f;
  }
  T* out = static_cast<T*>(a.out) + (static_cast<size_t>(b) * a.S + s) * a.H * a.dk + static_cast<size_t>(h) * a.dk;
  out[d] = static_cast<T>(row.len - row.n + s < 0 ? 0.f : v / l);
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

// Workgroups that fill the card (four on each of 256 CUs); a row's keys are split until there
// are as many, in pieces of at least kSpan keys.
int attention_splits(int B, int H, int Hkv, int S, int P) {
  const long long tiles = (static_cast<long long>(H / Hkv) * S + 15) / 16;
  const long long groups = tiles * Hkv * B, want = (1024 + groups - 1) / groups, most = (P + kSpan - 1) / kSpan;
  return static_cast<int>(want < most ? want : most);
}

template <typename T, int NB>
int attention_launch_nb(const Kv4AttnArgs& a, int splits, hipStream_t st) {
  const unsigned tiles = (static_cast<unsigned>(a.H / a.Hkv) * a.S + 15) / 16;
  kv4_attention_kernel<T, NB><<<dim3(tiles * splits, a.Hkv, a.B), 256, 0, st>>>(a, splits);
  NML_LAUNCHED();
  if (splits > 1) {
    kv4_combine_kernel<T><<<dim3(a.S, a.H, a.B), a.dk <= 64 ? 64 : a.dk <= 128 ? 128 : 256, 0, st>>>(a, splits);
    NML_LAUNCHED();
  }
  return 0;
}

template <typename T>
int attention_launch(const Kv4AttnArgs& a, hipStream_t st) {
  const int splits = attention_splits(a.B, a.H, a.Hkv, a.S, a.P), nb = (a.dk + kBlock - 1) / kBlock;
  if (nb == 1) return attention_launch_nb<T, 1>(a, splits, st);
  if (nb == 2) return attention_launch_nb<T, 2>(a, splits, st);
  if (nb <= 4) return attention_launch_nb<T, 4>(a, splits, st);
  return attention_launch_nb<T, 8>(a, splits, st);
}

}  // namespace

int launch_kv4_write(int dt, const Kv4WriteArgs& a, hipStream_t st) {
  return dt == F16 ? write_launch<half_t>(a, st) : write_launch<float>(a, st);
}

int launch_kv4_read(int dt, const Kv4ReadArgs& a, hipStream_t st) {
  return dt == F16 ? read_launch<half_t>(a, st) : read_launch<float>(a, st);
}

size_t kv4_attention_workspace(int B, int H, int Hkv, int S, int P, int dk) {
  const int splits = attention_splits(B, H, Hkv, S, P);
  return splits == 1 ? 0 : sizeof(float) * static_cast<size_t>(B) * H * S * splits * (dk + 2);
}

int launch_kv4_attention(int dt, const Kv4AttnArgs& a, hipStream_t st) {
  return dt == F16 ? attention_launch<half_t>(a, st) : attention_launch<float>(a, st);
}

}  // namespace nml
