// A KV cache in 4 bits: written, read back and attended to.
//
// Format (one head's vector of dk values, ⌈dk/32⌉ blocks of 32, the last padded with zeros):
// 32 E2M1 codes (0 ½ 1 1½ 2 3 4 6 with a sign; the first of two in a byte's low half) and one
// scale byte e that stands for 2^(e − 127), 255 for NaN: 17 bytes a block, 4.25 bits a value and
// 3.76 times fewer bytes than fp16 where dk is a multiple of 32. gfx950 converts two codes to two
// values, scale included, in one instruction, and rounds two values to two codes in another.
//
// With 2^k ≤ max|x| < 2^(k+1) the scale is 2^(k−2), or 2^(k−1) where max|x| ≥ 1.75·2^k: there
// saturating the largest value at 6 would cost more than the coarser step (signal to error on
// normal values 19.02 dB with the change at 1.75, 18.75 at 1.5, 18.79 without it; 16.33, 15.41
// and 16.30 with one channel of 32 six times as large).
#include <algorithm>

#include "kernels.hpp"

namespace nml {

namespace {

constexpr int kBlock = 32;            // values of one scale
constexpr int kBlockBytes = 16;       // and their codes
constexpr int kMinExp = -120;         // ½·2^-120 is a normal float32 and bf16
constexpr unsigned kScaleNaN = 255u;
// A writing or reading workgroup, and the blocks that a lane of it takes: four loads in flight
// (K and V of 4 × 4096 tokens of 16 heads × 128 float16 values: written and read back in 72 µs, 82
// with one load; read in 34 µs, 45 with one. 5.0 TB/s: bound by memory. A step's few tokens take
// the time of two launches).
constexpr int kWriters = 256, kEach = 4;

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

// Items of one row b in the order of the cache: (h, s, block), the block fastest, whatever the
// order of the other side, so that a workgroup writes whole lines of codes and scales (in the
// order of a (batch, seq, heads, dk) input 2 % slower). Four lanes share a block, eight values each.
struct Items {
  Div by_blocks, by_tokens;
  int nb, tokens, count;
};
struct Item {
  int s, h, blk;
};
__device__ __forceinline__ Item item_of(unsigned i, const Items& n) {
  const unsigned t = quotient(i, n.by_blocks), h = quotient(t, n.by_tokens);
  return Item{static_cast<int>(t - h * n.tokens), static_cast<int>(h), static_cast<int>(i - t * n.nb)};
}
Items items_of(int S, int H, int dk) {
  Items n;
  n.nb = (dk + kBlock - 1) / kBlock;
  n.tokens = S;
  n.count = S * H * n.nb;
  n.by_blocks = div_by(n.nb);
  n.by_tokens = div_by(S);
  return n;
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

// Codes and scale byte of a block that four lanes hold, eight values each (the lane's codes).
template <typename T>
__device__ __forceinline__ unsigned encode8(const float* x, unsigned& scale) {
  // max|x| on the bits: infinity and NaN are the largest
  unsigned top = 0, codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned w = __builtin_bit_cast(unsigned, x[i]) & 0x7fffffffu;
    top = top > w ? top : w;
  }
  top = quad_umax(top);
  scale = kScaleNaN;
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
  return codes;
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kWriters) void kv4_write_kernel(Kv4WriteArgs a, Items n) {
  const int b = blockIdx.y;
  const unsigned part = threadIdx.x & 3u;
  const unsigned first = blockIdx.x * static_cast<unsigned>(kEach * kWriters / 4) + (threadIdx.x >> 2);
  const bool is_v = blockIdx.z != 0;
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + b * a.stride_b;
  const int count = row_count(a.counts, b, a.S, a.err), pos = a.pos ? a.pos[b] : 0;
  float x[kEach][8];
  size_t at[kEach];
  bool here[kEach];
  // (a block's four lanes have the same item: they come and go together)
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const unsigned item = first + u * (kWriters / 4);
    const Item it = item_of(item, n);
    const long long p = static_cast<long long>(pos) + it.s;
    here[u] = item < static_cast<unsigned>(n.count) && it.s < count;
    if (here[u] && (p < 0 || p >= a.P)) {
      here[u] = false;
      if (a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    at[u] = ((static_cast<size_t>(b) * a.H + it.h) * a.P + p) * n.nb + it.blk;
    if (here[u]) load8<T, VEC>(src + it.h * a.stride_h + (a.src_at_pos ? p : it.s) * a.stride_s, it.blk * kBlock + part * 8, a.dk, x[u]);
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (!here[u]) continue;
    unsigned scale;
    const unsigned codes = encode8<T>(x[u], scale);
    *reinterpret_cast<unsigned*>((is_v ? a.v_codes : a.k_codes) + at[u] * kBlockBytes + part * 4) = codes;
    if (part == 0) (is_v ? a.v_scales : a.k_scales)[at[u]] = static_cast<uint8_t>(scale);
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(kWriters) void kv4_read_kernel(Kv4ReadArgs a, Items n) {
  typedef T v8 __attribute__((ext_vector_type(8), aligned(16)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  const int b = blockIdx.y;
  const unsigned part = threadIdx.x & 3u;
  const unsigned first = blockIdx.x * static_cast<unsigned>(kEach * kWriters / 4) + (threadIdx.x >> 2);
  const bool is_v = blockIdx.z != 0;
  const uint8_t *from = is_v ? a.v_codes : a.k_codes, *scales = is_v ? a.v_scales : a.k_scales;
  T* to = static_cast<T*>(is_v ? a.v_out : a.k_out);
  const int count = row_count(a.counts, b, a.S, a.err), pos = a.pos ? a.pos[b] : 0;
  Item it[kEach];
  unsigned codes[kEach], scale[kEach];
  bool here[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const unsigned item = first + u * (kWriters / 4);
    it[u] = item_of(item, n);
    here[u] = item < static_cast<unsigned>(n.count) && it[u].s < count && it[u].blk * kBlock + static_cast<int>(part) * 8 < a.dk;
    codes[u] = 0;
    scale[u] = 127;
    const long long p = static_cast<long long>(pos) + it[u].s;
    if (here[u]) {
      if (p >= 0 && p < a.P) {
        const size_t at = ((static_cast<size_t>(b) * a.H + it[u].h) * a.P + p) * n.nb + it[u].blk;
        codes[u] = *reinterpret_cast<const unsigned*>(from + at * kBlockBytes + part * 4);
        scale[u] = scales[at];
      } else if (a.err) {
        __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (!here[u]) continue;
    const float s = scale_value(scale[u]);
    const f2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], s, 0);
    const f2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], s, 1);
    const f2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], s, 2);
    const f2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[u], s, 3);
    float x[8] = {x0.x, x0.y, x1.x, x1.y, x2.x, x2.y, x3.x, x3.y};
    if (scale[u] == kScaleNaN) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
    }
    const int d0 = it[u].blk * kBlock + part * 8;
    T* out = to + ((static_cast<size_t>(b) * a.H + it[u].h) * (a.out_tokens ? a.out_tokens : a.S) + it[u].s) * a.dk + d0;
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
}

// ---------------------------------------------------------------------- attention
//
// The queries that share a KV head — its group's heads times the new tokens — are the columns of
// 16-wide MFMA tiles: S = K·Qᵀ takes 16 keys' blocks as its rows (a lane converts the codes it
// loaded and has its operand, no LDS), O = Vᵀ·Pᵀ takes the probabilities from the lanes where S
// left them, with the keys of the contraction in that order. V passes through LDS for the
// transpose of its read; Q is split and laid out in LDS once a workgroup. The codes' values are
// exact in bf16 and a query is split in two (float16) or three (float32) bf16 parts without loss, so
// scores are float32 sums of exact products. A float32 probability enters the product with V as as
// many parts: 24 bits in float32, 17 in float16, whose output has 11; Σ p is of the whole ones.
//
// A wave goes through tiles of 32 keys on its own: its loads of the next tile are in flight
// during this one; the running maximum that the exponentials refer to moves only when a score
// passes it by 2^8 (probabilities are then at most 2^8, all the same to float32), which skips
// the rescaling of O on nearly every tile. A workgroup's waves merge in LDS.
//
// A (row, KV head, 16 queries) is one workgroup's unless its keys are many: pieces of a long one
// go to several, as many in all as the card holds at once, and the last to finish merges them in
// their order.
//
// What bounds it: 8 rows of 8 Ki … 32 Ki keys, 8 KV heads of 128 with four query heads each, 38–45 µs
// from card to card, 4.0–4.7 TB/s of memory. 32 rows of 128 … 1280 keys, 16 heads of 64, 12 µs: 2 TB/s,
// the latency of a workgroup's few rounds. One row of 1023 keys 8 µs: 2.7 until the first tile is there and Q laid
// out, 0.8 a round, 1.8 for the merge and the store.

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

constexpr int kKeys = 32;                  // keys of a wave's tile
constexpr float kSlack = 8.f;              // in powers of two
// Scale bytes (2^65 and up) of values whose Σ p·v could pass float32's range (2^30 keys, p up to
// 2^kSlack). Looked for in float32 calls only: a float16 output holds no such values.
constexpr unsigned kLargeScale = 192;

// Waves of a workgroup: eight, which share a tile's keys where tiles are few; four where there are
// at least four times the workgroups of eight that the card holds, so that a short tile pays for
// fewer waves' startup and merge (16 heads of 64, µs with eight and four: 512 rows of up to 2048 keys
// 194, 157; 128 rows 54, 46; 128 rows of up to 8192 keys 154, 150; 512 rows of up to 512 keys and 8
// heads 60, 40; two waves 154, 49, 164, 34). At head dims above 128 LDS has room for eight either way.
constexpr int few_waves(int nb) { return nb <= 4 ? 4 : 8; }
constexpr int kManyTiles = 4;
// Workgroups that the card's 256 CUs hold at once, by registers and LDS.
__host__ __device__ constexpr int capacity(int nb, int waves) { return (nb == 1 ? 768 : nb <= 4 ? 512 : 256) * 8 / waves; }
// Spans that a piece has at least: what it costs to begin one and to merge it. (Head dim 64, 32 rows
// of 128 … 1280 keys: 12 µs at eight, where no row is split, 19 at two. 128, one row of 30 Ki keys
// with 8 KV heads: 15.6 µs at four, 18.5 at two, 18.9 at eight. 256, 4 rows of up to 8 Ki keys with
// 4 KV heads: 16.5 at two, 20.8 at four, 27.2 at eight.)
__host__ __device__ constexpr int least_spans(int nb, int waves) { return (nb <= 2 ? 8 : nb <= 4 ? 4 : 2) * 8 / waves; }

// ws: a counter for each tile in pieces (zero before and after every launch, in the same place
// for calls of any size), then for each piece its rows' maxima and Σ p, then their Σ p·v. Tiles in
// pieces are fewer than the card's workgroups (a piece is at least their even share), and so their
// pieces fewer than twice as many.
constexpr int kCounters = 2048, kCounterStep = 16;  // a line for each

// Places for pieces: those that the tiles' own workgroups leave on the card (a quarter of it where
// they leave none: for a row much longer than the others).
__host__ __device__ inline int room_for(long long tiles, int cap) {
  const int left = cap - static_cast<int>(tiles < cap ? tiles : cap);
  return left > cap / 4 ? left : cap / 4;
}

// Rows of the batch, 64 at a time with one in each lane: cached length and new tokens, in range;
// SPAN: keys of a workgroup's round.
template <int SPAN>
struct Rows {
  int len, n, spans;
  // Spans of the lane's row: at least one (its outputs are to be written), none past the batch.
  __device__ __forceinline__ bool load(const Kv4AttnArgs& a, int b) {
    const int at = min(b, a.B - 1), x = a.lens[at] + a.more, y = a.counts ? a.counts[at] : a.S;
    len = min(max(x, 0), a.P);
    n = min(max(y, 0), a.S);
    spans = b >= a.B ? 0 : n > 0 ? max(1, (len + SPAN - 1) / SPAN) : 1;
    return x == len && y == n;  // (were in range)
  }
};

// What this workgroup does: piece `piece` of `pieces` of tile (b, e), whose row has len keys and n
// new tokens; `slot`: where the tile's first piece is in ws. b < 0: nothing.
struct Work {
  int b, e, piece, pieces, slot, len, n, spans;
};
// More than 64 rows are shared out to the waves, a run of rows each (2048 rows × 8 heads of up to
// 512 keys of 64: 240 µs, of eight waves 310, 670 with every wave looking through them all); sums: of
// the waves.
template <int NB, int NW>
__device__ __forceinline__ Work find_work(const Kv4AttnArgs& a, int each, int lane, int wave, int (*sums)[3]) {
  Work w{};
  Rows<NW * kKeys> rows;
  const int run = a.B <= 64 ? 64 : (a.B + 64 * NW - 1) / (64 * NW) * 64;
  const int first = a.B <= 64 ? 0 : wave * run, end = min(first + run, a.B);
  int total = 0;
  bool good = true;
#pragma unroll 2
  for (int i = first; i < end; i += 64) {
    good &= rows.load(a, i + lane);
    total += rows.spans;
  }
  if (!good && blockIdx.x == 0 && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  total = __builtin_amdgcn_readlane(wave_scan(total), 63);
  if (a.B > 64) {
    if (lane == 0) sums[wave][0] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += sums[i][0];
  }
  const int room = room_for(static_cast<long long>(each) * a.B, capacity(NB, NW));
  const int least = max(least_spans(NB, NW), static_cast<int>((static_cast<long long>(total) * each + room - 1) / room));
  auto pieces_of = [&](int spans) { return spans <= least ? min(spans, 1) : (spans + least - 1) / least; };
  const int at = static_cast<int>(blockIdx.x / each);
  int before = 0, slots = 0, from = 0;
  if (a.B > 64) {
    int pieces = 0, split = 0;
#pragma unroll 2
    for (int i = first; i < end; i += 64) {
      rows.load(a, i + lane);
      const int p = pieces_of(rows.spans);
      pieces += p;
      split += p > 1 ? p : 0;
    }
    pieces = wave_scan(pieces);
    split = wave_scan(split);
    if (lane == 63) sums[wave][1] = pieces, sums[wave][2] = split;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i)  // the run that has this workgroup's row
      if (from == i * run && before + sums[i][1] <= at) {
        before += sums[i][1];
        slots += sums[i][2];
        from += run;
      }
  }
  for (int i = from; i < min(from + run, a.B); i += 64) {
    if (a.B > 64) rows.load(a, i + lane);
    const int pieces = pieces_of(rows.spans);
    const int sum = wave_scan(pieces), sum_slots = wave_scan(pieces > 1 ? pieces : 0);
    const unsigned long long past = __ballot(before + sum > at);
    if (past) {
      const int l = __ffsll(past) - 1;
      w.pieces = __builtin_amdgcn_readlane(pieces, l);
      w.spans = __builtin_amdgcn_readlane(rows.spans, l);
      w.len = __builtin_amdgcn_readlane(rows.len, l);
      w.n = __builtin_amdgcn_readlane(rows.n, l);
      const int start = before + __builtin_amdgcn_readlane(sum, l) - w.pieces;
      const int local = static_cast<int>(blockIdx.x) - start * each;
      w.b = i + l;
      w.e = w.pieces == 1 ? local : local / w.pieces;
      w.piece = local - w.e * w.pieces;
      w.slot = (slots + __builtin_amdgcn_readlane(sum_slots, l) - w.pieces) * each + w.e * w.pieces;
      return w;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(sum_slots, 63);
  }
  w.b = -1;
  return w;
}

// x = Σ of NP bf16 parts, two values at once (what is lost is below 2^(1 − 8·NP − NP) of x).
template <int NP>
__device__ __forceinline__ void split_bf16(f2 x, bf2* part) {
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    part[p] = __builtin_convertvector(x, bf2);
    if (p + 1 < NP) x -= __builtin_convertvector(part[p], f2);
  }
}

// What a lane holds of one tile: of keys l % 16 and 16 + l % 16, values 8·NB·(l / 16) on.
template <int NB>
struct Kv4Tile {
  static constexpr int W = NB > 4 ? 2 : 1;  // blocks a lane's values touch
  unsigned c[2][NB];
  uint8_t e[2][W];  // (as loaded: widened at their use, or the wait for them moves up to the load)
};

// Tile at `codes` and `scales` (those of its first key). Keys past `last` (of the tile): that key
// again; blocks that pad nb: the last one again.
template <int NB>
__device__ __forceinline__ void load_tile(Kv4Tile<NB>& t, const uint8_t* __restrict__ codes,
                                          const uint8_t* __restrict__ scales, int last, int nb, int lane) {
  constexpr int W = Kv4Tile<NB>::W;
  const int g = lane >> 4;
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const unsigned key = min(16 * s + (lane & 15), last);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const unsigned at = key * nb + min(g * NB / 4 + w, nb - 1);
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

// As scale_value (the conversions to bf16 take the exponent's bits alone: a byte of 0 is 2^-127 here
// too).
__device__ __forceinline__ float tile_scale(unsigned e) { return __builtin_bit_cast(float, e << 23); }

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

// V in LDS: a key's 32·NB values in a row, its 32-byte pairs exchanged by the key so that the
// 16 rows that a transposing read takes 32 bytes each of lie in different banks.
template <int NB>
__device__ __forceinline__ int v_pair(int key, int pair) {
  return pair ^ (NB >= 4 ? key & 7 : NB == 2 ? key >> 1 & 3 : key >> 2 & 1);
}

// Partial results pass between workgroups of any XCD: stores and loads at agent scope (past the
// L2s) and a count that each workgroup adds to once its stores have arrived. (With an acquire in
// the last one and plain loads, which empties that XCD's L2, 32 rows of 128 … 1280 keys took 32 µs
// instead of 17.)
__device__ __forceinline__ void put2(float* p, f2 v) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 get2(const float* p) {
  return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                  __HIP_MEMORY_SCOPE_AGENT));
}

// ADD: the row's last key and value come from a.new_k and a.new_v and are not in the cache yet. (Of
// its own: the calls without it take 2 % longer beside that code, 4 % on long rows.)
template <typename T, int NB, int NW, bool ADD>
__global__ __launch_bounds__(64 * NW, NB == 1 ? 6 : NB <= 4 ? 4 : 2) void kv4_attention_kernel(Kv4AttnArgs a) {
  constexpr int NP = sizeof(T) == 2 ? 2 : 3;
  constexpr int W = Kv4Tile<NB>::W, DT = 2 * NB;  // DT: 16-wide tiles of the head dim
  constexpr int kRow = 64 * NB;                   // bytes of a key's values in LDS
  constexpr int kWaveLds = kKeys * kRow;          // and as many of 16 rows of 32·NB floats
  constexpr int D = 32 * NB, kThreads = 64 * NW, kSpan = NW * kKeys;
  constexpr unsigned kLarge = NP == 3 ? kLargeScale : kScaleNaN;
  static_assert(NW >= NB, "a wave lays out a step of Q");
  __shared__ __align__(16) char lds[NW * kWaveLds];
  __shared__ __align__(16) bf8 qs[NP][NB][64];
  __shared__ float sm[NW][16], sl[NW][16];
  __shared__ __align__(16) unsigned new_codes[2][ADD ? 8 : 1][4];  // of the row's last key and value
  __shared__ uint8_t new_scales[2][ADD ? 8 : 1];
  __shared__ unsigned arrived;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int nb = (a.dk + kBlock - 1) / kBlock, R = a.group * a.S, tiles = (R + 15) / 16;
  const Work work = find_work<NB, NW>(a, a.Hkv * tiles, lane, w, reinterpret_cast<int(*)[3]>(lds));
  if (work.b < 0 || work.n == 0) return;
  const int hk = tiles == 1 ? work.e : work.e / tiles, tile = work.e - hk * tiles;
  const int per = work.pieces == 1 ? work.spans : (work.spans + work.pieces - 1) / work.pieces;
  const int k0 = work.piece * per * kSpan, k1 = min(work.len, k0 + per * kSpan);

  // The query of column c of this tile: row r of the KV head's R, token s of head hk·group + r / S.
  // It sees keys up to lim; a column without a query (or of the padding) runs along with zeros.
  auto token = [&](int r) { return a.S == 1 ? 0 : r % a.S; };
  auto head = [&](int r) { return hk * a.group + (a.S == 1 ? r : r / a.S); };
  const int r = tile * 16 + col, s = token(r);
  const bool live = r < R && s < work.n;
  const int lim = live ? work.len - work.n + s : 0x7fffffff;

  // Q as it lies in memory, eight values a lane (wave t: step t of the product), in flight while
  // the keys' loads are issued
  typedef T v8 __attribute__((ext_vector_type(8), aligned(16)));
  v8 raw = {};
  const int d0 = 8 * (g * NB + w);
  if (w < NB && live) {
    const T* qp = static_cast<const T*>(a.q) + ((static_cast<size_t>(work.b) * a.H + head(r)) * a.S + s) * a.dk;
    if ((a.dk & 7) == 0 && (reinterpret_cast<uintptr_t>(a.q) & 15) == 0) {
      if (d0 < a.dk) raw = *reinterpret_cast<const v8*>(qp + d0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (d0 + i < a.dk) raw[i] = qp[d0 + i];
    }
  }

  // A step's own key and value, not in the cache yet: the last wave of the workgroup that has that
  // key codes them, writes them there and leaves them in LDS for the tile that holds them.
  const bool adds = ADD && k0 < k1 && k1 == work.len;
  const int at_v = lane >> 5, at_blk = (lane & 31) >> 2, at_part = lane & 3;
  float fresh[8];
  if (adds && w == NW - 1) {
    const T* p = static_cast<const T*>(at_v ? a.new_v : a.new_k) + work.b * a.new_b + hk * a.new_h +
                 static_cast<long long>(work.len - 1) * a.dk;
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.new_k) | reinterpret_cast<uintptr_t>(a.new_v);
    if ((bits & 15) == 0 && ((a.dk | a.new_b | a.new_h) & 7) == 0) load8<T, true>(p, 32 * at_blk + 8 * at_part, a.dk, fresh);
    else load8<T, false>(p, 32 * at_blk + 8 * at_part, a.dk, fresh);
  }

  const size_t base = (static_cast<size_t>(work.b) * a.Hkv + hk) * a.P * nb;
  const uint8_t* kc = a.k_codes + base * kBlockBytes;
  const uint8_t* ks = a.k_scales + base;
  const uint8_t* vc = a.v_codes + base * kBlockBytes;
  const uint8_t* vs = a.v_scales + base;
  // A tile of keys from `at` on. Past the piece's end: its first key again and again, so that
  // every round issues as many loads (the waits before their use count them).
  Kv4Tile<NB> k, v;
  auto fetch = [&](int at) {
    const int from = at < k1 ? at : k0, last = at < k1 ? work.len - 1 - at : 0;
    const size_t o = static_cast<size_t>(from) * nb;
    load_tile<NB>(k, kc + o * kBlockBytes, ks + o, last, nb, lane);
    load_tile<NB>(v, vc + o * kBlockBytes, vs + o, last, nb, lane);
  };
  int j = k0 + w * kKeys;
  if (k0 < k1) fetch(j);

  if (w < NB) {
    bf8 q[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      bf2 part[NP];
      split_bf16<NP>(f2{static_cast<float>(raw[i]), static_cast<float>(raw[i + 1])}, part);
#pragma unroll
      for (int p = 0; p < NP; ++p) q[p][i] = part[p].x, q[p][i + 1] = part[p].y;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) qs[p][w][lane] = q[p];
  }
  if (adds && w == NW - 1) {
    unsigned scale_byte;
    const unsigned codes = encode8<T>(fresh, scale_byte);
    new_codes[at_v][at_blk][at_part] = codes;
    if (at_part == 0) new_scales[at_v][at_blk] = static_cast<uint8_t>(scale_byte);
    if (at_blk < nb) {
      const size_t to = static_cast<size_t>(work.len - 1) * nb + at_blk;
      *reinterpret_cast<unsigned*>(const_cast<uint8_t*>((at_v ? vc : kc) + to * kBlockBytes + at_part * 4)) = codes;
      if (at_part == 0) const_cast<uint8_t*>(at_v ? vs : ks)[to] = static_cast<uint8_t>(scale_byte);
    }
  }
  // that key (and those past it, which repeat it) in a tile from `at` on
  auto take_new = [&](Kv4Tile<NB>& t, int which, int at) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (at + 16 * h + col >= work.len - 1) {
#pragma unroll
        for (int y = 0; y < W; ++y) {
          const int blk = min(g * NB / 4 + y, nb - 1);
          t.e[h][y] = new_scales[which][blk];
#pragma unroll
          for (int i = 0; i < NB / W; ++i)
            t.c[h][y * (NB / W) + i] = new_codes[which][blk][NB >= 4 ? i : NB == 2 ? (g & 1) * 2 + i : g];
        }
      }
  };
  int least = lim;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) least = min(least, __shfl_xor(least, o, 64));
  const float scale = 1.44269504088896341f / a.scale;  // scores in powers of two
  // (finite, or −inf + slack would be NaN and the maximum never move: past 6·10^37 of a.scale)
  const float slack = fminf(kSlack * 0.69314718055994531f * a.scale, 3.402823466e38f);
  floatx4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, ref = 0.f, l = 0.f;  // m: of q·k; ref: m·scale + lift, finite; l: of this lane's keys
  int lift = 0;                             // above 0 once a large value of V has come by
  unsigned nan_blocks = 0;                  // blocks of the output that a NaN block of V reached
  char* mine = lds + w * kWaveLds;
  __syncthreads();

  for (; j < k1; j += kSpan) {
    if (adds && j + kKeys >= work.len) {
      take_new(k, 0, j);
      take_new(v, 1, j);
    }
    unsigned worst = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) worst = max(worst, max<unsigned>(k.e[0][i], k.e[1][i]));
    const bool nan = __ballot(worst == kScaleNaN) != 0;
    unsigned k_nan[2] = {0, 0};
    if (nan) {
#pragma unroll
      for (int t = 0; t < 2; ++t) k_nan[t] = take_nan<NB>(k, t, nullptr);
    }
    // S = K·Qᵀ: this lane's are keys 4g … 4g+3 of both subtiles with its query
    float x[8];
    {
      floatx4 acc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
      constexpr int F = NB < 2 || (NP == 3 && NB == 4) ? 1 : 2;  // (2 would spill there)
#pragma unroll
      for (int i0 = 0; i0 < NB; i0 += F) {
        bf8 q[NP][F];
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int f = 0; f < F; ++f) q[p][f] = qs[p][i0 + f][lane];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < F; ++f) {
          const int i = i0 + f;
          const bf8 k0v = convert8(k.c[0][i], tile_scale(k.e[0][W == 2 ? i / 4 : 0]));
          const bf8 k1v = convert8(k.c[1][i], tile_scale(k.e[1][W == 2 ? i / 4 : 0]));
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0v, q[p][f], acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1v, q[p][f], acc[1], 0, 0, 0);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = acc[i / 4][i % 4];
    }
    worst = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) worst = max(worst, max<unsigned>(v.e[0][i], v.e[1][i]));
    if (__ballot(worst >= kLarge)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        unsigned of[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        take_nan<NB>(v, t, of);
        const int seen = min(max(min(lim, k1 - 1) - (j + 16 * t) + 1, 0), 16);
        const unsigned vis = (1u << seen) - 1u;
#pragma unroll
        for (int i = 0; i < NB; ++i)
          if (of[i] & vis) nan_blocks |= 1u << i;
      }
      if constexpr (kLarge < kScaleNaN) {
        worst = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) worst = max(worst, max<unsigned>(v.e[0][i], v.e[1][i]));
        if (lift == 0 && __ballot(worst >= kLarge)) {
          // p from here on 2^-lift of what it was: Σ p·v of all the row's keys stays in range
          lift = static_cast<int>(kSlack) + 32 - __builtin_clz(work.len);
          ref += static_cast<float>(lift);
          const float f = __builtin_amdgcn_exp2f(-static_cast<float>(lift));
          l *= f;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[d] *= f;
        }
      }
    }
    // V to LDS, a key a row
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int key = 16 * t + col, chunk = g * NB + i;
        *reinterpret_cast<bf8*>(mine + key * kRow + v_pair<NB>(key, chunk >> 1) * 32 + (chunk & 1) * 16) =
            convert8(v.c[t][i], tile_scale(v.e[t][W == 2 ? i / 4 : 0]));
      }
    fetch(j + kSpan);
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
    if (__ballot(top > m + slack)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m, top), rn = mn == -INFINITY ? 0.f : mn * scale + static_cast<float>(lift);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - rn);
      m = mn;
      ref = rn;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    bf8 p[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      const f2 e = {__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale, -ref)),
                    __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], scale, -ref))};
      l += e.x;
      l += e.y;
      bf2 part[NP];
      split_bf16<NP>(e, part);
#pragma unroll
      for (int c = 0; c < NP; ++c) p[c][i] = part[c].x, p[c][i + 1] = part[c].y;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (LDS of this wave alone, in order)
    // O += Vᵀ·Pᵀ: four keys of either subtile and 16 dims a transposing read; reads of four steps
    // at once, so that the wave waits for LDS once for them (1–3 % of a call)
    constexpr int F = DT < 4 ? DT : 4;
#pragma unroll
    for (int d0 = 0; d0 < DT; d0 += F) {
      bf8 vv[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const int key = 4 * g + col / 4;  // (and 16 on: the same pair)
        const char* at = mine + key * kRow + v_pair<NB>(key, d0 + f) * 32 + (col % 4) * 8;
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * kRow));
        vv[f] = __builtin_bit_cast(bf8, s8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < NP; ++c)
#pragma unroll
        for (int f = 0; f < F; ++f)
          o[d0 + f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv[f], p[c], o[d0 + f], 0, 0, 0);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }

  // The waves' parts: o[d] holds dims 16d + 4g … + 3 of this lane's query.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) sm[w][col] = m == -INFINITY ? m : ref, sl[w][col] = l;
  const int rows = min(16, R - tile * 16);
  if (col < rows) {
    float* part = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (nan_blocks >> (d / 2) & 1u) o[d] = floatx4{1.f, 1.f, 1.f, 1.f} * __builtin_nanf("");
      *reinterpret_cast<floatx4*>(part + col * D + 16 * d + 4 * g) = o[d];
    }
  }
  __syncthreads();
  // Output value d of row c of the tile.
  auto finish = [&](int c, int d, float lt, float ot) {
    const int rr = tile * 16 + c, ss = token(rr);
    T* out = static_cast<T*>(a.out) + ((static_cast<size_t>(work.b) * a.S + ss) * a.H + head(rr)) * a.dk;
    if (ss < work.n && d < a.dk) out[d] = static_cast<T>(work.len - work.n + ss < 0 ? 0.f : ot / lt);
  };
  const int slot_rows = min(16, R);
  const size_t parts = a.slots;  // pieces that ws has room for
  float* ml = reinterpret_cast<float*>(static_cast<char*>(a.ws) + sizeof(unsigned) * kCounters * kCounterStep);
  float* po = ml + parts * slot_rows * 2;
  for (int i = 2 * threadIdx.x; i < rows * D; i += 2 * kThreads) {
    const int c = i / D, d = i % D;
    float mm = sm[0][c];
#pragma unroll
    for (int y = 1; y < NW; ++y) mm = fmaxf(mm, sm[y][c]);
    const float rf = mm == -INFINITY ? 0.f : mm;
    float lt = 0.f;
    f2 ot = {0.f, 0.f};
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float f = __builtin_amdgcn_exp2f(sm[y][c] - rf);  // (−inf: 0)
      const f2 p = *reinterpret_cast<const f2*>(lds + y * kWaveLds + 4 * i);
      lt += sl[y][c] * f;
      ot += p * f;
    }
    if (work.pieces == 1) {
      finish(c, d, lt, ot.x);
      finish(c, d + 1, lt, ot.y);
    } else {
      const size_t slot = static_cast<size_t>(work.slot + work.piece) * slot_rows;
      if (d == 0) put2(ml + (slot + c) * 2, f2{mm, lt});
      put2(po + slot * D + i, ot);
    }
  }
  if (work.pieces == 1) return;

  // The last of a tile's workgroups to arrive merges its pieces, in their order.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  unsigned* counter = static_cast<unsigned*>(a.ws) + static_cast<size_t>(work.slot) * kCounterStep;
  if (threadIdx.x == 0)
    arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (arrived + 1 != static_cast<unsigned>(work.pieces)) return;
  if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // four dims of a row a thread, the pieces over as many threads as there are
  constexpr int Q = D / 4, kBatch = 4;
  struct Sum {
    floatx4 o;
    float m, l;
  };
  Sum* sums = reinterpret_cast<Sum*>(lds);
  static_assert(kThreads * sizeof(Sum) <= sizeof(lds), "a sum a thread");
  const int cols = rows * Q, ways = cols >= kThreads ? 1 : kThreads / cols, way = ways == 1 ? 0 : threadIdx.x / cols;
  for (int i = threadIdx.x - way * cols; i < cols; i += kThreads) {
    const int c = i / Q, dq = i % Q;
    Sum t{floatx4{0.f, 0.f, 0.f, 0.f}, -INFINITY, 0.f};
    for (int y = way; y < work.pieces && way < ways; y += kBatch * ways) {
      f2 st[kBatch], p[kBatch][2];
#pragma unroll
      for (int z = 0; z < kBatch; ++z) {  // (every load of a batch before the first use)
        st[z] = f2{-INFINITY, 0.f};
        p[z][0] = p[z][1] = f2{0.f, 0.f};
        if (y + z * ways < work.pieces) {
          const size_t at = static_cast<size_t>(work.slot + y + z * ways) * slot_rows + c;
          st[z] = get2(ml + 2 * at);
          p[z][0] = get2(po + at * D + 4 * dq);
          p[z][1] = get2(po + at * D + 4 * dq + 2);
        }
      }
      float mn = t.m;
#pragma unroll
      for (int z = 0; z < kBatch; ++z) mn = fmaxf(mn, st[z].x);
      const float rf = mn == -INFINITY ? 0.f : mn, f0 = __builtin_amdgcn_exp2f(t.m - rf);
      t.m = mn;
      t.l *= f0;
      t.o *= f0;
#pragma unroll
      for (int z = 0; z < kBatch; ++z) {
        const float f = __builtin_amdgcn_exp2f(st[z].x - rf);
        t.l += st[z].y * f;
        t.o += floatx4{p[z][0].x, p[z][0].y, p[z][1].x, p[z][1].y} * f;
      }
    }
    if (ways > 1) {
      sums[threadIdx.x] = t;
      __syncthreads();
      if (way == 0)
        for (int y = 1; y < ways; ++y) {
          const Sum v = sums[y * cols + i];
          const float mn = fmaxf(t.m, v.m), rf = mn == -INFINITY ? 0.f : mn;
          const float f0 = __builtin_amdgcn_exp2f(t.m - rf), f1 = __builtin_amdgcn_exp2f(v.m - rf);
          t.m = mn;
          t.l = t.l * f0 + v.l * f1;
          t.o = t.o * f0 + v.o * f1;
        }
    }
    if (way == 0)
#pragma unroll
      for (int x = 0; x < 4; ++x) finish(c, 4 * dq + x, t.l, t.o[x]);
  }
}

unsigned quads(const Items& n) { return static_cast<unsigned>((4LL * n.count + kEach * kWriters - 1) / (kEach * kWriters)); }

template <typename T>
int write_launch(const Kv4WriteArgs& a, hipStream_t st) {
  const Items n = items_of(a.S, a.H, a.dk);
  const dim3 grid(quads(n), a.B, 2);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v);
  const bool vec = (bits & 15) == 0 && ((a.dk | a.stride_b | a.stride_h | a.stride_s) & 7) == 0;
  if (vec) kv4_write_kernel<T, true><<<grid, kWriters, 0, st>>>(a, n);
  else kv4_write_kernel<T, false><<<grid, kWriters, 0, st>>>(a, n);
  NML_LAUNCHED();
  return 0;
}

template <typename T>
int read_launch(const Kv4ReadArgs& a, hipStream_t st) {
  const Items n = items_of(a.S, a.H, a.dk);
  const dim3 grid(quads(n), a.B, 2);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.k_out) | reinterpret_cast<uintptr_t>(a.v_out);
  if ((bits & 15) == 0 && (a.dk & 7) == 0) kv4_read_kernel<T, true><<<grid, kWriters, 0, st>>>(a, n);
  else kv4_read_kernel<T, false><<<grid, kWriters, 0, st>>>(a, n);
  NML_LAUNCHED();
  return 0;
}

// Waves of a workgroup; most pieces of one tile, and in all those of tiles in pieces that there
// can be.
struct Pieces {
  int waves;
  long long tiles, most, slots;
};
Pieces attention_pieces(int B, int H, int Hkv, int S, int P, int dk) {
  Pieces p;
  const int nb = (dk + kBlock - 1) / kBlock;
  p.tiles = (static_cast<long long>(H / Hkv) * S + 15) / 16 * Hkv * B;
  p.waves = p.tiles >= kManyTiles * capacity(nb, 8) ? few_waves(nb) : 8;
  const int span = p.waves * kKeys, spans = (P - 1) / span + 1;
  p.most = (spans - 1) / least_spans(nb, p.waves) + 1;
  p.slots = p.most == 1 ? 0 : std::min(p.tiles * p.most, 2LL * room_for(p.tiles, capacity(nb, p.waves)));
  return p;
}

template <typename T, int NB, int NW>
int attention_launch_nw(const Kv4AttnArgs& a, const Pieces& p, hipStream_t st) {
  // every tile's workgroup, and those that pieces add
  const unsigned grid = static_cast<unsigned>(std::min(p.tiles + p.slots, p.tiles * p.most));
  if (a.new_k) kv4_attention_kernel<T, NB, NW, true><<<grid, 64 * NW, 0, st>>>(a);
  else kv4_attention_kernel<T, NB, NW, false><<<grid, 64 * NW, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

template <typename T, int NB>
int attention_launch_nb(Kv4AttnArgs a, hipStream_t st) {
  const Pieces p = attention_pieces(a.B, a.H, a.Hkv, a.S, a.P, a.dk);
  a.slots = static_cast<int>(p.slots);
  if (p.waves == 8) return attention_launch_nw<T, NB, 8>(a, p, st);
  return attention_launch_nw<T, NB, few_waves(NB)>(a, p, st);
}

template <typename T>
int attention_launch(const Kv4AttnArgs& a, hipStream_t st) {
  const int nb = (a.dk + kBlock - 1) / kBlock;
  if (nb == 1) return attention_launch_nb<T, 1>(a, st);
  if (nb == 2) return attention_launch_nb<T, 2>(a, st);
  if (nb <= 4) return attention_launch_nb<T, 4>(a, st);
  return attention_launch_nb<T, 8>(a, st);
}

}  // namespace

int launch_kv4_write(int dt, const Kv4WriteArgs& a, hipStream_t st) {
  return dt == F16 ? write_launch<half_t>(a, st) : write_launch<float>(a, st);
}

int launch_kv4_read(int dt, const Kv4ReadArgs& a, hipStream_t st) {
  return dt == F16 ? read_launch<half_t>(a, st) : read_launch<float>(a, st);
}

size_t kv4_attention_workspace(int B, int H, int Hkv, int S, int P, int dk) {
  const Pieces p = attention_pieces(B, H, Hkv, S, P, dk);
  if (p.slots == 0) return 0;
  const long long R = static_cast<long long>(H / Hkv) * S, nb = (dk + kBlock - 1) / kBlock;
  const long long d = kBlock * (nb <= 2 ? nb : nb <= 4 ? 4 : 8);
  return sizeof(unsigned) * kCounters * kCounterStep + sizeof(float) * p.slots * std::min<long long>(16, R) * (2 + d);
}

int launch_kv4_attention(int dt, const Kv4AttnArgs& a, hipStream_t st) {
  return dt == F16 ? attention_launch<half_t>(a, st) : attention_launch<float>(a, st);
}

}  // namespace nml
