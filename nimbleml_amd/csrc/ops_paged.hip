// A KV cache in pages: written, and attended to by a row's newest tokens.
//
// The cache is two pools, (pages, kv_heads, page, dk): a page holds `page` (a power of two) positions
// of one row, a head's positions in a run. Row b's position p is position p % page of page
// table[b·max_pages + p / page].
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "paged.hpp"

namespace nml {

namespace {

typedef unsigned u4 __attribute__((ext_vector_type(4)));

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

// A writing workgroup, and the units that a lane of it takes, their loads in flight together. With inputs that change
// from call to call: 4 × 4096 tokens of 16 heads of 128 float16 values, 55.7 µs with two, 4.8 TB/s of reads and
// writes; 59.7 with one, 60.1 with four, 172 with eight; stored past the caches, which a prompt's keys leave again before
// they are read: 59 with stores that stay there. One token of 32 rows, 16 heads of 64: 3.0 with its launch.
constexpr int kWriters = 256, kEach = 2;

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
    if (here[k]) __builtin_nontemporal_store(x[k], pages + to[k]);
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
//
// The queries that share a KV head, its group's heads times the new tokens, are the columns of 16-wide
// MFMA tiles, the heads of a token side by side: S = K·Qᵀ takes 16 keys as its rows, straight from
// the registers that the keys were loaded into, O = Vᵀ·Pᵀ takes the probabilities from the lanes where S
// left them. float16: v_mfma_f32_16x16x32_f16, V transposed by the reads of LDS that each wave
// passes it through; a probability enters the product as two float16 parts (22 bits; Σ p is of the
// whole one). float32: v_mfma_f32_16x16x4f32, whose operand a lane's values of V are as loaded.
//
// A wave goes through tiles of 32 (float16) or 16 keys on its own: its loads of the next tile, and of
// the page numbers of the one after, are in flight during this one. The running maximum that the
// exponentials refer to moves only when a score passes it by 2^8, which skips the rescaling of O on
// nearly every tile. A workgroup's waves merge in LDS.
//
// A (row, KV head, 16 queries) is one workgroup's unless its keys are many: pieces of a long one go to
// several, as many in all as the card holds at once, and the last to finish merges them in their
// order.
//
// Bound by HBM where keys are many: 16 rows of 1 to 8 Ki keys, 32 heads over 8 of 128, float16, 66 µs,
// 4.6 TB/s of keys and values (a copy 4.8). Where few, by a chain of dependent steps: lengths, page
// numbers, keys, rounds, merge and the pieces' merge: one row of 1023 keys, 16 heads of 64, 9.0 µs; 16
// rows of up to 2048 and up to 5 tokens, 8 heads of 32, float32, 14.0. (Where work is cut finely enough the
// merge is what is left: its loads are in batches of 16 pieces, of four where there are no more.) Below, where
// changing inputs are not mentioned, both sides of a choice were timed over one set.

typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kSlack = 8.f;  // in powers of two
constexpr float kScaleLog = 1.44269504088896341f;

template <typename T>
constexpr int tile_keys() {
  return sizeof(T) == 2 ? 32 : 16;
}
// float16 probabilities times 2^7: at most 2^15, and with all their bits down to 2^-21 of the largest.
template <typename T>
constexpr float up_log2() {
  return sizeof(T) == 2 ? 7.f : 0.f;
}

// Head dims in steps of 32: 1, 2, 4 or 8 of them.
constexpr int steps_of(int dk) { return dk <= 32 ? 1 : dk <= 64 ? 2 : dk <= 128 ? 4 : 8; }
// Waves of a workgroup. Few begin and merge sooner, and more workgroups even out rows of different length; at a head dim
// of 64 two, else four. (µs, with inputs that change from call to call: 16 rows of 1 to 8 Ki keys, 32 heads over 8 of 128, 66
// with four and 76 with eight; of 64, 43 with two and 41 with four, one row of 1023, 16 heads of 64, 9.9 and 11.5,
// 128 rows of 100 to 1000 64.6 and 66.0; the same three of 32 24.2 and 21.2, 8.9 and 10.1, 33 and 35, and 16 rows of up
// to 2048 and five tokens, 8 heads of 32, float32, 18.6 and 15.5.)
__host__ __device__ constexpr int group_waves(int nb) { return nb == 2 ? 2 : 4; }
// Waves a SIMD that the registers are held to (at head dim 256 a wave's tile takes more than half of them: 16
// rows of 1 to 4 Ki keys, 16 heads over 2, float16 33 µs and float32 47; held to two waves 38 and 68, with
// spills), and the workgroups that the card's CUs then hold at once.
__host__ __device__ constexpr int waves_of(int nb) { return nb <= 2 ? 4 : nb == 8 ? 1 : 2; }
constexpr int kCus = 256;
__host__ __device__ constexpr int capacity(int nb) { return kCus * 4 * waves_of(nb) / group_waves(nb); }
// Pieces that few tiles are cut into, and one more for each of them at most: a wave for each SIMD.
__host__ __device__ constexpr int even_pieces(int waves) { return kCus * 4 / waves; }
// Spans (a tile for each wave) that a piece has at least: what it costs to begin one and to merge it. (One row
// of 1023 keys, 16 heads of 64: 9.2 µs at two spans of 64 keys, 10.6 at four, 8.9 at one; of 100 keys 6.9, 6.9, 8.7.)
__host__ __device__ constexpr int least_spans(int nb) { return nb == 2 ? 2 : 1; }
// Pieces that a thread of a merge takes its four values of in the time of a round (16000 keys, 16 heads over one
// of 128: 26 µs, 27 at eight, 65 with a piece for each span and batches of four; 8000 keys, 32 heads over 4 of
// 64: 14.0, 13.4, 17.7).
constexpr float kMerged = 16.f;

// ws: a counter for each tile in pieces, then for each piece its rows' references and Σ p, then their
// Σ p·v. Tiles in pieces are fewer than the card's workgroups (a piece is at least their even share),
// and so their pieces fewer than twice as many.

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
  __device__ __forceinline__ bool load(const PagedAttnArgs& a, int b) {
    const int at = min(b, a.B - 1), x = a.lens[at], y = a.counts ? a.counts[at] : a.S;
    len = min(max(x, 0), a.max_pages << a.shift);
    n = min(max(y, 0), a.S);
    spans = b >= a.B ? 0 : n > 0 ? max(1, (len + SPAN - 1) / SPAN) : 1;
    return x == len && y == n;  // (were in range)
  }
};

// What this workgroup does: piece `piece` of `pieces` of tile (b, hk, tile), whose row has len keys and n
// new tokens; `slot`: where the tile's first piece is in ws. b < 0: nothing.
struct Work {
  int b, hk, tile, piece, pieces, slot, len, n, spans;
};
// More than 64 rows are shared out to the waves, a run of rows each; sums: of the waves.
template <int SPAN, int NW>
__device__ __forceinline__ Work find_work(const PagedAttnArgs& a, int tiles, int cap, int fewest, float merge, int lane, int wave, int (*sums)[3]) {
  Work w{};
  Rows<SPAN> rows;
  const int each = a.Hkv * tiles;
  const int run = a.B <= 64 ? 64 : (a.B + 64 * NW - 1) / (64 * NW) * 64;
  const int first = a.B <= 64 ? 0 : wave * run, end = min(first + run, a.B);
  int total = 0;
  bool good = true;
#pragma unroll 2
  for (int i = first; i < end; i += 64) {
    good &= rows.load(a, i + lane);
    total += rows.spans;
  }
  if (!good && blockIdx.x == 0) tell(a.err);
  total = __builtin_amdgcn_readlane(wave_scan(total), 63);
  if (a.B > 64) {
    if (lane == 0) sums[wave][0] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) total += sums[i][0];
  }
  const int room = room_for(static_cast<long long>(each) * a.B, cap);
  int least = max(fewest, static_cast<int>((static_cast<long long>(total) * each + room - 1) / room));
  // What a piece takes of the merge, `merge` of a round, against its own rounds: s spans to a piece, s² = merge ·
  // the row's in the mean.
  const float mean = static_cast<float>(total) * __builtin_amdgcn_rcpf(static_cast<float>(a.B));
  least = max(least, static_cast<int>(__builtin_ceilf(__builtin_amdgcn_sqrtf(mean * merge))));
  // Few tiles, which pieces of any size leave even: a wave for each SIMD, beside which a second one adds
  // pieces to merge but no bandwidth (30000 keys, 32 heads over 8 of 128: 29.5 µs, 33.5 with two). More tiles, of
  // different length, are evener in more pieces (16 rows of 1 to 8 Ki: 55, 73 with one).
  constexpr int even = even_pieces(NW);
  if (static_cast<long long>(each) * a.B <= even / 4)
    least = max(least, static_cast<int>((static_cast<long long>(total) * each + even - 1) / even));
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
    rows.load(a, i + lane);
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
      // A KV head's piece is of all of its tiles: they are 8 workgroups apart, on one XCD, whose L2 has its
      // keys for them (five tokens over 30000 keys, two tiles: 52 µs, 58 with a tile's pieces side by side).
      int both = local;
      w.tile = 0;
      if (tiles > 1) {
        const int heads = a.Hkv * w.pieces, turn = local / (8 * tiles), in = local - turn * (8 * tiles);
        const int width = min(8, heads - 8 * turn);
        w.tile = width == 8 ? in >> 3 : in / width;
        both = 8 * turn + in - w.tile * width;
      }
      w.hk = w.pieces == 1 ? both : both / w.pieces;
      w.piece = both - w.hk * w.pieces;
      w.slot = (slots + __builtin_amdgcn_readlane(sum_slots, l) - w.pieces) * each + (w.hk * tiles + w.tile) * w.pieces;
      return w;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(sum_slots, 63);
  }
  w.b = -1;
  return w;
}

// Values k … of a vector of 8 or 16 bytes, zeros behind them.
template <typename V>
__device__ __forceinline__ V past(V v, int k) {
  constexpr int N = sizeof(v) / 4, E = sizeof(v[0]);
  typedef unsigned words __attribute__((ext_vector_type(N)));
  words w = __builtin_bit_cast(words, v);
  const int bytes = k * E;
  if (N == 4 && bytes & 8) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = i + 2 < N ? w[(i + 2) % N] : 0u;
  }
  if (bytes & 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = i + 1 < N ? w[(i + 1) % N] : 0u;
  }
  if (E == 2 && bytes & 2) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = w[i] >> 16 | (i + 1 < N ? w[(i + 1) % N] << 16 : 0u);
  }
  return __builtin_bit_cast(V, w);
}

// N values from d0 on of a vector of dk, zeros past its end. VEC: one aligned load (dk and the vectors' places
// are multiples of N values, so that all are in or out). Else one load that starts at any value, of the
// last N values where fewer are left, and a shift by those before d0 (8 rows of 1 to 4 Ki keys, 32 heads over
// 8 of 100, float16, 49 µs; value by value 114).
template <typename T, int N, bool VEC>
__device__ __forceinline__ auto load_values(const T* p, int d0, int dk) {
  typedef T vec __attribute__((ext_vector_type(N), aligned(N * sizeof(T))));
  typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  vec r;
#pragma unroll
  for (int i = 0; i < N; ++i) r[i] = static_cast<T>(0.f);
  if (VEC) {
    if (d0 < dk) r = *reinterpret_cast<const vec*>(p + d0);
  } else if (dk >= N) {
    if (d0 < dk) {
      const int at = min(d0, dk - N);
      r = *reinterpret_cast<const loose*>(p + at);
      r = past(r, d0 - at);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (d0 + i < dk) r[i] = p[d0 + i];
  }
  return r;
}

// float16: what a lane (col = lane % 16, g = lane / 16) holds of a tile: of keys col and 16 + col, values
// 32i + 8g … + 7 of step i, of K and V alike. V goes through LDS, a key a row, its 32-byte pairs
// exchanged by the key so that the 16 rows that a transposing read takes 32 bytes each of lie in
// different banks. Output tile t: dims 16t + 4g + r in register r.
template <typename T, int NB, bool VEC>
struct Tile {
  static constexpr int kTiles = 2 * NB;  // 16-wide tiles of the head dim
  static constexpr int kRow = 64 * NB;   // bytes of a key's values in LDS
  static constexpr int kQ = NB;          // 16-byte pieces of a query a lane
  half8 k[2][NB], v[2][NB];
  static __device__ __forceinline__ int q_dim(int i, int g) { return 32 * i + 8 * g; }
  static __device__ __forceinline__ int out_dim(int t, int r, int g) { return 16 * t + 4 * g + r; }
  static __device__ __forceinline__ int id_key(int i, int lane) { return 16 * i + (lane & 15); }
  static __device__ __forceinline__ void load(half8 (*x)[NB], const half_t* p, const size_t* at, int dk, int g) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NB; ++i) x[s][i] = load_values<half_t, 8, VEC>(p + at[s] * dk, q_dim(i, g), dk);
  }
  __device__ __forceinline__ void load_k(const half_t* p, const size_t* at, int dk, int g, int) { load(k, p, at, dk, g); }
  __device__ __forceinline__ void load_v(const half_t* p, const size_t* at, int dk, int g, int) { load(v, p, at, dk, g); }
  // x[4s + r]: the score of key 16s + 4g + r with this lane's query
  __device__ __forceinline__ void scores(const half8 (*qs)[64], float* x, int lane) const {
    floatx4 acc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const half8 q = qs[i][lane];
#pragma unroll
      for (int s = 0; s < 2; ++s) acc[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s][i], q, acc[s], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = acc[i / 4][i % 4];
  }
  static __device__ __forceinline__ int pair_of(int key, int pair) {
    return pair ^ (NB >= 4 ? key & 7 : NB == 2 ? key >> 1 & 3 : key >> 2 & 1);
  }
  __device__ __forceinline__ void stage(char* lds, int lane) const {
    const int col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const int key = 16 * s + col, chunk = 4 * i + g;
        *reinterpret_cast<half8*>(lds + key * kRow + pair_of(key, chunk >> 1) * 32 + (chunk & 1) * 16) = v[s][i];
      }
  }
  // O += Vᵀ·Pᵀ, p[i] the probability of x[i]'s key
  static __device__ __forceinline__ void add(const char* lds, const float* p, floatx4* o, int lane) {
    const int col = lane & 15, g = lane >> 4;
    half8 part[2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[0][i] = static_cast<half_t>(p[i]);
      part[1][i] = static_cast<half_t>(p[i] - static_cast<float>(part[0][i]));
    }
    constexpr int F = kTiles < 4 ? kTiles : 4;
#pragma unroll
    for (int d0 = 0; d0 < kTiles; d0 += F) {
      half8 vv[F];
#pragma unroll
      for (int f = 0; f < F; ++f) {
        typedef __attribute__((address_space(3))) s4 lds_s4;
        typedef short s8 __attribute__((ext_vector_type(8)));
        const int key = 4 * g + col / 4;  // (and 16 on: the same pair)
        const char* at = lds + key * kRow + pair_of(key, d0 + f) * 32 + (col % 4) * 8;
        const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)at);
        const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + 16 * kRow));
        vv[f] = __builtin_bit_cast(half8, s8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int f = 0; f < F; ++f)
          o[d0 + f] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv[f], part[c], o[d0 + f], 0, 0, 0);
    }
  }
};

// float32: of key col, values 16i + 4g … + 3 of K; of keys 4g + r, W values from W·(16j + col) on of V. Output
// tile t = W·j + e: dims W·(16j + 4g + r) + e in register r.
template <int NB, bool VEC>
struct Tile<float, NB, VEC> {
  static constexpr int kTiles = 2 * NB, kQ = 2 * NB;
  static constexpr int kRow = 0;
  static constexpr int W = NB == 1 ? 2 : 4, J = kTiles / W;
  typedef float vec __attribute__((ext_vector_type(W)));
  floatx4 k[2 * NB];
  vec v[4][J];
  static __device__ __forceinline__ int q_dim(int i, int g) { return 16 * i + 4 * g; }
  static __device__ __forceinline__ int out_dim(int t, int r, int g) { return W * (16 * (t / W) + 4 * g + r) + t % W; }
  static __device__ __forceinline__ int id_key(int i, int lane) { return i == 0 ? lane & 15 : 4 * (lane >> 4); }
  __device__ __forceinline__ void load_k(const float* p, const size_t* at, int dk, int g, int) {
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) k[i] = load_values<float, 4, VEC>(p + at[0] * dk, q_dim(i, g), dk);
  }
  __device__ __forceinline__ void load_v(const float* p, const size_t* at, int dk, int, int col) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j) v[r][j] = load_values<float, W, VEC>(p + at[1 + r] * dk, W * (16 * j + col), dk);
  }
  __device__ __forceinline__ void scores(const floatx4 (*qs)[64], float* x, int lane) const {
    floatx4 acc[4];  // (four chains of sums, each a quarter as long: outputs of 604 keys of 64 4.5e-7 off, with two 6.2e-7)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      const floatx4 q = qs[i][lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[i][e], q[e], acc[e], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (acc[0][i] + acc[1][i]) + (acc[2][i] + acc[3][i]);
  }
  __device__ __forceinline__ void stage(char*, int) const {}
  __device__ __forceinline__ void add(const char*, const float* p, floatx4* o, int) const {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < W; ++e)
          o[W * j + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[r][j][e], p[r], o[W * j + e], 0, 0, 0);
  }
};

template <typename T, int NB, bool VEC>
__global__ __launch_bounds__(64 * group_waves(NB), waves_of(NB)) void paged_attention_kernel(PagedAttnArgs a) {
  typedef Tile<T, NB, VEC> Keys;
  constexpr int NW = group_waves(NB);
  constexpr int KT = tile_keys<T>(), KX = KT / 4, DT = Keys::kTiles;
  constexpr int D = 32 * NB, kWaveLds = 64 * D;  // 16 rows of D floats; a tile of V takes as much
  constexpr int kThreads = 64 * NW, kSpan = NW * KT, kIds = 2;
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int QN = 16 / sizeof(T);
  static_assert(Keys::kRow * KT <= kWaveLds, "a tile of V");
  typedef T qvec __attribute__((ext_vector_type(QN)));
  __shared__ __align__(16) char lds[NW * kWaveLds];
  __shared__ __align__(16) qvec qs[Keys::kQ][64];
  __shared__ float sm[NW][16], sl[NW][16];
  __shared__ unsigned arrived;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, g = lane >> 4;
  const int R = a.group * a.S, tiles = (R + 15) / 16;
  const float merge = static_cast<float>(min(16, R)) * (D / (4.f * kThreads * kMerged));
  const Work work = find_work<kSpan, NW>(a, tiles, capacity(NB), least_spans(NB), merge, lane, w, reinterpret_cast<int(*)[3]>(lds));
  // (Tiles of padding alone: all of a tile's workgroups leave here, so that its counter stays zero. 16 rows of 1 or 2
  // tokens of up to 100 over 3000 keys, 8 heads of 64, float32, six tiles of seven: 162 µs and 91; where every second
  // tile is such, which then reads what the other has brought to the L2, no less.)
  if (work.b < 0 || work.tile * 16 >= work.n * a.group) return;
  const int hk = work.hk, tile = work.tile;
  const int per = work.pieces == 1 ? work.spans : (work.spans + work.pieces - 1) / work.pieces;

  // The query of column c of this tile: row r of the KV head's R, token r / group of head hk·group +
  // r % group. It sees keys up to lim; a column without a query (or of the padding) runs along with
  // zeros.
  auto token = [&](int r) { return a.group == 1 ? r : r / a.group; };
  auto head = [&](int r) { return hk * a.group + (a.group == 1 ? 0 : r % a.group); };
  const int r = tile * 16 + col, s = token(r);
  const bool live = r < R && s < work.n;
  const int lim = live ? work.len - work.n + s : 0x7fffffff;
  // keys that a query of the tile sees
  const int seen = max(0, min(work.len, work.len - work.n + min(token(min(tile * 16 + 15, R - 1)), work.n - 1) + 1));
  const int k0 = work.piece * per * kSpan, k1 = min(seen, k0 + per * kSpan);

  const RowPages pages{a.table + static_cast<size_t>(work.b) * a.max_pages, a.shift, a.num_pages, a.Hkv, hk};
  const T *kp = static_cast<const T*>(a.k_pages), *vp = static_cast<const T*>(a.v_pages);
  // A tile of keys from `at` on. Past the piece's end: its first one again and again, so that every
  // round issues as many loads (the waits before their use count them). Past the last key: that one.
  bool bad = false;
  int ids[kIds];
  auto key_at = [&](int at, int i) { return min((at < k1 ? at : k0) + i, work.len - 1); };
  auto fetch_ids = [&](int at) {
#pragma unroll
    for (int i = 0; i < kIds; ++i) ids[i] = pages.number(key_at(at, Keys::id_key(i, lane)));
  };
  Keys t;
  size_t place[kHalf ? 2 : 5];
  auto find = [&](int at) {
    if constexpr (kHalf) {
#pragma unroll
      for (int i = 0; i < 2; ++i) place[i] = pages.place(key_at(at, Keys::id_key(i, lane)), ids[i], bad);
    } else {
      place[0] = pages.place(key_at(at, Keys::id_key(0, lane)), ids[0], bad);
#pragma unroll
      for (int i = 0; i < 4; ++i)  // (four keys of one page, or the last key for those past it)
        place[1 + i] = pages.place(key_at(at, Keys::id_key(1, lane) + i), ids[1], bad);
    }
  };
  // (an element's bounds tests are formed where they are used: kept, they take a pair of registers each)
  auto fetch_k = [&] {
    int gg = g;
    if (!VEC) asm volatile("" : "+v"(gg));
    t.load_k(kp, place, a.dk, gg, col);
  };
  auto fetch_v = [&] {
    int gg = g, cc = col;
    if (!VEC) asm volatile("" : "+v"(gg), "+v"(cc));
    t.load_v(vp, place, a.dk, gg, cc);
  };
  int j = k0 + w * KT;
  if (k0 < k1) {
    fetch_ids(j);
    find(j);
    fetch_k();
    fetch_v();
    fetch_ids(j + kSpan);
  }

  // Q into LDS, 16 bytes a lane and piece, in the order of the products' steps
#pragma unroll
  for (int i0 = 0; i0 < Keys::kQ; i0 += NW) {
    const int i = i0 + w;
    if (i < Keys::kQ) {
      qvec q;
#pragma unroll
      for (int e = 0; e < QN; ++e) q[e] = static_cast<T>(0.f);
      if (live) {
        const T* qp = static_cast<const T*>(a.q) + ((static_cast<size_t>(work.b) * a.H + head(r)) * a.S + s) * a.dk;
        q = load_values<T, QN, VEC>(qp, Keys::q_dim(i, g), a.dk);
      }
      qs[i][lane] = q;
    }
  }
  int least = lim;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) least = min(least, __shfl_xor(least, o, 64));
  const float scale = kScaleLog / a.scale;  // scores in powers of two
  // (finite, or −inf + slack would be NaN and the maximum never move)
  const float slack = fminf(kSlack * 0.69314718055994531f * a.scale, 3.402823466e38f);
  floatx4 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, ref = 0.f, l = 0.f;  // m: of q·k; ref: m·scale less the factor of p, finite; l: of this lane's keys
  char* mine = lds + w * kWaveLds;
  __syncthreads();

  for (; j < k1; j += kSpan) {
    float x[KX];
    t.scores(qs, x, lane);
    t.stage(mine, lane);
    find(j + kSpan);
    fetch_ids(j + 2 * kSpan);
    fetch_k();
    if constexpr (kHalf) fetch_v();
    if (j + KT - 1 > least || j + KT > work.len) {
#pragma unroll
      for (int i = 0; i < KX; ++i) {
        const int key = j + 16 * (i / 4) + 4 * g + i % 4;
        if (key > lim || key >= work.len) x[i] = -INFINITY;
      }
    }
    float top = x[0];
#pragma unroll
    for (int i = 1; i < KX; ++i) top = fmaxf(top, x[i]);
    if (__ballot(top > m + slack)) {
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float mn = fmaxf(m, top), rn = mn == -INFINITY ? 0.f : mn * scale - up_log2<T>();
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - rn);
      m = mn;
      ref = rn;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    float p[KX];
#pragma unroll
    for (int i = 0; i < KX; ++i) {
      p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], scale, -ref));
      l += p[i];
    }
    if constexpr (kHalf) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (LDS of this wave alone, in order)
    t.add(mine, p, o, lane);
    if constexpr (kHalf) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    else fetch_v();
  }
  if (__ballot(bad) && lane == 0) tell(a.err);

  // An infinite or NaN value makes 0·∞ of keys that a query does not see and ∞ − ∞ of a
  // probability's second part, and sums of values near float32's largest pass its range: outputs
  // that are not finite are formed again, key by key, keys without weight left out, of
  // probabilities 2^-lift as large.
  bool wrong = false;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) wrong |= !__builtin_isfinite(o[d][i]);
  if (__ballot(wrong && live)) {
    const float lift = sizeof(T) == 2 ? 0.f : kSlack + 32.f - static_cast<float>(__builtin_clz(work.len));
    const float f = __builtin_amdgcn_exp2f(-lift);
    ref += lift;
    l *= f;
    floatx4 fresh[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) fresh[d] = floatx4{0.f, 0.f, 0.f, 0.f};
    for (int j0 = k0 + w * KT; j0 < k1; j0 += kSpan)
      for (int key = j0; key < min(j0 + KT, k1); ++key) {
        const size_t at = pages.place(key, pages.number(key), bad) * a.dk;
        float x = 0.f;
        int gg = g;
        asm volatile("" : "+v"(gg));
#pragma unroll 1
        for (int i = 0; i < Keys::kQ; ++i) {
          const qvec q = qs[i][lane], k = load_values<T, QN, VEC>(kp + at, Keys::q_dim(i, gg), a.dk);
#pragma unroll
          for (int e = 0; e < QN; ++e) x = __builtin_fmaf(static_cast<float>(q[e]), static_cast<float>(k[e]), x);
        }
        x += __shfl_xor(x, 16, 64);
        x += __shfl_xor(x, 32, 64);
        const float p = key > lim ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(x, scale, -ref));
        if (p != 0.f) {
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int dim = Keys::out_dim(d, i, gg);
              if (dim < a.dk) fresh[d][i] = __builtin_fmaf(p, static_cast<float>(vp[at + dim]), fresh[d][i]);
            }
        }
      }
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] = __builtin_isfinite(o[d][i]) ? o[d][i] * f : fresh[d][i];
  }

  // The waves' parts.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (g == 0) sm[w][col] = m == -INFINITY ? m : ref, sl[w][col] = l;
  const int rows = min(16, R - tile * 16);
  if (col < rows) {
    float* part = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[col * D + Keys::out_dim(d, i, g)] = o[d][i];
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
  float* ml = reinterpret_cast<float*>(static_cast<char*>(a.ws) + kCounterBytes);
  float* po = ml + parts * slot_rows * 2;
  // (float32: parts times 2^-4 and 2^-12, whose sums of near the largest values stay finite)
  constexpr float kRoom1 = sizeof(T) == 2 ? 0.f : 4.f, kRoom2 = sizeof(T) == 2 ? 0.f : 12.f;
  for (int i = 2 * threadIdx.x; i < rows * D; i += 2 * kThreads) {
    const int c = i / D, d = i % D;
    float mm = sm[0][c];
#pragma unroll
    for (int y = 1; y < NW; ++y) mm = fmaxf(mm, sm[y][c]);
    const float rf = (mm == -INFINITY ? 0.f : mm) + kRoom1;
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
      if (d == 0) put2(ml + (slot + c) * 2, f2{mm == -INFINITY ? mm : rf, lt});
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
  constexpr int Q = D / 4;
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
    auto add = [&](auto batch) {  // pieces whose loads are in flight together
      constexpr int kBatch = decltype(batch)::value;
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
        for (int z = 0; z < kBatch; ++z) mn = fmaxf(mn, st[z].x + kRoom2);
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
    };
    if (work.pieces > 8 * ways) add(std::integral_constant<int, 16>{});
    else add(std::integral_constant<int, 4>{});
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

// Most pieces of one tile, and in all those of tiles in pieces that there can be.
struct Pieces {
  long long tiles, most, slots;
};
template <typename T>
Pieces attention_pieces(int B, int H, int Hkv, int S, int P, int dk) {
  Pieces p;
  const int nb = steps_of(dk), span = group_waves(nb) * tile_keys<T>(), spans = (P - 1) / span + 1;
  p.tiles = (static_cast<long long>(H / Hkv) * S + 15) / 16 * Hkv * B;
  p.most = (spans - 1) / least_spans(nb) + 1;
  p.slots = p.most == 1 ? 0 : std::min(p.tiles * p.most, 2LL * room_for(p.tiles, capacity(nb)));
  const int even = even_pieces(group_waves(nb));
  if (p.tiles <= even / 4) p.slots = std::min(p.slots, even + p.tiles);
  return p;
}

template <typename T, int NB, bool VEC>
int attention_launch_nb(PagedAttnArgs a, hipStream_t st) {
  const Pieces p = attention_pieces<T>(a.B, a.H, a.Hkv, a.S, a.max_pages << a.shift, a.dk);
  a.slots = static_cast<int>(p.slots);
  // every tile's workgroup, and those that pieces add
  const unsigned grid = static_cast<unsigned>(std::min(p.tiles + p.slots, p.tiles * p.most));
  paged_attention_kernel<T, NB, VEC><<<grid, 64 * group_waves(NB), 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

template <typename T, int NB>
int attention_launch_vec(const PagedAttnArgs& a, hipStream_t st) {
  constexpr int per = 16 / sizeof(T);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_pages) |
                         reinterpret_cast<uintptr_t>(a.v_pages);
  if ((bits & 15) == 0 && a.dk % per == 0) return attention_launch_nb<T, NB, true>(a, st);
  return attention_launch_nb<T, NB, false>(a, st);
}

template <typename T>
int attention_launch(const PagedAttnArgs& a, hipStream_t st) {
  switch (steps_of(a.dk)) {
    case 1: return attention_launch_vec<T, 1>(a, st);
    case 2: return attention_launch_vec<T, 2>(a, st);
    case 4: return attention_launch_vec<T, 4>(a, st);
  }
  return attention_launch_vec<T, 8>(a, st);
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

int paged_attention_span(int dt, int dk) {
  return std::min(64, group_waves(steps_of(dk)) * (dt == F16 ? tile_keys<half_t>() : tile_keys<float>()));
}

size_t paged_attention_workspace(int dt, int B, int H, int Hkv, int S, int P, int dk) {
  // (which kernel takes a call depends on its buffers' alignment too)
  const size_t many = paged_prefill_applies(dt, H, Hkv, S, dk) ? paged_prefill_workspace(dt, B, H, Hkv, S, P, dk) : 0;
  const Pieces p = dt == F16 ? attention_pieces<half_t>(B, H, Hkv, S, P, dk) : attention_pieces<float>(B, H, Hkv, S, P, dk);
  if (p.slots == 0) return many;
  const long long R = static_cast<long long>(H / Hkv) * S, d = 32 * steps_of(dk);
  return std::max<size_t>(many, kCounterBytes + sizeof(float) * p.slots * std::min<long long>(16, R) * (2 + d));
}

int launch_paged_attention(int dt, const PagedAttnArgs& a, hipStream_t st) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_pages) |
                         reinterpret_cast<uintptr_t>(a.v_pages) | reinterpret_cast<uintptr_t>(a.out);
  if ((bits & 15) == 0 && paged_prefill_applies(dt, a.H, a.Hkv, a.S, a.dk)) return launch_paged_prefill(dt, a, st);
  return dt == F16 ? attention_launch<half_t>(a, st) : attention_launch<float>(a, st);
}

}  // namespace nml
