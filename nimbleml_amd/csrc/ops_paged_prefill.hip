// Attention over a paged KV cache for many new tokens: a piece of a prompt behind what the cache
// holds already.
//
// A KV head's queries (its group's heads times the new tokens, the heads of a token side by side) are
// taken 128 at a time by a workgroup of four waves, 32 a wave, over tiles of 64 keys in LDS:
//   Sᵀ = K·Qᵀ    v_mfma_f32_32x32x16_f16, Qᵀ in registers; lane l then holds query l % 32 and keys
//                8(r/4) + 4(l/32) + r % 4 of each 32 in register r;
//   Oᵀ += Vᵀ·Pᵀ  Pᵀ straight from those registers, Vᵀ by transposing reads of V as it lies in memory,
//                in the same order of the keys;
// so that each lane has its own query's maximum, sum and output column. The reference of the
// exponentials moves only when a maximum passes it by 2^8 in p. A probability enters the product with V as
// two float16 values, the nearest one towards zero and what it leaves: at most 2^-20 of it is lost (of
// those below 2^-21 of the largest, 2^-31 of that), and Σ p is of the two, so that an output is off by
// little more than its own rounding to float16. As one float16 value an output would be off as far
// again (2.9·10^-4 of its norm, 2.1·10^-4), for a third fewer matrix instructions: 2048 tokens over 8192 keys,
// 32 heads of 128 over 8, 341 µs and 425 on one box; two rows of them with 16 heads of 64, 244 and 277.
//
// One barrier a tile: K is written to LDS two tiles ahead and V one, from registers that were loaded a
// tile before, and the scores of the next tile are formed beside the probabilities of this one. A
// wave's loads of 16 bytes a lane are of whole rows of one page, whose number is known a tile earlier,
// so that a load's address is a scalar and a fixed offset of the lane.
//
// Where the tiles of queries leave CUs idle the keys are cut into pieces, whose parts a second launch
// merges.
//
// Bound by the matrix pipe, which has three products for the formula's two, and the exponentials beside it. 2048 tokens
// over 8192 keys, 32 heads of 128 over 8, float16: 405 to 440 µs by the box, 594 TFLOP/s of the formula's and 890 on the
// pipe, where a product of 8192³ reaches 1464; two rows of them with 16 heads of 64: 284, 420 and 630 (as many
// exponentials for half the products); 16 over 4 of 256: 722, 330 and 500 (one wave a SIMD, and values moved between
// its two halves of the registers).
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace nml {

namespace {

constexpr int kK = 64;  // keys of a tile
// Waves of a workgroup, and the queries of its tile. (Eight waves, which share what is written to LDS: 1024 tokens over
// 4096 keys, 16 heads over 4 of 96, 76 µs, 71 with four; 6 ragged rows of up to 512 tokens, 12 heads of 80, 64 and 57;
// 2048 over 8192, 32 over 8 of 128, 440 and 439; two rows of them, 16 heads of 64, 324 and 286.)
constexpr int kWaves = 4, kQ = 32 * kWaves;
constexpr float kLog2e = 1.44269504088896341f;
typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));

// Keys a piece has at least, in tiles (2 rows of 100 tokens over up to 1000 keys, 16 heads of 64: 17.7 µs at
// four, 22.4 at eight, 18.2 at one).
constexpr int kLeastTiles = 4;

// Workgroups that the card holds at once, eight waves a CU (columns above 128, which take more than half of
// the registers: four): where the tiles are fewer their keys are cut into pieces. (Pieces for twice as many: 128 tokens
// over 16 Ki keys, 16 heads over 4 of 128, 88 in place of 62 µs, 1024 over 4096, 16 over 4 of 192, 170 in place of 161;
// 2048 over 8192, 16 over 4 of 256, which are 256 tiles whole, 700 in place of 723.)
__host__ __device__ constexpr int held(int DK) { return DK > 128 ? 256 : 512; }

// A row of the batch: its length and new tokens, in range, tiles of queries of a KV head (0: nothing to
// do), tiles of keys. Every lane has one where the rows are gone through 64 at a time.
struct Row {
  int len, n, nq, kt;
  bool good;  // length and count were in range
  static __device__ __forceinline__ Row load(const PagedAttnArgs& a, int b) {
    const int at = min(b, a.B - 1);
    return make(a, a.lens[at], a.counts ? a.counts[at] : a.S, b < a.B);
  }
  // One row for all lanes, in scalars.
  static __device__ __forceinline__ Row one(const PagedAttnArgs& a, int b) {
    const int y = a.counts ? a.counts[b] : a.S;
    return make(a, __builtin_amdgcn_readfirstlane(a.lens[b]), __builtin_amdgcn_readfirstlane(y), true);
  }
  static __device__ __forceinline__ Row make(const PagedAttnArgs& a, int x, int y, bool there) {
    Row r;
    r.len = min(max(x, 0), a.max_pages << a.shift);
    r.n = min(max(y, 0), a.S);
    r.good = r.len == x && r.n == y;
    r.nq = there ? (r.n * a.group + kQ - 1) / kQ : 0;
    r.kt = (r.len + kK - 1) / kK;
    return r;
  }
  // What its queries have to go over, in pairs of tiles: the first of them have fewer keys than the last. (At least
  // half of nq·kt.)
  __device__ __forceinline__ long long work(int group) const {
    const long long keys = max(len - n + kQ / group, 0) + static_cast<long long>(len);
    return nq * (keys / (2 * kK) + 1);
  }
};

// Where the keys are in pieces, a piece has about `per` tiles of them: an even share, for as many workgroups as the
// card holds (H), of what all rows have to do, W. Row b's tiles of queries have up to p_b ≤ ⌈kt_b / per⌉ pieces,
// and those that are in pieces places for p_b parts each. As p_b − 1 < kt_b / per and Σ nq_b·kt_b·Hkv ≤ 2W ≤
// 2H·per, the pieces past the tiles' first are at most 2H, and so are the tiles in pieces. What the host makes room
// for is bounded the same way (grid_of).
struct Plan {
  int per, live;  // key tiles of a piece; tiles of queries of all rows and KV heads
  int same;       // tiles of queries of each row, where all have as many, else 0
  // Pieces of a row's tiles at most, as long as each other, of a quarter more than `per` at most: so that they do not
  // pass what the card holds by little (1024 tokens over 4096 keys, 16 heads over 4 of 96, 73 µs, 96 where pieces are `per`
  // at most), and that a row of little more than a piece stays whole (two rows of 2048 tokens over 8192 keys, 16
  // heads of 64, 283 µs, 297 with a second piece of an eighth). Pieces of `per` and a short one behind them took 90 in
  // place of 63 for 30 rows of 128 tokens over 2000 keys, 8 heads of 64.
  __host__ __device__ int pieces(int kt) const {
    const int p = (kt - per / 2 + per - 1) / per;
    return 4 * kt <= 5 * per ? 1 : p < 2 ? 2 : p;
  }
};

// mine: this lane's row, where there are no more than 64.
template <int DK>
__device__ __forceinline__ Plan plan_of(const PagedAttnArgs& a, int lane, bool first, Row& mine) {
  long long work;
  int live, nq0;
  bool good, same = true;
  if (a.B == 1) {  // (the scans and their vector values take two launches 1.5 µs)
    mine = Row::one(a, 0);
    work = mine.work(a.group);
    live = nq0 = mine.nq;
    good = mine.good;
  } else {
    work = live = nq0 = 0;
    good = true;
    for (int i = 0; i < a.B; i += 64) {
      mine = Row::load(a, i + lane);
      work += mine.work(a.group);
      live += mine.nq;
      good &= mine.good;
      if (i == 0) nq0 = __builtin_amdgcn_readfirstlane(mine.nq);
      same &= i + lane >= a.B || mine.nq == nq0;
    }
    auto sum = [](int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); };
    // (W is below 2^46: 2^22 queries by 2^24 pairs of tiles)
    work = (static_cast<long long>(sum(static_cast<int>(work >> 20))) << 20) + sum(static_cast<int>(work & 0xfffff));
    live = sum(live);
    same = __all(same);
  }
  if (!good && first) tell(a.err);
  constexpr int H = held(DK);
  const long long share = (work * a.Hkv + H - 1) / H;
  return Plan{static_cast<int>(max(static_cast<long long>(kLeastTiles), min(share, 1LL << 28))), live * a.Hkv, same ? nq0 : 0};
}

// What a workgroup does: queries from q0 on of KV head hk of row b, key tiles t0 … t0 + nt − 1, piece
// `piece` of `pieces`, whose first has its part at `slot`.
struct Tile {
  int b, hk, q0, len, n, kend, t0, nt, piece, pieces, slot;
  // The keys of the queries, in pieces of which the row's keys have p. False: this piece is not there.
  __device__ __forceinline__ bool cut(const PagedAttnArgs& a, int p) {
    const int last = min((q0 + kQ - 1) / a.group, n - 1);  // the last token
    kend = max(len - n + last + 1, 0);
    const int tiles = (kend + kK - 1) / kK, per = p == 1 ? max(tiles, 1) : ((len + kK - 1) / kK + p - 1) / p;
    pieces = max(1, (tiles + per - 1) / per);
    t0 = piece * per;
    nt = min(per, tiles - t0);
    return piece < pieces;
  }
  // All of it in scalar registers: the compiler does not see that lanes agree on it, and spills 56 vector registers at
  // float32 head dims of 256 in place of 10.
  __device__ __forceinline__ void scalars() {
    for (int* x : {&b, &hk, &q0, &len, &n, &kend, &t0, &nt, &piece, &pieces, &slot}) *x = __builtin_amdgcn_readfirstlane(*x);
  }
};

// The row that has item `at` of items that the rows have one after another: `items` of a row with p pieces
// (of a tile) of them. False: none has it. t.piece: the item's number in its row.
template <typename F>
__device__ __forceinline__ bool find_row(const PagedAttnArgs& a, const Plan& plan, const Row& mine, int at, int lane, F items, Tile& t, int& nq, int& p) {
  if (a.B == 1) {
    const Row r = Row::one(a, 0);
    t.b = t.slot = 0;
    t.len = r.len;
    t.n = r.n;
    t.piece = at;
    nq = r.nq;
    p = plan.pieces(r.kt);
    return at < items(nq * a.Hkv, p);
  }
  int before = 0, slots = 0;
  for (int i = 0; i < a.B; i += 64) {
    const Row r = a.B <= 64 ? mine : Row::load(a, i + lane);
    const int pieces = plan.pieces(r.kt), tiles = r.nq * a.Hkv;
    const int own = items(tiles, pieces), own_slots = pieces > 1 ? tiles * pieces : 0;
    const int sum = wave_scan(own), sum_slots = wave_scan(own_slots);
    const unsigned long long past = __ballot(before + sum > at);
    if (past) {
      const int l = __ffsll(past) - 1;
      t.b = i + l;
      t.len = __builtin_amdgcn_readlane(r.len, l);
      t.n = __builtin_amdgcn_readlane(r.n, l);
      t.piece = at - before - __builtin_amdgcn_readlane(sum - own, l);
      t.slot = slots + __builtin_amdgcn_readlane(sum_slots - own_slots, l);
      nq = __builtin_amdgcn_readlane(r.nq, l);
      p = __builtin_amdgcn_readlane(pieces, l);
      return true;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(sum_slots, 63);
  }
  return false;
}

// False: nothing to do. a.slots: 0 where no keys are in pieces.
template <int DK>
__device__ __forceinline__ bool find_tile(const PagedAttnArgs& a, int nq, Tile& t) {
  const int lane = threadIdx.x & 63;
  if (a.slots == 0) {
    // (row, KV head) fastest: with a multiple of 8 of them each has its XCD, whose L2 then holds its keys. The
    // last queries, which have the most keys, first.
    const int heads = a.B * a.Hkv, rest = static_cast<int>(blockIdx.x) / heads, bh = static_cast<int>(blockIdx.x) - rest * heads;
    t.b = bh / a.Hkv;
    t.hk = bh - t.b * a.Hkv;
    t.q0 = (nq - 1 - rest) * kQ;
    const Row r = Row::one(a, t.b);
    if (rest == 0 && !r.good && threadIdx.x == 0) tell(a.err);
    t.len = r.len;
    t.n = r.n;
    t.piece = t.slot = 0;
    return t.q0 < t.n * a.group && t.cut(a, 1);
  }
  // Every tile's first piece, then the others, which a tile of few keys may not have (among the first they leave
  // half of the CUs idle). Where all rows have as many tiles of queries, in the order above; else row after row.
  Row mine;
  const Plan plan = plan_of<DK>(a, lane, blockIdx.x == 0, mine);
  const int first = static_cast<int>(blockIdx.x);
  const bool more = first >= plan.live;
  int at = more ? first - plan.live : first, p = 1;
  if (!more && plan.same > 0) {
    const int heads = a.B * a.Hkv, rest = at / heads, bh = at - rest * heads, b = bh / a.Hkv;
    at = (b * plan.same + rest) * a.Hkv + (bh - b * a.Hkv);
  }
  if (!find_row(a, plan, mine, at, lane, [&](int tiles, int pieces) { return more ? tiles * (pieces - 1) : tiles; }, t, nq, p))
    return false;
  const int rest = t.piece / a.Hkv;
  t.hk = t.piece - rest * a.Hkv;
  const int turn = rest / nq, qt = nq - 1 - (rest - turn * nq);
  t.piece = turn + (more ? 1 : 0);
  t.q0 = qt * kQ;
  t.slot += (t.hk * nq + qt) * p;
  return t.cut(a, p);
}

// Where a piece's part goes: per query its reference (in powers of two) and Σ p, then its Σ p·v.
struct Parts {
  float *ml, *po;
  __device__ explicit Parts(const PagedAttnArgs& a) {
    ml = reinterpret_cast<float*>(static_cast<char*>(a.ws) + kCounterBytes);  // (behind what other calls keep there)
    po = ml + static_cast<size_t>(a.slots) * kQ * 2;
  }
};

// The pieces' parts merged in their order, four dims of a query a thread. (A launch of its own: by the
// last workgroup of a tile, as in ops_paged.hip, 32 pieces of 128 queries took 100 µs.)
constexpr int kMergers = 256;
template <typename T, int DK>
__global__ __launch_bounds__(kMergers) void paged_merge_kernel(PagedAttnArgs a) {
  constexpr int L = DK / 4, kRows = kMergers / L, kBlocks = (kQ + kRows - 1) / kRows;
  // (a block of rows of a tile in pieces)
  const int lane = threadIdx.x & 63;
  Row mine;
  const Plan plan = plan_of<DK>(a, lane, false, mine);
  if (a.B <= 64 && !__any(plan.pieces(mine.kt) > 1)) return;
  Tile w;
  int nq = 1, p = 1;
  if (!find_row(a, plan, mine, static_cast<int>(blockIdx.x) / kBlocks, lane, [](int tiles, int pieces) { return pieces > 1 ? tiles : 0; }, w, nq, p))
    return;
  w.hk = w.piece / nq;
  const int qt = w.piece - w.hk * nq;
  w.q0 = qt * kQ;
  w.slot += w.piece * p;
  w.piece = 0;
  w.cut(a, p);
  if (w.pieces == 1) return;
  const int c = blockIdx.x % kBlocks * kRows + threadIdx.x / L, d = threadIdx.x % L * 4;
  if (threadIdx.x / L >= kRows || c >= kQ || w.q0 + c >= w.n * a.group || d >= a.dk) return;
  const Parts parts(a);
  const size_t first = w.slot;
  // (float32: parts times 2^-12, whose sums of near the largest values stay finite)
  constexpr float kRoom = sizeof(T) == 2 ? 0.f : 12.f;
  float top = -INFINITY;
  for (int y = 0; y < w.pieces; ++y) top = fmaxf(top, parts.ml[2 * ((first + y) * kQ + c)]);
  const float rf = (top == -INFINITY ? 0.f : top) + kRoom;
  float lt = 0.f;
  floatx4 ot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int y = 0; y < w.pieces; ++y) {
    const size_t q = (first + y) * kQ + c;
    const f2 st = *reinterpret_cast<const f2*>(parts.ml + 2 * q);
    const floatx4 x = *reinterpret_cast<const floatx4*>(parts.po + q * DK + d);
    const float f = __builtin_amdgcn_exp2f(st.x - rf);
    lt += st.y * f;
    ot += x * f;
  }
  const int rr = w.q0 + c, tk = rr / a.group;
  T* to = static_cast<T*>(a.out) + ((static_cast<size_t>(w.b) * a.S + tk) * a.H + w.hk * a.group + rr % a.group) * a.dk + d;
  const bool sees = w.len - w.n + tk >= 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) to[e] = static_cast<T>(sees ? ot[e] / lt : 0.f);
}

// DK: head dims up to it, in steps of 8.
template <int DK>
__global__ __launch_bounds__(64 * kWaves, DK > 128 ? 1 : 2) void paged_prefill_f16_kernel(PagedAttnArgs a, int nq) {
#pragma clang fp contract(off)
  constexpr int KS = DK / 16, OT = DK / 32, VG = DK / 8;
  constexpr int L = DK <= 64 ? 8 : DK <= 128 ? 16 : 32;  // lanes of a row, 16 bytes each
  constexpr int RW = 64 / L;              // rows of a wave's load
  constexpr int CH = kK / (RW * kWaves);  // loads of a wave for a tile
  constexpr int KP = DK + 8, VP = DK == 96 ? DK : DK + 32;  // halves of a row in LDS: V's 16 banks apart for its reads
  __shared__ __align__(16) half_t Ks[2][kK][KP];
  __shared__ __align__(16) half_t Vs[2][kK][VP];
  Tile w;
  if (!find_tile<DK>(a, nq, w)) return;
  w.scalars();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dk = a.dk, R = w.n * a.group, hi = lane >> 5;
  const int qw = w.q0 + wave * 32, myq = qw + (lane & 31);  // the wave's first query, this lane's
  const bool live = myq < R;
  const int tok = min(myq, R - 1) / a.group, head = w.hk * a.group + min(myq, R - 1) % a.group;
  const int lim = w.len - w.n + tok;  // the last key that this lane's query sees
  const float cscale = kLog2e / a.scale;
  constexpr float kUp = 7.f;  // p times 2^7: at most 2^15, with all of float16's bits down to 2^-21
  // What a score in powers of two is raised by under reference x (rounded once: all that refers to x takes this)
  auto raise_of = [&](float x) { return kUp - (x == -INFINITY ? 0.f : x) * cscale; };
  const float lazy = fminf(8.0f / cscale, 3.402823466e38f);
  const half8 z8 = {0, 0, 0, 0, 0, 0, 0, 0};
  half8 qb[KS];
  {
    const half_t* qp = static_cast<const half_t*>(a.q) + ((static_cast<size_t>(w.b) * a.H + head) * a.S + tok) * dk;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qb[ks] = live && ks * 16 + hi * 8 < dk ? *reinterpret_cast<const half8*>(qp + ks * 16 + hi * 8) : z8;
  }
  // tiles that this wave reads, and the first of them that needs its mask ends past `unmasked`
  const int wlast = w.len - w.n + min((qw + 31) / a.group, w.n - 1);
  int ntw = qw >= R || wlast < 0 ? 0 : min(w.nt, max(0, wlast / kK + 1 - w.t0));
  int unmasked = w.len - w.n + qw / a.group;
  // (as vector values: scalar tests fold into the loop's, the bodies merge, and head dim 128 spills a
  // hundred registers)
  asm volatile("" : "+v"(ntw), "+v"(unmasked));

  // Page numbers of a tile's rows, lane i those of load i; a wave's load i takes rows from
  // (i·kWaves + wave)·RW on. Past the last key: its page (rows in bounds, that the mask takes out).
  const RowPages pages{a.table + static_cast<size_t>(w.b) * a.max_pages, a.shift, a.num_pages, a.Hkv, w.hk};
  const int lastkey = max(w.kend - 1, 0);
  bool bad = false;
  auto first_row = [&](int i) { return (i * kWaves + wave) * RW; };
  auto fetch_ids = [&](int t) { return pages.number(min(t * kK + first_row(lane < CH ? lane : 0), lastkey)); };
  const int col = lane % L, row = lane / L;
  const int dpos = col * 8;
  const bool mine = VG == L ? dpos < dk : col < VG && dpos < dk;
  const unsigned loff = static_cast<unsigned>((row * dk + (mine ? dpos : 0)) * 2);
  auto fetch = [&](const void* pool, int t, int ids, half8 (&dst)[CH]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int key = t * kK + first_row(i);
      const size_t at = pages.place(key, __builtin_amdgcn_readlane(ids, i), bad);
      const char* p = static_cast<const char*>(pool) + at * dk * 2;
      dst[i] = mine ? *reinterpret_cast<const half8*>(p + loff) : z8;
    }
  };
  half8 kn[CH], vn[CH];
  auto put_k = [&](auto buf_c) {
    constexpr int buf = decltype(buf_c)::value;
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (VG == L || col < VG) *reinterpret_cast<half8*>(&Ks[buf][first_row(i) + row][dpos]) = kn[i];
  };
  auto put_v = [&](auto buf_c, int t) {
    constexpr int buf = decltype(buf_c)::value;
    if ((t + 1) * kK > w.kend) {  // (what lies past the last key may be anything)
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if (t * kK + first_row(i) + row >= w.kend) vn[i] = z8;
    }
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (VG == L || col < VG) *reinterpret_cast<half8*>(&Vs[buf][first_row(i) + row][dpos]) = vn[i];
  };
  auto scores = [&](auto buf_c, floatx16 (&s)[2]) {
    constexpr int buf = decltype(buf_c)::value;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const half8 ka = *reinterpret_cast<const half8*>(&Ks[buf][t * 32 + (lane & 31)][ks * 16 + hi * 8]);
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qb[ks], s[t], 0, 0, 0);
      }
    }
  };

  float m = -INFINITY, l = 0.f;  // reference (in units of q·k) and Σ p·2^7 of this lane's query
  float mnew = -INFINITY;
  bool grow = false;
  floatx16 o[OT];
#pragma unroll
  for (int t = 0; t < OT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[t][r] = 0.f;

  // Masking of tile t's scores, their maximum, and the reference that its probabilities will use.
  auto prep = [&](auto mask_c, int t, floatx16 (&s)[2]) {
    if constexpr (decltype(mask_c)::value) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = t * kK + u * 32 + 8 * (r >> 2) + 4 * hi + (r & 3);
          if (key > lim) s[u][r] = -INFINITY;
        }
    }
    float mloc = s[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (u + r > 0) mloc = fmaxf(mloc, s[u][r]);
    float mx = fmaxf(m, mloc);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    grow = __any(mx > m + lazy);
    mnew = grow ? mx : m;
  };
  auto masked = [&](int t) { return (t + 1) * kK - 1 > unmasked; };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using T_ = std::true_type;
  using F_ = std::false_type;
  auto body = [&](auto par_c, auto next_c, auto mask_next_c, int t, floatx16 (&cur)[2], floatx16 (&nxt)[2]) {
    constexpr int PAR = decltype(par_c)::value;
    constexpr bool NEXT = decltype(next_c)::value;
    if (grow) {
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(raise_of(mnew) - raise_of(m));
      l *= alpha;
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    m = mnew;
    if constexpr (NEXT) scores(std::integral_constant<int, PAR ^ 1>{}, nxt);
    const float nmx = raise_of(m);
    const half2v ones = {static_cast<_Float16>(1.0f), static_cast<_Float16>(1.0f)};
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      half8 pb[2];
#pragma unroll
      for (int jj = 0; jj < 8; jj += 2) {
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[blk >> 1][8 * (blk & 1) + jj], cscale, nmx));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(cur[blk >> 1][8 * (blk & 1) + jj + 1], cscale, nmx));
        const half2v hp = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(p0, p1));
        const half2v lp = __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(p0 - static_cast<float>(hp[0]), p1 - static_cast<float>(hp[1])));
        l = __builtin_amdgcn_fdot2(hp, ones, l, false);
        l = __builtin_amdgcn_fdot2(lp, ones, l, false);
        pb[0][jj] = hp[0];
        pb[0][jj + 1] = hp[1];
        pb[1][jj] = lp[0];
        pb[1][jj + 1] = lp[1];
      }
      // k-slot j of lane half hi: key 8(j / 4) + 4·hi + j % 4 of the 16. A transposing read gives a lane
      // four keys of its dim from the rows that its 16 lanes point at, 8 bytes each.
      typedef __attribute__((address_space(3))) s4 lds_s4;
      // (the two products of an output apart: 2048 tokens over 8192 keys, 32 heads of 128 over 8, 420 µs in pairs
      // and 428 side by side; 16 over 4 of 256 737 in pairs, 720 in fours, 763)
      constexpr int F = DK > 128 ? 4 : 2;
      const half_t* at = &Vs[PAR][blk * 16 + 4 * hi + ((lane & 15) >> 2)][16 * ((lane >> 4) & 1) + 4 * (lane & 3)];
#pragma unroll
      for (int d = 0; d < OT; d += F) {
        half8 va[F];
#pragma unroll
        for (int f = 0; f < F && d + f < OT; ++f) {
          const s4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + (d + f) * 32));
          const s4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + (d + f) * 32 + 8 * VP));
          va[f] = __builtin_bit_cast(half8, s8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int f = 0; f < F && d + f < OT; ++f) o[d + f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va[f], pb[c], o[d + f], 0, 0, 0);
      }
    }
    if constexpr (NEXT) prep(mask_next_c, t + 1, nxt);
  };
  int ids_v = 0, ids_k = 0;  // of the next tiles to load
  auto iter = [&](auto par_c, int j, floatx16 (&cur)[2], floatx16 (&nxt)[2]) {
    constexpr int PAR = decltype(par_c)::value;
    const int t = w.t0 + j;
    __syncthreads();
    if (j + 2 < w.nt) put_k(par_c);
    if (j + 1 < w.nt) put_v(std::integral_constant<int, PAR ^ 1>{}, t + 1);
    if (j + 2 < w.nt) fetch(a.v_pages, t + 2, ids_v, vn);
    if (j + 3 < w.nt) fetch(a.k_pages, t + 3, ids_k, kn);
    ids_v = ids_k;
    if (j + 4 < w.nt) ids_k = fetch_ids(t + 4);
    if (j >= ntw) return;
    if (j + 1 >= ntw)
      body(par_c, F_{}, F_{}, t, cur, nxt);
    else if (masked(t + 1))
      body(par_c, T_{}, T_{}, t, cur, nxt);
    else
      body(par_c, T_{}, F_{}, t, cur, nxt);
  };

  floatx16 sA[2], sB[2];
  if (w.nt > 0) {  // K(0), V(0), K(1) into LDS; K(2), V(1) into registers; tile 0's scores
    const int t = w.t0, i0 = fetch_ids(t), i1 = fetch_ids(t + 1);
    ids_v = fetch_ids(t + 2);
    ids_k = fetch_ids(t + 3);
    fetch(a.k_pages, t, i0, kn);
    fetch(a.v_pages, t, i0, vn);
    put_k(I0{});
    put_v(I0{}, t);
    if (w.nt > 1) {
      fetch(a.k_pages, t + 1, i1, kn);
      fetch(a.v_pages, t + 1, i1, vn);
      put_k(I1{});
    }
    if (w.nt > 2) fetch(a.k_pages, t + 2, ids_v, kn);
    __syncthreads();
    if (ntw > 0) {
      scores(I0{}, sA);
      if (masked(t))
        prep(T_{}, t, sA);
      else
        prep(F_{}, t, sA);
    }
  }
  for (int j = 0; j < w.nt; j += 2) {
    iter(I0{}, j, sA, sB);
    if (j + 1 < w.nt) iter(I1{}, j + 1, sB, sA);
  }
  if (__any(bad) && lane == 0) tell(a.err);
  l += __shfl_xor(l, 32, 64);

  // An infinite or NaN value makes 0·∞ of keys that a query does not see: outputs that are not
  // finite are formed again, key by key, keys without weight left out.
  {
    bool wrong = false;
#pragma unroll
    for (int d = 0; d < OT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) wrong |= !__builtin_isfinite(o[d][r]);
    if (__any(wrong && live)) {
      const float nmx = raise_of(m);
      floatx16 fresh[OT];
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) fresh[d][r] = 0.f;
      const int end = min(min(w.kend, (w.t0 + w.nt) * kK), wlast + 1);
      for (int key = w.t0 * kK; key < end; ++key) {
        const size_t at = pages.place(key, pages.number(key), bad) * dk;
        const half_t *kr = static_cast<const half_t*>(a.k_pages) + at, *vr = static_cast<const half_t*>(a.v_pages) + at;
        int h = hi;
        asm volatile("" : "+v"(h));  // (the bounds tests formed here, not kept for the loop)
        float s = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (ks * 16 + h * 8 < dk) {
            const half8 kk = *reinterpret_cast<const half8*>(kr + ks * 16 + h * 8);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              s = __builtin_fmaf(static_cast<float>(qb[ks][e]), static_cast<float>(kk[e]), s);
          }
        s += __shfl_xor(s, 32, 64);
        const float p = key > lim ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(s, cscale, nmx));
        if (p != 0.f) {
#pragma unroll
          for (int d = 0; d < OT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int dim = d * 32 + 8 * (r >> 2) + 4 * h + (r & 3);
              if (dim < dk) fresh[d][r] = __builtin_fmaf(p, static_cast<float>(vr[dim]), fresh[d][r]);
            }
        }
      }
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!__builtin_isfinite(o[d][r])) o[d][r] = fresh[d][r];
    }
  }

  if (w.pieces == 1) {
    if (!live) return;
    half_t* out = static_cast<half_t*>(a.out) + ((static_cast<size_t>(w.b) * a.S + tok) * a.H + head) * dk;
    const float inv = lim < 0 ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < OT; ++d)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int dim = d * 32 + 8 * g + 4 * hi;
        half4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = static_cast<half_t>(lim < 0 ? 0.f : o[d][4 * g + e] * inv);
        if (dim < dk) *reinterpret_cast<half4*>(out + dim) = v;
      }
    return;
  }
  const Parts parts(a);
  const size_t q = (static_cast<size_t>(w.slot) + w.piece) * kQ + wave * 32 + (lane & 31);
  if (hi == 0) *reinterpret_cast<f2*>(parts.ml + 2 * q) = f2{m == -INFINITY ? m : -raise_of(m), l};
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      floatx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = o[d][4 * g + e];
      *reinterpret_cast<floatx4*>(parts.po + q * DK + d * 32 + 8 * g + 4 * hi) = v;
    }
}

// float32: the same tiles on v_mfma_f32_32x32x2f32, whose two steps of a contraction are dims 8i + e and
// 8i + 4 + e of K, so that a lane's 16 bytes of a row feed four of them, and whose 32 rows are every W-th
// dim of V, so that one read feeds W tiles of the output. A tile of keys costs 16 times the cycles on
// the matrix pipe that its softmax takes beside it: one buffer and two barriers a tile, with the other
// workgroup of the CU in between. (1024 tokens over 4096 keys: 8 heads of 64, 90 µs, 84 TFLOP/s; 8 over 2 of
// 128, 161, 93; 16 over 4 of 192, 1000 over 4000, 470, 92; a product of 8192³ reaches 153.)
template <int DK>
__global__ __launch_bounds__(256, DK > 128 ? 1 : 2) void paged_prefill_f32_kernel(PagedAttnArgs a, int nq) {
  // Keys of a tile here: 32 where 64 would take more registers than there are (1000 tokens over 4000 keys, 16
  // heads over 4 of 192, 470 µs, 475; 512 over 2048, 8 of 256, 105, 135; of 128 156.7, 158.5).
  constexpr int KT = DK > 96 ? 32 : kK;
  constexpr int KS = DK / 8, OT = DK / 32, VG = DK / 4;
  constexpr int W = OT % 4 == 0 ? 4 : OT % 2 == 0 ? 2 : 1;
  constexpr int L = DK == 32 ? 8 : DK == 64 ? 16 : DK <= 128 ? 32 : 64;  // lanes of a row, 16 bytes each
  constexpr int RW = 64 / L, CH = KT / (RW * kWaves);
  constexpr int P = DK + 4;  // floats of a row in LDS
  typedef float vecw __attribute__((ext_vector_type(W)));
  __shared__ __align__(16) float Ks[KT][P];
  __shared__ __align__(16) float Vs[KT][P];
  Tile w;
  if (!find_tile<DK>(a, nq, w)) return;
  w.scalars();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dk = a.dk, R = w.n * a.group, hi = lane >> 5, l32 = lane & 31;
  const int qw = w.q0 + wave * 32, myq = qw + l32;
  const bool live = myq < R;
  const int tok = min(myq, R - 1) / a.group, head = w.hk * a.group + min(myq, R - 1) % a.group;
  const int lim = w.len - w.n + tok;
  const float cscale = kLog2e / a.scale;
  const float lazy = fminf(8.0f / cscale, 3.402823466e38f);
  const floatx4 z4 = {0.f, 0.f, 0.f, 0.f};
  floatx4 qb[KS];
  {
    const float* qp = static_cast<const float*>(a.q) + ((static_cast<size_t>(w.b) * a.H + head) * a.S + tok) * dk;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qb[ks] = live && ks * 8 + hi * 4 < dk ? *reinterpret_cast<const floatx4*>(qp + ks * 8 + hi * 4) : z4;
  }
  const int t0 = w.t0 * (kK / KT), nt = min(w.nt * (kK / KT), (w.kend + KT - 1) / KT - t0);
  const int wlast = w.len - w.n + min((qw + 31) / a.group, w.n - 1);
  const int ntw = qw >= R || wlast < 0 ? 0 : min(nt, max(0, wlast / KT + 1 - t0));
  const int unmasked = w.len - w.n + qw / a.group;

  const RowPages pages{a.table + static_cast<size_t>(w.b) * a.max_pages, a.shift, a.num_pages, a.Hkv, w.hk};
  const int lastkey = max(w.kend - 1, 0);
  bool bad = false;
  auto first_row = [&](int i) { return (i * kWaves + wave) * RW; };
  auto fetch_ids = [&](int t) { return pages.number(min(t * KT + first_row(lane < CH ? lane : 0), lastkey)); };
  const int col = lane % L, row = lane / L, dpos = col * 4;
  const bool mine = dpos < dk, stores = VG == L || col < VG;
  const unsigned loff = static_cast<unsigned>((row * dk + (mine ? dpos : 0)) * 4);
  floatx4 kn[CH], vn[CH];
  auto fetch = [&](int t, int ids) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const size_t at = pages.place(t * KT + first_row(i), __builtin_amdgcn_readlane(ids, i), bad) * dk * 4 + loff;
      kn[i] = mine ? *reinterpret_cast<const floatx4*>(static_cast<const char*>(a.k_pages) + at) : z4;
      vn[i] = mine ? *reinterpret_cast<const floatx4*>(static_cast<const char*>(a.v_pages) + at) : z4;
    }
  };
  auto put = [&](int t) {
#pragma unroll
    for (int i = 0; i < CH; ++i)
      if (stores) {
        const int r = first_row(i) + row;
        *reinterpret_cast<floatx4*>(&Ks[r][dpos]) = kn[i];
        // (what lies past the last key may be anything)
        *reinterpret_cast<floatx4*>(&Vs[r][dpos]) = t * KT + r < w.kend ? vn[i] : z4;
      }
  };
  float m = -INFINITY, l = 0.f;
  floatx16 o[OT];
#pragma unroll
  for (int d = 0; d < OT; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[d][r] = 0.f;
  int ids = 0;
  if (nt > 0) {
    fetch(t0, fetch_ids(t0));
    ids = fetch_ids(t0 + 1);
  }
  for (int j = 0; j < nt; ++j) {
    const int t = t0 + j;
    __syncthreads();  // (the tile before is read)
    put(t);
    __syncthreads();
    if (j + 1 < nt) fetch(t + 1, ids);
    if (j + 2 < nt) ids = fetch_ids(t + 2);
    if (j >= ntw) continue;
    floatx16 s[KT / 32];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[u][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const floatx4 ka = *reinterpret_cast<const floatx4*>(&Ks[u * 32 + l32][ks * 8 + hi * 4]);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(ka[e], qb[ks][e], s[u], 0, 0, 0);
      }
    }
    if ((t + 1) * KT - 1 > unmasked) {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (t * KT + u * 32 + 8 * (r >> 2) + 4 * hi + (r & 3) > lim) s[u][r] = -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[u][r]);
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__any(mx > m + lazy)) {
      mx = fmaxf(mx, m);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mx) * cscale);
      m = mx;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f((s[u][r] - ref) * cscale);
        l += p;
        s[u][r] = p;
      }
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float* vrow = &Vs[u * 32 + 8 * (r >> 2) + 4 * hi + (r & 3)][W * l32];
#pragma unroll
        for (int d = 0; d < OT; d += W) {
          const vecw v = *reinterpret_cast<const vecw*>(vrow + 32 * d);
#pragma unroll
          for (int e = 0; e < W; ++e) o[d + e] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e], s[u][r], o[d + e], 0, 0, 0);
        }
      }
  }
  if (__any(bad) && lane == 0) tell(a.err);
  l += __shfl_xor(l, 32, 64);
  // dim of register r of output tile d
  auto dim_of = [&](int d, int r, int h) { return 32 * W * (d / W) + W * (8 * (r >> 2) + 4 * h + (r & 3)) + d % W; };
  float lifted = 0.f;  // the part is 2^-lifted of what its reference m makes it

  // Outputs that are not finite are formed again, as in the float16 kernel, of probabilities 2^-lift as
  // large: sums of values near float32's largest pass its range too.
  {
    bool wrong = false;
#pragma unroll
    for (int d = 0; d < OT; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) wrong |= !__builtin_isfinite(o[d][r]);
    if (__any(wrong && live)) {
      const float lift = 40.f - static_cast<float>(__builtin_clz(w.len)), f = __builtin_amdgcn_exp2f(-lift);
      const float base = m == -INFINITY ? 0.f : m;
      lifted = lift;
      l *= f;
      floatx16 fresh[OT];
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) fresh[d][r] = 0.f;
      const int end = min(min(w.kend, (t0 + nt) * KT), wlast + 1);
      for (int key = t0 * KT; key < end; ++key) {
        const size_t at = pages.place(key, pages.number(key), bad) * dk;
        const float *kr = static_cast<const float*>(a.k_pages) + at, *vr = static_cast<const float*>(a.v_pages) + at;
        int h = hi, c = l32;
        asm volatile("" : "+v"(h), "+v"(c));  // (the bounds tests formed here, not kept for the loop)
        float x = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          if (ks * 8 + h * 4 < dk) {
            const floatx4 kk = *reinterpret_cast<const floatx4*>(kr + ks * 8 + h * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x = __builtin_fmaf(qb[ks][e], kk[e], x);
          }
        x += __shfl_xor(x, 32, 64);
        const float p = key > lim ? 0.f : __builtin_amdgcn_exp2f((x - base) * cscale - lift);
        if (p != 0.f) {
#pragma unroll
          for (int d = 0; d < OT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int dim = dim_of(d, r, h);
              if (dim < dk) fresh[d][r] = __builtin_fmaf(p, vr[dim], fresh[d][r]);
            }
        }
      }
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = __builtin_isfinite(o[d][r]) ? o[d][r] * f : fresh[d][r];
    }
  }

  // two neighbouring dims at a time
  auto each_pair = [&](auto f) {
    if constexpr (W == 1) {
#pragma unroll
      for (int d = 0; d < OT; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 2) f(dim_of(d, r, hi), f2{o[d][r], o[d][r + 1]});
    } else {
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int d = 0; d < OT; d += 2) f(dim_of(d, r, hi), f2{o[d][r], o[d + 1][r]});
    }
  };
  if (w.pieces == 1) {
    if (!live) return;
    float* out = static_cast<float*>(a.out) + ((static_cast<size_t>(w.b) * a.S + tok) * a.H + head) * dk;
    const float inv = lim < 0 ? 0.f : 1.f / l;
    each_pair([&](int dim, f2 v) {
      if (dim < dk) *reinterpret_cast<f2*>(out + dim) = lim < 0 ? f2{0.f, 0.f} : f2{v.x * inv, v.y * inv};
    });
    return;
  }
  const Parts parts(a);
  const size_t q = (static_cast<size_t>(w.slot) + w.piece) * kQ + wave * 32 + l32;
  // A part's reference is in powers of two: what m·cscale, which may be large, and its sum with the lift are off
  // by their roundings goes into the part (halved first, so that the largest values stay finite).
  lifted += 1.f;
  float ref = -INFINITY, f = 0.5f;
  if (m != -INFINITY) {
    const float up = m * cscale;
    ref = up + lifted;
    if (__builtin_isfinite(ref)) f *= __builtin_amdgcn_exp2f(__builtin_fmaf(m, cscale, -up) + (up - (ref - lifted)));
  }
  if (hi == 0) *reinterpret_cast<f2*>(parts.ml + 2 * q) = f2{ref, l * f};
  each_pair([&](int dim, f2 v) { *reinterpret_cast<f2*>(parts.po + q * DK + dim) = f2{v.x * f, v.y * f}; });
}

// Columns of the kernel that takes a head dim.
int columns_of(int dt, int dk) {
  return dk <= 32 && dt == F32 ? 32 : dk <= 64 ? 64 : dk <= 96 ? 96 : dk <= 128 ? 128 : dk <= 192 ? 192 : 256;
}

// Tiles of queries, the workgroups that take them and their pieces, places for parts (0: no keys are in pieces) and
// tiles that may be in pieces.
struct Grid {
  int nq;
  long long groups, slots, split;
};
Grid grid_of(int dt, int B, int H, int Hkv, int S, int P, int dk) {
  Grid g;
  g.nq = (H / Hkv * S + kQ - 1) / kQ;
  const long long tiles = static_cast<long long>(g.nq) * Hkv * B, all = held(columns_of(dt, dk));
  const int most = Plan{kLeastTiles, 0, 0}.pieces((P - 1) / kK + 1);  // pieces of a tile
  g.groups = tiles;
  g.slots = g.split = 0;
  // One row's tiles that fill the card stay whole. Those of several may be of one row alone that has many new
  // tokens, or many more keys than the others; of more than 64, whose lengths a workgroup has to go through in several
  // turns, only where tiles are few (500 rows of 80 tokens over 400 keys, 4 heads of 64: 162 µs, 99 whole).
  if (most == 1 || (B == 1 && tiles >= all) || (B > 64 && 2 * tiles > all)) return g;
  g.groups = tiles + std::min(2 * all, tiles * (most - 1));
  g.split = std::min(tiles, 2 * all);
  g.slots = std::min(2 * all + g.split, tiles * most);
  return g;
}

template <typename T, int DK>
int launch_kernels(const PagedAttnArgs& a, const Grid& g, hipStream_t st) {
  const unsigned n = static_cast<unsigned>(g.groups);
  if constexpr (sizeof(T) == 2) paged_prefill_f16_kernel<DK><<<n, 64 * kWaves, 0, st>>>(a, g.nq);
  else paged_prefill_f32_kernel<DK><<<n, 64 * kWaves, 0, st>>>(a, g.nq);
  NML_LAUNCHED();
  if (g.slots == 0) return 0;
  constexpr int kRows = kMergers / (DK / 4);
  paged_merge_kernel<T, DK><<<static_cast<unsigned>(g.split * ((kQ + kRows - 1) / kRows)), kMergers, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

template <int DK>
int launch_columns(int dt, const PagedAttnArgs& a, const Grid& g, hipStream_t st) {
  return dt == F32 ? launch_kernels<float, DK>(a, g, st) : launch_kernels<half_t, DK>(a, g, st);
}

}  // namespace

// Queries of a KV head from which on this pays (µs here and with 16 queries at a time). float16: 64, one row of
// 3000 keys, 16 heads of 64 22.4 and 20.7, 8 of 128 27.2 and 22.5, 4 of 256 41 and 36, 8 rows of 1500 32 and 37, 36 and
// 37, 47 and 62; 96 22.8 and 24.9, 27.8 and 26.1, 42 and 36, 8 rows 33 and 48, 38 and 54, 49 and 62; the fewer
// the tiles and the keys the later, one row of 400 past 256 (17.0 and 15.9). float32, whose matrix
// instructions cost what they multiply, padding or not: 100 over 4000 keys of 128 58 and 33, 200 over 2000 of 64 36 and 42;
// of 256 200 over 2048 103 and 87, 512 110 and 145.
bool paged_prefill_applies(int dt, int H, int Hkv, int S, int dk) {
  return dk % (dt == F16 ? 8 : 4) == 0 && S > 1 && H / Hkv * S >= (dt == F16 ? 65 : dk <= 128 ? 128 : 256);
}

size_t paged_prefill_workspace(int dt, int B, int H, int Hkv, int S, int P, int dk) {
  const Grid g = grid_of(dt, B, H, Hkv, S, P, dk);
  return g.slots == 0 ? 0 : kCounterBytes + sizeof(float) * g.slots * kQ * (2 + columns_of(dt, dk));
}

int launch_paged_prefill(int dt, PagedAttnArgs a, hipStream_t st) {
  const Grid g = grid_of(dt, a.B, a.H, a.Hkv, a.S, a.max_pages << a.shift, a.dk);
  a.slots = static_cast<int>(g.slots);
  switch (columns_of(dt, a.dk)) {
    case 32: return launch_kernels<float, 32>(a, g, st);
    case 64: return launch_columns<64>(dt, a, g, st);
    case 96: return launch_columns<96>(dt, a, g, st);
    case 128: return launch_columns<128>(dt, a, g, st);
    case 192: return launch_columns<192>(dt, a, g, st);
  }
  return launch_columns<256>(dt, a, g, st);
}

}  // namespace nml
