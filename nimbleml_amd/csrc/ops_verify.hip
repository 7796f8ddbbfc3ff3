// Drafted tokens verified against the target's distribution, from given uniform numbers u. Of a
// row's drafts d_0 … d_{c−1}, drawn from q_i = softmax(draft logits_i / T) (without draft logits:
// chosen outright, q_i = 1 at d_i), and the target's p_i = softmax(logits_i / T), i = 0 … c,
//   d_i is accepted iff u_i·q_i(d_i) < p_i(d_i), up to the first that is not, r (none: r = c);
//   one more token follows, of weights max(p_r − q_r, 0) where r < c (p_r where all are 0), of p_c
//   where r = c: the first v with Σ_{j≤v} w_j > u_n·Σ w,
// which makes every token one of the target's distribution. T ≤ 0: d_i is accepted iff it is the
// target's largest logit (the lowest id of equal ones), and the token that follows is that one.
//
// Two launches. The first goes over every row of logits once, a workgroup to a part of a row: the
// largest logit and Σ exp((x − m)/T). In the second a workgroup takes a part of the row that the
// last token is drawn from: every one of them finds r from the parts' sums, sums its part's weights
// and counts itself; the last of a sequence finds the part where the running sum passes u_n·Σ w,
// forms that part's weights again and writes the sequence's answer.
//
// Exponentials and sums are in 64 bits: a token is where a running sum of V weights passes a number,
// and with 32 bits about one in 10^3 … 10^4 tokens would be the neighbour of the one that the formula
// gives. A 64-bit multiply-add runs at the rate of a 32-bit one on this card, and an exponential takes
// 14 such operations: the first launch is bound by them (and the loads before), the second by its
// chain of dependent steps, two passes over a part with a count of arrivals in between. One sequence of four
// drafts, 32000 float32 logits a row: 3.5 and 8.6 µs; 32 of up to five, 50304 float16 logits: 15.2 and 11.8.
#include "kernels.hpp"

namespace nml {

namespace {

constexpr int kThreads = 256, kMaxRows = kMaxDrafts + 1;
// Elements of a part of a row, a thread's times kThreads: few where the rows are few, so that a lone
// call's chain is short. (µs of both launches, few or many by size / always few / always many: one
// sequence of four drafts, 32000 float32, 11.5 / 11.7 / 19.7; 32 of up to five, 50304 float16, 27.0 / 27.0 /
// 29.4; 64 of eight, 32000 float16, 44.8 / 51.8 / 46.3.)
constexpr int kSmall = 8, kLarge = 32;
constexpr int kLine = 32;  // words from one sequence's counter to the next: a line of its own

// exp((x − m)/T) of x ≤ m, c = log₂ e / T (the difference first: the logits may be large): 2^n times a
// polynomial in f, n + f the exponent, |f| ≤ ½, whose coefficients are fitted to 2^f for the least
// relative error (8·10^-13, by exchange); 0 below 2^-1000, NaN of NaN. The addend 1.5·2^52 rounds to an
// integer, which the sum's low word then is.
__device__ __forceinline__ double exp64(float x, double c, double m) {
  const double t = (static_cast<double>(x) - m) * c;
  const double k = t + 6755399441055744.0, f = t - (k - 6755399441055744.0);
  double p = 1.3175858091404474e-06;
  p = __builtin_fma(p, f, 1.5309737421601964e-05);
  p = __builtin_fma(p, f, 0.0001540385174883757);
  p = __builtin_fma(p, f, 0.0013333452062250341);
  p = __builtin_fma(p, f, 0.0096181285428622344);
  p = __builtin_fma(p, f, 0.055504109393417086);
  p = __builtin_fma(p, f, 0.24022650698880371);
  p = __builtin_fma(p, f, 0.69314718054651414);
  p = __builtin_fma(p, f, 0.9999999999997623);
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, p) +
                                  (static_cast<unsigned long long>(static_cast<unsigned>(__builtin_bit_cast(unsigned long long, k))) << 52);
  return t < -1000.0 ? 0.0 : __builtin_bit_cast(double, bits);
}
// m, but finite where nothing is above −inf (every exponential is 0 then).
__device__ __forceinline__ double reference(float m) { return m == -INFINITY ? 0.0 : static_cast<double>(m); }

// Lane moves of 64-bit values on the data-parallel-primitive path (lanes without a source: 0).
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double dpp_d(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), CTRL, ROWS, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
__device__ __forceinline__ double lane_d(double v, int l) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(b), l), hi = __builtin_amdgcn_readlane(static_cast<int>(b >> 32), l);
  return __builtin_bit_cast(double, static_cast<unsigned long long>(hi) << 32 | lo);
}
// Over the 16 lanes of a row, in each of them.
__device__ __forceinline__ double row16_sum_d(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  return v + dpp_d<kDppMirror>(v);
}
__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp_move<kDppXor1>(v));
  v = fmaxf(v, dpp_move<kDppXor2>(v));
  v = fmaxf(v, dpp_move<kDppHalfMirror>(v));
  return fmaxf(v, dpp_move<kDppMirror>(v));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v = row16_sum_d(v);
  return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
// Inclusive sum over the wave's lanes.
__device__ __forceinline__ double wave_scan64(double v) {
  v += dpp_d<0x111>(v);       // row_shr:1
  v += dpp_d<0x112>(v);       // row_shr:2
  v += dpp_d<0x114>(v);       // row_shr:4
  v += dpp_d<0x118>(v);       // row_shr:8
  v += dpp_d<0x142, 0xa>(v);  // row_bcast:15
  v += dpp_d<0x143, 0xc>(v);  // row_bcast:31
  return v;
}

// Of a part of a row (or a row): the largest logit and Σ exp((x − m)/T), NaN where the row has no
// distribution (a NaN or +inf in it); greedy: the key of its best element in the sum's place.
struct Stat {
  double z;
  float m;
  int pad;
};

// Order of (logit, lower id first) as unsigned words: NaN above everything.
__device__ __forceinline__ unsigned long long key_of(float x, int i) {
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  const unsigned o = x != x ? 0xffffffffu : u & 0x80000000u ? ~u : u | 0x80000000u;
  return static_cast<unsigned long long>(o) << 32 | ~static_cast<unsigned>(i);
}

__device__ __forceinline__ unsigned long long wave_umax64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

// Elements i … i + E − 1 of a row that starts anywhere (−inf past its end).
template <typename T>
struct Group {
  static constexpr int E = 16 / static_cast<int>(sizeof(T));
  typedef T vec __attribute__((ext_vector_type(E)));
  typedef T loose __attribute__((ext_vector_type(E), aligned(sizeof(T))));
  static __device__ __forceinline__ vec load(const T* row, int i, int V) {
    if (i + E <= V) return *reinterpret_cast<const loose*>(row + i);
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = i + e < V ? row[i + e] : static_cast<T>(-INFINITY);
    return v;
  }
};

// Rows of one sequence: its n + 1 rows of the target's logits, then its n of the draft's.
__device__ __forceinline__ int drafted_of(const VerifyArgs& a, int b, bool tell) {
  if (!a.counts) return a.n;
  const int c = a.counts[b], k = c < 0 ? 0 : (c > a.n ? a.n : c);
  if (tell && c != k && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return k;
}

template <typename T, int EACH, bool GREEDY>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  typedef Group<T> G;
  constexpr int E = G::E, N = EACH / E, NW = kThreads / 64;
  __shared__ float ms[NW];
  __shared__ double zs[NW];
  __shared__ unsigned long long ks[NW];
  const int part = blockIdx.x, rows = a.n + 1 + (a.draft ? a.n : 0);
  const int b = blockIdx.y / rows, i = blockIdx.y - b * rows;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  // (the second launch's counter of this sequence)
  if (part == 0 && i == 0 && tid == 0) a.counter[b * kLine] = 0;
  const int c = drafted_of(a, b, part == 0 && i == 0 && tid == 0);
  const bool draft = i > a.n;
  if (draft ? i - a.n - 1 >= c : i > c) return;
  const T* x = draft ? static_cast<const T*>(a.draft) + (static_cast<size_t>(b) * a.n + (i - a.n - 1)) * a.ld_draft
                     : static_cast<const T*>(a.logits) + (static_cast<size_t>(b) * (a.n + 1) + i) * a.ld;
  const int first = part * kThreads * EACH;
  typename G::vec v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = first + (k * kThreads + tid) * E;
    if (at < a.V) v[k] = G::load(x, at, a.V);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = static_cast<T>(-INFINITY);
  }
  Stat* out = static_cast<Stat*>(a.stats) + static_cast<size_t>(blockIdx.y) * a.row_parts + part;
  if (GREEDY) {
    unsigned long long best = 0;
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = first + (k * kThreads + tid) * E + e;
        const unsigned long long key = key_of(static_cast<float>(v[k][e]), at);
        if (at < a.V && key > best) best = key;
      }
    best = wave_umax64(best);
    if (lane == 0) ks[w] = best;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int y = 1; y < NW; ++y) best = best > ks[y] ? best : ks[y];
      *out = Stat{__builtin_bit_cast(double, best), 0.f, 0};
    }
    return;
  }
  float m = -INFINITY;  // (NaN is not seen here; it reaches the sum, and so does +inf, as ∞ − ∞)
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, static_cast<float>(v[k][e]));
  m = wave_max_dpp(m);
  if (lane == 0) ms[w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  const double ref = reference(m);
  double z = 0.0;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) z += exp64(static_cast<float>(v[k][e]), a.c, ref);
  z = wave_sum64(z);
  if (lane == 0) zs[w] = z;
  __syncthreads();
  if (tid == 0) *out = Stat{(zs[0] + zs[1]) + (zs[2] + zs[3]), m, 0};
}

// A row from its parts, by 16 lanes (each has the result): m and Σ exp((x − m)/T), NaN without a
// distribution.
// own: its part l16, loaded ahead.
__device__ __forceinline__ Stat part_of(const Stat* s, int parts, int l16) { return l16 < parts ? s[l16] : Stat{0.0, -INFINITY, 0}; }
__device__ __forceinline__ Stat row_stat(const Stat* s, Stat own, int parts, double c, int l16) {
  float m = own.m;
  for (int k = l16 + 16; k < parts; k += 16) m = fmaxf(m, s[k].m);
  m = row16_max(m);
  const double ref = reference(m);
  double z = own.z * exp64(own.m, c, ref);
  for (int k = l16 + 16; k < parts; k += 16) z += s[k].z * exp64(s[k].m, c, ref);
  z = row16_sum_d(z);
  return Stat{m == -INFINITY ? __builtin_nan("") : z, m, 0};
}

// Sums pass between the workgroups of a sequence at agent scope (past the L2s).
__device__ __forceinline__ void put64(double* p, double v) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get64(const double* p) {
  return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT));
}

// The answer of sequence b: r accepted drafts and the token after them (−1: no distribution).
__device__ __forceinline__ void answer(const VerifyArgs& a, const int64_t* drafts, int b, int r, int64_t token, int tid) {
  for (int i = tid; i <= a.n; i += kThreads)
    a.tokens[static_cast<size_t>(b) * (a.n + 1) + i] = i < r ? drafts[i] : i == r ? token : -1;
  if (tid == 0) {
    a.accepted[b] = r;
    if (token < 0 && a.err) __hip_atomic_fetch_or(a.err, 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_greedy_kernel(VerifyArgs a) {
  __shared__ unsigned long long best[kMaxRows];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c = drafted_of(a, b, false);
  if (tid < c) {  // (drafts behind the first that is refused are told too)
    const int64_t d = a.drafts[static_cast<size_t>(b) * a.n + tid];
    if ((d < 0 || d >= a.V) && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const Stat* s = static_cast<const Stat*>(a.stats) + static_cast<size_t>(b) * (a.n + 1) * a.row_parts;
  for (int i = w; i <= c; i += kThreads / 64) {
    unsigned long long k = 0;
    for (int y = lane; y < a.row_parts; y += 64) {
      const unsigned long long o = __builtin_bit_cast(unsigned long long, s[i * a.row_parts + y].z);
      k = k > o ? k : o;
    }
    k = wave_umax64(k);
    if (lane == 0) best[i] = k;
  }
  __syncthreads();
  int r = 0;
  int64_t token = -1;
  for (;; ++r) {
    const unsigned o = static_cast<unsigned>(best[r] >> 32);
    token = o == 0xffffffffu || o <= 0x007fffffu ? -1 : static_cast<int64_t>(~static_cast<unsigned>(best[r]));
    if (r == c || token < 0) break;
    const int64_t d = a.drafts[static_cast<size_t>(b) * a.n + r];
    if (d != token) break;
  }
  answer(a, a.drafts + static_cast<size_t>(b) * a.n, b, r, token, tid);
}

template <typename T, int EACH>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
#pragma clang fp contract(off)  // (equal probabilities leave nothing: no product of one side kept unrounded)
  typedef Group<T> G;
  constexpr int E = G::E, N = EACH / E, NW = kThreads / 64;
  __shared__ Stat ps[kMaxRows], qs[kMaxRows];
  __shared__ int64_t ids[kMaxRows];
  __shared__ double sums[NW], before_, goal_;
  __shared__ int r_, part_, hits[NW], ends[NW];
  __shared__ bool last_;
  const int part = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t* drafts = a.drafts + static_cast<size_t>(b) * a.n;
  const double* u = a.u + static_cast<size_t>(b) * (a.n + 1);
  auto target = [&](int i) { return static_cast<const T*>(a.logits) + (static_cast<size_t>(b) * (a.n + 1) + i) * a.ld; };
  auto drafted = [&](int i) { return static_cast<const T*>(a.draft) + (static_cast<size_t>(b) * a.n + i) * a.ld_draft; };
  // All that the acceptance takes is loaded before anything is waited for but the drafts and their count, which
  // say what logits are read: those of drafts past the count are not there. (Of their rows' parts, which may
  // hold anything, nothing is used.)
  const int c = drafted_of(a, b, false);
  const int rows = a.n + 1 + (a.draft ? a.n : 0), l16 = tid & 15;
  const Stat* stats = static_cast<const Stat*>(a.stats) + static_cast<size_t>(b) * rows * a.row_parts;
  auto row_at = [&](int i) { return stats + static_cast<size_t>(i) * a.row_parts; };
  int i = tid >> 4;
  Stat ahead{};
  if (i < rows) ahead = part_of(row_at(i), a.row_parts, l16);
  bool ok = true;
  float dp = 0.f, dq = 0.f;
  double du = 0.0;
  if (tid < a.n) {  // (the first wave)
    const int64_t d = drafts[tid];
    du = u[tid];
    ok = d >= 0 && d < a.V;
    if (ok && tid < c) {
      dp = static_cast<float>(target(tid)[d]);
      if (a.draft) dq = static_cast<float>(drafted(tid)[d]);
    }
    ids[tid] = d;
  }
  const double last_u = u[a.n];
  while (i < rows) {
    const Stat s = row_stat(row_at(i), ahead, a.row_parts, a.c, l16);
    if (l16 == 0) {
      if (i <= a.n) ps[i] = s;
      else qs[i - a.n - 1] = s;
    }
    i += kThreads / 16;
    if (i < rows) ahead = part_of(row_at(i), a.row_parts, l16);
  }
  if (!a.draft && tid < a.n) qs[tid] = Stat{1.0, 0.f, 0};
  __syncthreads();
  if (w == 0) {
    if (lane >= c) ok = true;
    else if (!ok && part == 0 && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (lane < c && ok) {
      const double pd = exp64(dp, a.c, reference(ps[lane].m)) / ps[lane].z;
      const double qd = a.draft ? exp64(dq, a.c, reference(qs[lane].m)) / qs[lane].z : 1.0;
      ok = du * qd < pd;  // (false where either has no distribution)
    }
    const unsigned long long no = __ballot(!ok);
    if (lane == 0) r_ = no ? __ffsll(no) - 1 : c;
  }
  __syncthreads();
  const int r = r_;
  const Stat p = ps[r], q = qs[r];
  const bool refused = r < c;
  if (!(p.z > 0.0) || (refused && !(q.z > 0.0))) {
    if (part == 0) answer(a, ids, b, r, -1, tid);
    return;
  }
  const T *xp = target(r), *xq = refused && a.draft ? drafted(r) : nullptr;
  const int64_t d = refused && !a.draft ? ids[r] : -1;
  const double ip = 1.0 / p.z, iq = 1.0 / q.z, mp = reference(p.m), mq = xq ? reference(q.m) : 0.0;
  // The weights of EACH elements, in groups of E that lie `step` apart from `first` on: what p has above q
  // (`over`), or p; past the row's end 0.
  double wt[EACH];
  auto weigh = [&](int first, int step, bool over) {
    typename G::vec vp[N], vq[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int at = first + k * step;
#pragma unroll
      for (int e = 0; e < E; ++e) vp[k][e] = vq[k][e] = static_cast<T>(-INFINITY);
      if (at < a.V) {
        vp[k] = G::load(xp, at, a.V);
        if (xq) vq[k] = G::load(xq, at, a.V);
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const double all = exp64(static_cast<float>(vp[k][e]), a.c, mp) * ip;
        double left = fmax(all - exp64(static_cast<float>(vq[k][e]), a.c, mq) * iq, 0.0);
        if (first + k * step + e == d) left = 0.0;
        wt[k * E + e] = over ? left : all;
      }
  };
  // Twice through the same code (which the second time is there): for this part's sum of weights; and,
  // by the last workgroup of the sequence to arrive, for the part where the running sum passes the
  // goal, EACH elements in a row to a thread. A refused draft whose p is nowhere above q (by
  // rounding alone): the token is p's, whose sum is 1, part by part.
  enum { kSum, kFind, kWalk } mode = kSum;
  double* mine = static_cast<double*>(a.sums) + static_cast<size_t>(b) * a.parts;
  int at = part, end_before = -1;
  double before = 0.0, goal = 0.0;
#pragma unroll 1
  for (;;) {
    const int first = mode == kSum ? at * kThreads * EACH + tid * E : (at * kThreads + tid) * EACH;
    weigh(first, mode == kSum ? kThreads * E : E, mode != kWalk && refused);
    double own = 0.0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) own += wt[k];
    const double scan = wave_scan64(own);
    __syncthreads();  // (what the time before left in LDS is read)
    if (lane == 63) sums[w] = scan;
    __syncthreads();
    if (mode == kSum) {
      if (tid == 0) {
        put64(mine + part, (sums[0] + sums[1]) + (sums[2] + sums[3]));
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        last_ = __hip_atomic_fetch_add(a.counter + b * kLine, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == static_cast<unsigned>(a.parts);
      }
      __syncthreads();
      if (!last_) return;
      if (w == 0) {  // the part where the running sum passes the goal (none: the last with a weight)
        const double kept = lane < a.parts ? get64(mine + lane) : 0.0;  // (the first 64)
        double total = kept;
        for (int k = lane + 64; k < a.parts; k += 64) total += get64(mine + k);
        total = wave_sum64(total);
        const double to = last_u * total;
        double carry = 0.0, start = 0.0;
        int found = -1;
        for (int k0 = 0; k0 < a.parts; k0 += 64) {
          const double s = k0 == 0 ? kept : k0 + lane < a.parts ? get64(mine + k0 + lane) : 0.0;
          const double run = carry + wave_scan64(s);
          const unsigned long long past = __ballot(run > to && s > 0.0), any = __ballot(s > 0.0);
          if (any) {
            const int l = past ? __ffsll(past) - 1 : 63 - __clzll(any);
            found = k0 + l;
            start = lane_d(run - s, l);
          }
          if (past) break;
          carry = lane_d(run, 63);
        }
        if (lane == 0) part_ = found, before_ = start, goal_ = to;
      }
      __syncthreads();
      mode = part_ < 0 ? kWalk : kFind;
      at = max(part_, 0);
      before = part_ < 0 ? 0.0 : before_;
      goal = part_ < 0 ? last_u : goal_;
      continue;
    }
    double run = before + (scan - own);
    for (int y = 0; y < w; ++y) run += sums[y];
    // this thread's first element past the goal, and its last with a weight; then the part's
    int hit = -1, end = -1;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      run += wt[k];
      if (wt[k] > 0.0) {
        end = first + k;
        if (hit < 0 && run > goal) hit = end;
      }
    }
    const unsigned long long past = __ballot(hit >= 0), any = __ballot(end >= 0);
    if (lane == (past ? __ffsll(past) - 1 : 0)) hits[w] = hit;
    if (lane == (any ? 63 - __clzll(any) : 0)) ends[w] = end;
    __syncthreads();
    int token = -1;
#pragma unroll
    for (int y = NW - 1; y >= 0; --y) {
      if (hits[y] >= 0) token = hits[y];
      end_before = max(end_before, ends[y]);
    }
    if (mode == kWalk && token < 0 && at + 1 < a.parts) {
      before += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      ++at;
      continue;
    }
    // (none: the running sum ends below what its parts add up to, by rounding: the last with a weight)
    answer(a, ids, b, r, token < 0 ? end_before : token, tid);
    return;
  }
}

// Elements of a part to a thread, of `rows` rows of V: as many as leave two workgroups for every CU.
int each_of(long long rows, int V) { return rows * V >= 512LL * kThreads * kLarge ? kLarge : kSmall; }
int parts_of(long long rows, int V) {
  const int part = kThreads * each_of(rows, V);
  return (V + part - 1) / part;
}
// Rows of logits that a call may have to go over.
long long rows_of(int B, int n) { return static_cast<long long>(B) * (2 * n + 1); }

template <typename T, int EACH>
int stats_launch(const VerifyArgs& a, hipStream_t st) {
  const dim3 grid(a.row_parts, static_cast<unsigned>(a.B) * (a.n + 1 + (a.draft ? a.n : 0)));
  if (a.greedy) verify_stats_kernel<T, EACH, true><<<grid, kThreads, 0, st>>>(a);
  else verify_stats_kernel<T, EACH, false><<<grid, kThreads, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

template <typename T>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
  NML_TRY((each_of(rows_of(a.B, a.n), a.V) == kLarge ? stats_launch<T, kLarge>(a, st) : stats_launch<T, kSmall>(a, st)));
  const dim3 grid(a.parts, a.B);
  if (a.greedy) verify_greedy_kernel<T><<<a.B, kThreads, 0, st>>>(a);
  else if (each_of(a.B, a.V) == kLarge) verify_draw_kernel<T, kLarge><<<grid, kThreads, 0, st>>>(a);
  else verify_draw_kernel<T, kSmall><<<grid, kThreads, 0, st>>>(a);
  NML_LAUNCHED();
  return 0;
}

// The workspace: a Stat for each part of a row, a sum for each part of a sequence's deciding row, a counter.
struct Layout {
  size_t stats, sums, all;
  Layout(int B, int n, int V) {
    stats = sizeof(Stat) * rows_of(B, n) * parts_of(rows_of(B, n), V);
    sums = stats + sizeof(double) * parts_of(B, V) * B;
    all = sums + sizeof(unsigned) * kLine * B;
  }
};

}  // namespace

size_t verify_workspace(int B, int n, int V) { return Layout(B, n, V).all; }

int launch_verify(int dt, VerifyArgs a, void* ws, hipStream_t st) {
  const Layout at(a.B, a.n, a.V);
  a.row_parts = parts_of(rows_of(a.B, a.n), a.V);
  a.parts = parts_of(a.B, a.V);
  char* p = static_cast<char*>(ws);
  a.stats = p;
  a.sums = p + at.stats;
  a.counter = reinterpret_cast<unsigned*>(p + at.sums);
  return dt == F16 ? verify_launch<half_t>(a, st) : verify_launch<float>(a, st);
}

}  // namespace nml
