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
// gives. A 64-bit multiply-add runs at the rate of a 32-bit one on this card, and the exponential
// below takes 14 of them.
#include "kernels.hpp"

namespace nml {

namespace {

constexpr int kThreads = 256, kEach = 32, kPart = kThreads * kEach;  // elements of a part of a row
constexpr int kMaxRows = kMaxDrafts + 1;

// 2^t for t ≤ 0: 2^⌊t⌉ times the exponential series of (t − ⌊t⌉)·ln 2 up to the tenth power (what
// is left out is below 3·10^-13 of it).
__device__ __forceinline__ double exp2_64(double t) {
  t = fmax(t, -1200.0);  // (−inf: 0; a NaN is found by other means)
  const double n = rint(t), f = (t - n) * 0.693147180559945309417;
  double p = 1.0 / 3628800.0;
  p = p * f + 1.0 / 362880.0;
  p = p * f + 1.0 / 40320.0;
  p = p * f + 1.0 / 5040.0;
  p = p * f + 1.0 / 720.0;
  p = p * f + 1.0 / 120.0;
  p = p * f + 1.0 / 24.0;
  p = p * f + 1.0 / 6.0;
  p = p * f + 0.5;
  p = p * f + 1.0;
  p = p * f + 1.0;
  return ldexp(p, static_cast<int>(n));
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

template <typename T, bool GREEDY>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  typedef Group<T> G;
  constexpr int E = G::E, N = kEach / E, NW = kThreads / 64;
  __shared__ float ms[NW];
  __shared__ double zs[NW];
  __shared__ unsigned long long ks[NW];
  const int part = blockIdx.x, rows = a.n + 1 + (a.draft ? a.n : 0);
  const int b = blockIdx.y / rows, i = blockIdx.y - b * rows;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  // (the second launch's counter of this sequence)
  if (part == 0 && i == 0 && tid == 0) a.counter[b] = 0;
  const int c = drafted_of(a, b, part == 0 && i == 0 && tid == 0);
  const bool draft = i > a.n;
  if (draft ? i - a.n - 1 >= c : i > c) return;
  const T* x = draft ? static_cast<const T*>(a.draft) + (static_cast<size_t>(b) * a.n + (i - a.n - 1)) * a.ld_draft
                     : static_cast<const T*>(a.logits) + (static_cast<size_t>(b) * (a.n + 1) + i) * a.ld;
  const int first = part * kPart;
  typename G::vec v[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = first + (k * kThreads + tid) * E;
    if (at < a.V) v[k] = G::load(x, at, a.V);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] = static_cast<T>(-INFINITY);
  }
  Stat* out = static_cast<Stat*>(a.stats) + static_cast<size_t>(blockIdx.y) * a.parts + part;
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
  float m = -INFINITY;
  bool none = false;  // a NaN or +inf
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float f = static_cast<float>(v[k][e]);
      m = fmaxf(m, f);
      none |= !(f < INFINITY);
    }
  m = wave_max_dpp(m);
  if (lane == 0) ms[w] = m;
  const bool bad = __syncthreads_or(none);
  m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
  const double ref = m == -INFINITY ? 0.0 : static_cast<double>(m);
  double z = 0.0;
  if (!bad) {
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) z += exp2_64((static_cast<double>(static_cast<float>(v[k][e])) - ref) * a.c);
  }
  z = wave_sum_d(z);
  if (lane == 0) zs[w] = z;
  __syncthreads();
  if (tid == 0) *out = Stat{bad ? __builtin_nan("") : (zs[0] + zs[1]) + (zs[2] + zs[3]), m, 0};
}

// Row `i` of sequence b from its parts, by one wave: m and Σ exp((x − m)/T), NaN without a
// distribution.
__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, int b, int i, int lane) {
  const int rows = a.n + 1 + (a.draft ? a.n : 0);
  const Stat* s = static_cast<const Stat*>(a.stats) + (static_cast<size_t>(b) * rows + i) * a.parts;
  float m = -INFINITY;
  for (int k = lane; k < a.parts; k += 64) m = fmaxf(m, s[k].m);
  m = wave_max_dpp(m);
  double z = 0.0;
  for (int k = lane; k < a.parts; k += 64)
    z += s[k].z * exp2_64(s[k].m == m ? 0.0 : (static_cast<double>(s[k].m) - static_cast<double>(m)) * a.c);
  z = wave_sum_d(z);
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

__device__ __forceinline__ double wave_scan_d(double v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}

// The answer of sequence b: r accepted drafts and the token after them (−1: no distribution).
__device__ __forceinline__ void answer(const VerifyArgs& a, int b, int r, int64_t token, int tid) {
  for (int i = tid; i <= a.n; i += kThreads)
    a.tokens[static_cast<size_t>(b) * (a.n + 1) + i] = i < r ? a.drafts[static_cast<size_t>(b) * a.n + i] : i == r ? token : -1;
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
  const Stat* s = static_cast<const Stat*>(a.stats) + static_cast<size_t>(b) * (a.n + 1) * a.parts;
  for (int i = w; i <= c; i += kThreads / 64) {
    unsigned long long k = 0;
    for (int y = lane; y < a.parts; y += 64) {
      const unsigned long long o = __builtin_bit_cast(unsigned long long, s[i * a.parts + y].z);
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
    if ((d < 0 || d >= a.V) && tid == 0 && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (d != token) break;
  }
  answer(a, b, r, token, tid);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
  typedef Group<T> G;
  constexpr int E = G::E, N = kEach / E, NW = kThreads / 64;
  __shared__ Stat ps[kMaxRows], qs[kMaxRows];
  __shared__ double sums[2][NW];
  __shared__ int r_, at_, part_;
  __shared__ double before_, goal_;
  __shared__ bool left_, last_;
  const int part = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int c = drafted_of(a, b, false);
  for (int i = w; i <= c; i += NW) {
    const Stat p = row_stat(a, b, i, lane);
    const Stat q = a.draft && i < c ? row_stat(a, b, a.n + 1 + i, lane) : Stat{1.0, 0.f, 0};
    if (lane == 0) ps[i] = p, qs[i] = q;
  }
  __syncthreads();
  const int64_t* drafts = a.drafts + static_cast<size_t>(b) * a.n;
  const double* u = a.u + static_cast<size_t>(b) * (a.n + 1);
  auto target = [&](int i) { return static_cast<const T*>(a.logits) + (static_cast<size_t>(b) * (a.n + 1) + i) * a.ld; };
  auto drafted = [&](int i) { return static_cast<const T*>(a.draft) + (static_cast<size_t>(b) * a.n + i) * a.ld_draft; };
  if (w == 0) {  // a draft a lane
    bool ok = true;
    if (lane < c) {
      const int64_t d = drafts[lane];
      ok = d >= 0 && d < a.V;
      if (!ok && part == 0 && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (ok) {
        const double pd = exp2_64((static_cast<double>(static_cast<float>(target(lane)[d])) - ps[lane].m) * a.c) / ps[lane].z;
        const double qd = !a.draft ? 1.0 : exp2_64((static_cast<double>(static_cast<float>(drafted(lane)[d])) - qs[lane].m) * a.c) / qs[lane].z;
        ok = u[lane] * qd < pd;  // (false where either has no distribution)
      }
    }
    const unsigned long long no = __ballot(!ok);
    if (lane == 0) r_ = no ? __ffsll(no) - 1 : c;
  }
  __syncthreads();
  const int r = r_;
  const Stat p = ps[r], q = qs[r];
  const bool refused = r < c;
  if (!(p.z > 0.0) || (refused && !(q.z > 0.0))) {
    if (part == 0) answer(a, b, r, -1, tid);
    return;
  }
  const T *xp = target(r), *xq = refused && a.draft ? drafted(r) : nullptr;
  const int64_t d = refused && !a.draft ? drafts[r] : -1;
  const double ip = 1.0 / p.z, iq = 1.0 / q.z;
  // the weights of element i: what p has above q, and p
  auto weigh = [&](float fp, float fq, int i, double& left, double& all) {
    all = exp2_64((static_cast<double>(fp) - p.m) * a.c) * ip;
    left = all;
    if (xq) left = fmax(all - exp2_64((static_cast<double>(fq) - q.m) * a.c) * iq, 0.0);
    if (i == d) left = 0.0;
  };
  double left = 0.0, all = 0.0;
  for (int k = 0; k < N; ++k) {
    const int at = part * kPart + (k * kThreads + tid) * E;
    if (at >= a.V) break;
    const typename G::vec vp = G::load(xp, at, a.V);
    typename G::vec vq = vp;
    if (xq) vq = G::load(xq, at, a.V);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      double l1, a1;
      weigh(static_cast<float>(vp[e]), static_cast<float>(vq[e]), at + e, l1, a1);
      left += l1;
      all += a1;
    }
  }
  left = wave_sum_d(left);
  all = wave_sum_d(all);
  if (lane == 0) sums[0][w] = left, sums[1][w] = all;
  __syncthreads();
  double* mine = static_cast<double*>(a.sums) + 2 * static_cast<size_t>(b) * a.parts;
  if (tid == 0) {
    put64(mine + 2 * part, (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]));
    put64(mine + 2 * part + 1, (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last_ = __hip_atomic_fetch_add(a.counter + b, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == static_cast<unsigned>(a.parts);
  }
  __syncthreads();
  if (!last_) return;

  // The last of the sequence: the part where the running sum passes the goal, by one wave.
  if (w == 0) {
    double total[2] = {0.0, 0.0};
    for (int k = lane; k < a.parts; k += 64) total[0] += get64(mine + 2 * k), total[1] += get64(mine + 2 * k + 1);
    total[0] = wave_sum_d(total[0]);
    total[1] = wave_sum_d(total[1]);
    const int which = total[0] > 0.0 ? 0 : 1;
    const double goal = u[a.n] * total[which];
    double carry = 0.0, before = 0.0;
    int found = -1, some = 0;
    double some_before = 0.0;
    for (int k0 = 0; k0 < a.parts && found < 0; k0 += 64) {
      const double s = k0 + lane < a.parts ? get64(mine + 2 * (k0 + lane) + which) : 0.0;
      const double run = carry + wave_scan_d(s, lane);
      const unsigned long long past = __ballot(run > goal && s > 0.0), any = __ballot(s > 0.0);
      const int l = past ? __ffsll(past) - 1 : any ? 63 - __clzll(any) : 0;
      const double b4 = __shfl(run - s, l, 64);
      if (past) found = k0 + l, before = b4;
      else if (any) some = k0 + l, some_before = b4;
      carry = __shfl(run, 63, 64);
    }
    if (lane == 0) {
      part_ = found < 0 ? some : found;
      before_ = found < 0 ? some_before : before;
      goal_ = goal;
      left_ = which == 0;
      at_ = 0x7fffffff;
    }
  }
  __syncthreads();
  // its weights again, kEach in a row to a thread
  const int first = part_ * kPart + tid * kEach;
  double own = 0.0, wt[kEach];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int at = first + k * E;
    typename G::vec vp, vq;
    if (at < a.V) {
      vp = G::load(xp, at, a.V);
      vq = vp;
      if (xq) vq = G::load(xq, at, a.V);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      double l1 = 0.0, a1 = 0.0;
      if (at < a.V) weigh(static_cast<float>(vp[e]), static_cast<float>(vq[e]), at + e, l1, a1);
      own += wt[k * E + e] = left_ ? l1 : a1;
    }
  }
  const double scan = wave_scan_d(own, lane);
  if (lane == 63) sums[0][w] = scan;
  __syncthreads();
  double run = before_ + (scan - own);
  for (int y = 0; y < w; ++y) run += sums[0][y];
  int hit = 0x7fffffff, end = -1;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    run += wt[k];
    if (wt[k] > 0.0) {
      end = first + k;
      if (hit == 0x7fffffff && run > goal_) hit = first + k;
    }
  }
  atomicMin(&at_, hit);
  __syncthreads();
  int at = at_;
  if (at == 0x7fffffff) {  // the running sum ends below what its parts add up to: the last with a weight
    __syncthreads();
    if (tid == 0) at_ = -1;
    __syncthreads();
    atomicMax(&at_, end);
    __syncthreads();
    at = at_;
  }
  answer(a, b, r, at, tid);
}

template <typename T>
int verify_launch(const VerifyArgs& a, hipStream_t st) {
  const int rows = a.n + 1 + (a.draft ? a.n : 0);
  const dim3 grid(a.parts, static_cast<unsigned>(a.B) * rows);
  if (a.greedy) {
    verify_stats_kernel<T, true><<<grid, kThreads, 0, st>>>(a);
    NML_LAUNCHED();
    verify_greedy_kernel<T><<<a.B, kThreads, 0, st>>>(a);
  } else {
    verify_stats_kernel<T, false><<<grid, kThreads, 0, st>>>(a);
    NML_LAUNCHED();
    verify_draw_kernel<T><<<dim3(a.parts, a.B), kThreads, 0, st>>>(a);
  }
  NML_LAUNCHED();
  return 0;
}

size_t stats_bytes(int B, int n, int parts) { return sizeof(Stat) * (2 * static_cast<size_t>(n) + 1) * parts * B; }
int parts_of(int V) { return (V + kPart - 1) / kPart; }

}  // namespace

size_t verify_workspace(int B, int n, int V) {
  const size_t parts = parts_of(V);
  return stats_bytes(B, n, static_cast<int>(parts)) + 2 * sizeof(double) * parts * B + sizeof(unsigned) * B;
}

int launch_verify(int dt, VerifyArgs a, void* ws, hipStream_t st) {
  a.parts = parts_of(a.V);
  char* p = static_cast<char*>(ws);
  a.stats = p;
  a.sums = p + stats_bytes(a.B, a.n, a.parts);
  a.counter = reinterpret_cast<unsigned*>(static_cast<double*>(a.sums) + 2 * static_cast<size_t>(a.parts) * a.B);
  return dt == F16 ? verify_launch<half_t>(a, st) : verify_launch<float>(a, st);
}

}  // namespace nml
