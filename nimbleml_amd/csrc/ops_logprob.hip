// Log probabilities of given tokens from logits, with the distribution's entropy and its best
// alternatives, and their gradient with respect to the logits. With m = max x, t = x − m and
// Z = Σ exp t:
//   logp = t[target] − log Z,  entropy = log Z − Σ exp(t)·t / Z,  p = exp(t) / Z
//   d logits = dlogp·([v = target] − p) − dentropy·p·(log p + entropy)
// m and Z go from the forward to the gradient apart (m + log Z in one float32 would lose log Z
// beside a large m, as of a row at the type's lowest value). Sums and statistics are float32 for
// either dtype. A logit of −inf has probability 0 and adds nothing; a row of nothing else has no
// distribution: logp and entropy are NaN, as log_softmax's.
//
// A workgroup takes a row and goes over it once: each thread keeps Σ exp(t) and Σ exp(t)·t of its
// logits relative to a reference of its own, which moves only when a logit passes it by 8 (so the
// sums are scaled a few times a row, not once a logit); the threads' sums meet at the end. Rows
// are read as the aligned 16-byte pieces that hold them (a row of an odd vocabulary starts
// anywhere); what such a piece holds of the neighbouring rows is not read but taken as −inf.
// Bound by memory: 4096 rows of 50304 float16 logits in 80 µs, 5.2 TB/s; the gradient, which reads
// and writes them once (ignored rows: writes), of 4096 rows of 32000 with every seventh ignored in
// 90 µs, 5.4 TB/s. exp is exp2 of t·log₂ e rounded to float32: log probabilities of rows of 32000 to
// 50304 are 6.4e-8 to 7e-8 relative off the exact ones, a float32 rounding (5e-8 to 6e-8 in
// elementary float32 operations). A few rows are bound by the latency of the passes (32 rows of
// 32000 float32 logits: 5.5 µs, 11.8 with 20 alternatives).
#include "kernels.hpp"
#include "row_pieces.hpp"

namespace nml {

namespace {

// Rows that leave CUs idle with four waves each (two a CU): up to here sixteen waves take one.
constexpr int kFewRows = 512;
// Rows of one launch: its threads are counted in 32 bits.
constexpr int kLaunchRows = 1 << 21;
// Gathered candidates of the alternatives; more than this takes the rounds below.
constexpr int kCandidates = 1024;

// Order of logits as unsigned words: NaN above everything (by one word below the largest, which with
// id 0 would be the bound that the first of the rounds starts under), −0 equal to +0.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xfffffffeu;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The logit of such a word.
__device__ __forceinline__ float value_of(unsigned o) {
  return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ unsigned long long wave_umax64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

constexpr float kLowest = -1e4f;          // exp of it is 0, its product with that too
// A thread's part of Σ exp(x − ref) and Σ exp(x − ref)·(x − ref), and the largest x it has seen.
struct Part {
  float top, ref, z, zt;
  // of another reference r (at least the largest x, or this part's own)
  __device__ __forceinline__ void move(float r) {
    const float d = fmaxf(ref - r, kLowest), f = exp_of(d);
    zt = f * (zt + z * d);
    z *= f;
    ref = r;
  }
};

template <typename T>
__device__ __forceinline__ void add_piece(Part& s, const typename RowPieces<T>::vec& v) {
  const float top = piece_max<T>(v);  // (NaN is not seen here; it reaches the sums)
  s.top = fmaxf(s.top, top);
  if (__ballot(top > s.ref + 8.f)) s.move(fmaxf(s.ref, top));
#pragma unroll
  for (int e = 0; e < RowPieces<T>::E; ++e) {
    const float t = static_cast<float>(v[e]) - s.ref, p = exp_of(t);
    s.z += p;
    s.zt += p * fmaxf(t, kLowest);
  }
}

// NCH pieces a thread, all loaded at once and kept for the alternatives; NCH = 0: any number, four
// in flight, read again for the alternatives.
template <typename T, int NT, int NCH>
__global__ __launch_bounds__(NT) void logprob_kernel(LogprobArgs a) {
  constexpr int NW = NT / 64;
  typedef RowPieces<T> Row;
  constexpr int E = Row::E;
  typedef typename Row::vec vec;
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  __shared__ Part parts[NW];
  __shared__ float thr_w[NW];
  __shared__ unsigned long long best_w[NW];
  __shared__ unsigned long long cand[kCandidates];
  __shared__ int ncand, counts[NW];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t y = a.targets ? a.targets[r] : 0;
  if (a.targets && a.has_ignore && y == a.ignore_index) {
    if (tid == 0) {
      if (a.logp) a.logp[r] = 0.f;
      if (a.entropy) a.entropy[r] = 0.f;
      if (a.m) a.m[r] = 0.f;
      if (a.l) a.l[r] = 0.f;
    }
    for (int i = tid; i < a.top_k; i += NT) {
      a.top_ids[static_cast<size_t>(r) * a.top_k + i] = -1;
      a.top_logp[static_cast<size_t>(r) * a.top_k + i] = 0.f;
    }
    return;
  }
  const T* l = static_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  const Row row(l, a.V);
  const bool bad = a.targets && (y < 0 || y >= a.V);
  const float target = a.targets && !bad ? static_cast<float>(l[y]) : __builtin_nanf("");
  u4 reg[NCH > 0 ? NCH : 1];
  auto none = [] {
    vec v;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = static_cast<T>(-INFINITY);
    return v;
  };
  if (NCH > 0) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + NT * k;
      reg[k] = __builtin_bit_cast(u4, c < row.n ? row.load(c) : none());
    }
  }
  // f(piece's first element, its values) for each of this thread's pieces (a wave together: for
  // lanes past the row −inf)
  auto each = [&](auto f) {
    if (NCH > 0) {
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        if (NT * k + 64 * w < row.n) {
          int c = tid + NT * k;
          asm volatile("" : "+v"(reg[k]), "+v"(c));  // (as loaded, nothing made of it kept from pass to pass)
          f(row.first(c), __builtin_bit_cast(vec, reg[k]));
          __builtin_amdgcn_sched_barrier(0);
        }
    } else {
      constexpr int F = 4;
      for (int c = tid; c - lane < row.n; c += F * NT) {
        vec v[F];
#pragma unroll
        for (int k = 0; k < F; ++k) v[k] = c + NT * k < row.n ? row.load(c + NT * k) : none();
#pragma unroll
        for (int k = 0; k < F; ++k)
          if (c - lane + NT * k < row.n) f(row.first(c + NT * k), v[k]);
      }
    }
  };
  Part s{-INFINITY, kNone, 0.f, 0.f};
  each([&](int, const vec& v) { add_piece<T>(s, v); });
  const float mine = s.top;
  // the wave's sums, then the row's, relative to the largest logit (−inf where nothing is above:
  // then to a finite reference, and the row has no distribution)
  {
    const float top = wave_max_dpp(s.top), ref = wave_max_dpp(s.ref);
    s.move(fmaxf(ref, top));
    s.z = wave_sum_dpp(s.z);
    s.zt = wave_sum_dpp(s.zt);
    s.top = top;
    if (lane == 0) parts[w] = s;
  }
  __syncthreads();
  // (one wave's part a lane: with every thread going over all sixteen 32 rows of 32000 logits and
  // 20 alternatives took 12.6 µs instead of 12.2)
  Part p = lane < NW ? parts[lane] : Part{-INFINITY, kNone, 0.f, 0.f};
  const float mx = wave_max_dpp(p.top);
  p.move(fmaxf(mx, kNone));
  float z = wave_sum_dpp(p.z);
  const float zt = wave_sum_dpp(p.zt);
  if (mx == -INFINITY) z = __builtin_nanf("");
  const float lz = logf(z);
  if (tid == 0) {
    if (bad && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.logp) a.logp[r] = (target - mx) - lz;
    if (a.entropy) a.entropy[r] = lz - zt / z;
    if (a.m) a.m[r] = mx;
    if (a.l) a.l[r] = z;
  }
  if (a.top_k == 0) return;

  // A value that at least top_k logits reach: in each wave whose lanes all hold some of the row,
  // the q-th largest of the lanes' maxima, the least of them over those waves.
  const int full = min(NW, row.n / 64);
  float thr = -INFINITY;
  if (tid == 0) ncand = 0;
  if (full > 0) {
    const int q = (a.top_k + full - 1) / full;
    float top = mine, m = 0.f;
    bool out = false;
    for (int i = 0; i < q; ++i) {
      m = wave_max_dpp(out ? -INFINITY : top);
      const unsigned long long at = __ballot(!out && top == m);
      if (lane == __ffsll(at) - 1) out = true;
    }
    if (lane == 0) thr_w[w] = m;
    __syncthreads();
    thr = thr_w[0];
    for (int i = 1; i < full; ++i) thr = fminf(thr, thr_w[i]);
  }
  __syncthreads();
  auto key = [](float x, int i) { return static_cast<unsigned long long>(order_of(x)) << 32 | ~static_cast<unsigned>(i); };
  const bool ordered = z == z;  // no NaN among the logits
  if (ordered && NCH > 0) {
    // kept pieces: a first pass counts, a second one writes to places known by then (what a piece
    // holds past the row counts where the bound is −inf, with a word below every logit's)
    int n = 0;
    each([&](int, const vec& v) {
#pragma unroll
      for (int e = 0; e < E; ++e) n += static_cast<float>(v[e]) >= thr;
    });
    int at = wave_scan(n);
    if (lane == 63) counts[w] = at;
    at -= n;
    __syncthreads();
    const int before = wave_scan(lane < NW ? counts[lane] : 0);
    if (w > 0) at += __builtin_amdgcn_readlane(before, w - 1);
    if (tid == 0) ncand = __builtin_amdgcn_readlane(before, 63);
    each([&](int i, const vec& v) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (static_cast<float>(v[e]) >= thr) {
          if (at < kCandidates) cand[at] = i + e >= 0 && i + e < a.V ? key(static_cast<float>(v[e]), i + e) : 0;
          ++at;
        }
    });
  } else if (ordered) {
    each([&](int i, const vec& v) {
      if (!__ballot(piece_max<T>(v) >= thr)) return;
      // places for the wave's candidates of this piece at once
      unsigned long long take[E];
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        take[e] = __ballot(static_cast<float>(v[e]) >= thr && i + e >= 0 && i + e < a.V);
        n += __popcll(take[e]);
      }
      int at = 0;
      if (lane == 0) at = atomicAdd(&ncand, n);
      at = __builtin_amdgcn_readfirstlane(at);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int mine = at + __builtin_amdgcn_mbcnt_hi(static_cast<unsigned>(take[e] >> 32),
                                                        __builtin_amdgcn_mbcnt_lo(static_cast<unsigned>(take[e]), 0));
        if (take[e] >> lane & 1 && mine < kCandidates) cand[mine] = key(static_cast<float>(v[e]), i + e);
        at += __popcll(take[e]);
      }
    });
  }
  __syncthreads();
  int64_t* ids = a.top_ids + static_cast<size_t>(r) * a.top_k;
  float* lps = a.top_logp + static_cast<size_t>(r) * a.top_k;
  auto put = [&](int at, unsigned long long k) {
    ids[at] = ~static_cast<unsigned>(k);
    lps[at] = (value_of(static_cast<unsigned>(k >> 32)) - mx) - lz;
  };
  const int n = ncand;
  if (ordered && n <= kCandidates) {  // each candidate's place: how many come before it
    constexpr int kShare = 8;         // lanes to a candidate
    for (int i0 = 0; i0 < n; i0 += NT / kShare) {
      const int i = i0 + tid / kShare;
      const unsigned long long k = i < n ? cand[i] : ~0ull;
      int before = 0;
      for (int j = tid % kShare; j < n; j += kShare) before += cand[j] > k;
      before += __shfl_xor(before, 1, 64);
      before += __shfl_xor(before, 2, 64);
      before += __shfl_xor(before, 4, 64);
      if (i < n && tid % kShare == 0 && before < a.top_k) put(before, k);
    }
    return;
  }
  // Many equal logits (masked vocabularies) or NaN: the next one in order, top_k times (every key is
  // below the first bound).
  unsigned long long last = ~0ull;
  for (int t = 0; t < a.top_k; ++t) {
    unsigned long long best = 0;
    each([&](int i, const vec& v) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= 0 && i + e < a.V) {
          const unsigned long long k = key(static_cast<float>(v[e]), i + e);
          if (k < last && k > best) best = k;
        }
    });
    best = wave_umax64(best);
    if (lane == 0) best_w[w] = best;
    __syncthreads();
    best = best_w[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) best = best > best_w[i] ? best : best_w[i];
    __syncthreads();
    if (tid == 0) put(t, best);
    last = best;
  }
}

// A thread takes 16-byte pieces of one row; the output in such pieces too where it is aligned as
// the input is.
template <typename T>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogprobBwdArgs a) {
  typedef RowPieces<T> Row;
  constexpr int E = Row::E;
  typedef typename Row::vec vec;
  const int r = blockIdx.y;
  const Row row(static_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld, a.V);
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= row.n) return;
  T* out = static_cast<T*>(a.dlogits) + static_cast<size_t>(r) * a.ld_d;
  const int64_t y = a.targets[r];
  const bool ignored = a.has_ignore && y == a.ignore_index, bad = !ignored && (y < 0 || y >= a.V);
  const float m = a.m[r], lz = logf(a.l[r]), h = a.dentropy ? a.entropy[r] : 0.f;
  float dl = a.dlogp ? a.dlogp[r] : 0.f;
  const float dh = a.dentropy ? a.dentropy[r] : 0.f;
  if (bad) {
    if (c == 0 && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    dl = __builtin_nanf("");
  }
  const int i0 = row.first(c);
  vec d;
  if (ignored) {
#pragma unroll
    for (int e = 0; e < E; ++e) d[e] = static_cast<T>(0.f);
  } else {
    const vec x = row.load(c);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float lp = (static_cast<float>(x[e]) - m) - lz, p = exp_of(lp);
      float g = -p * (dl + dh * (fmaxf(lp, kLowest) + h));
      if (i0 + e == y) g += dl;
      d[e] = static_cast<T>(g);
    }
  }
  if (i0 >= 0 && i0 + E <= a.V && (reinterpret_cast<uintptr_t>(out + i0) & 15) == 0) {
    *reinterpret_cast<vec*>(out + i0) = d;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (i0 + e >= 0 && i0 + e < a.V) out[i0 + e] = d[e];
  }
}

template <typename T>
int logprobs_launch(const LogprobArgs& a, hipStream_t st) {
  constexpr int E = RowPieces<T>::E;
  const int pieces = (a.V + 2 * (E - 1)) / E;  // at most, wherever a row starts
#define NML_LOGPROB(NT, NCH) logprob_kernel<T, NT, NCH><<<b.rows, NT, 0, st>>>(b)
  for (long long r0 = 0; r0 < a.rows; r0 += kLaunchRows) {  // (r0 passes the largest int)
    LogprobArgs b = a;
    b.rows = static_cast<int>(a.rows - r0 < kLaunchRows ? a.rows - r0 : kLaunchRows);
    b.logits = static_cast<const T*>(a.logits) + static_cast<size_t>(r0) * a.ld;
    if (a.targets) b.targets = a.targets + r0;
    if (a.logp) b.logp = a.logp + r0;
    if (a.entropy) b.entropy = a.entropy + r0;
    if (a.m) b.m = a.m + r0;
    if (a.l) b.l = a.l + r0;
    if (a.top_k) b.top_ids = a.top_ids + static_cast<size_t>(r0) * a.top_k;
    if (a.top_k) b.top_logp = a.top_logp + static_cast<size_t>(r0) * a.top_k;
    // Few rows: all of a row's loads at once, over as many lanes as a workgroup has (32 rows of
    // 50304 float16 logits, 20 alternatives: 14.5 µs, 21.4 with four waves a row; 32000 float32
    // ones 12.6 and 20.3). Many rows overlap each other's latency: four waves a row, without the
    // wait for the last of sixteen (4096 rows of 50304 float16 logits: 80 µs, 128 with sixteen).
    if (pieces <= 256 * 4) NML_LOGPROB(256, 4);
    else if (b.rows > kFewRows) NML_LOGPROB(256, 0);
    else if (pieces <= 1024 * 4) NML_LOGPROB(1024, 4);
    else if (pieces <= 1024 * 8) NML_LOGPROB(1024, 8);
    else NML_LOGPROB(1024, 0);
    NML_LAUNCHED();
  }
#undef NML_LOGPROB
  return 0;
}

template <typename T>
int logprobs_bwd_launch(const LogprobBwdArgs& a, hipStream_t st) {
  constexpr int E = RowPieces<T>::E;
  const int pieces = (a.V + 2 * (E - 1)) / E;
  for (long long r0 = 0; r0 < a.rows; r0 += 65535) {  // rows of one launch (r0 passes the largest int)
    LogprobBwdArgs b = a;
    b.rows = static_cast<int>(a.rows - r0 < 65535 ? a.rows - r0 : 65535);
    b.logits = static_cast<const T*>(a.logits) + static_cast<size_t>(r0) * a.ld;
    b.dlogits = static_cast<T*>(a.dlogits) + static_cast<size_t>(r0) * a.ld_d;
    b.targets = a.targets + r0;
    b.m = a.m + r0;
    b.l = a.l + r0;
    if (a.entropy) b.entropy = a.entropy + r0;
    if (a.dlogp) b.dlogp = a.dlogp + r0;
    if (a.dentropy) b.dentropy = a.dentropy + r0;
    logprob_bwd_kernel<T><<<dim3((pieces + 255) / 256, b.rows), 256, 0, st>>>(b);
    NML_LAUNCHED();
  }
  return 0;
}

}  // namespace

int launch_logprobs(int dt, const LogprobArgs& a, hipStream_t st) {
  if (a.rows == 0) return 0;
  return dt == F16 ? logprobs_launch<half_t>(a, st) : logprobs_launch<float>(a, st);
}

int launch_logprobs_backward(int dt, const LogprobBwdArgs& a, hipStream_t st) {
  if (a.rows == 0) return 0;
  return dt == F16 ? logprobs_bwd_launch<half_t>(a, st) : logprobs_bwd_launch<float>(a, st);
}

}  // namespace nml
