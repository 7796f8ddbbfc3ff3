// Log probabilities of given tokens from logits, with the distribution's entropy and its best
// alternatives, and their gradient with respect to the logits. With m = max x, t = x − m and
// Z = Σ exp t:
//   logp = t[target] − log Z,  entropy = log Z − Σ exp(t)·t / Z,  p = exp(t) / Z
//   d logits = dlogp·([v = target] − p) − dentropy·p·(log p + entropy)
// m and Z go from the forward to the gradient apart (m + log Z in one float32 would lose log Z
// beside a large m, as of a row at the type's lowest value). Sums and statistics are float32 for
// either dtype. A logit of −inf has probability 0 and adds
// nothing; a row of nothing else has no distribution: logp and entropy are NaN, as log_softmax's.
//
// A workgroup takes a row. Rows are read as the aligned 16-byte pieces that hold them (a row of
// an odd vocabulary starts anywhere); what such a piece holds of the neighbouring rows is not
// read but taken as −inf.
#include "kernels.hpp"

namespace nml {

namespace {

// Gathered candidates of the alternatives; more than this takes the rounds below.
constexpr int kCandidates = 1024;

__device__ __forceinline__ float exp_of(float t) { return __builtin_amdgcn_exp2f(t * 1.44269504088896341f); }

// Order of logits as unsigned words: NaN above everything, −0 equal to +0.
__device__ __forceinline__ unsigned order_of(float x) {
  if (x != x) return 0xffffffffu;
  const unsigned u = __builtin_bit_cast(unsigned, x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

__device__ __forceinline__ unsigned long long wave_umax64(unsigned long long v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor(v, o, 64);
    v = v > w ? v : w;
  }
  return v;
}

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
    vec r;
#pragma unroll
    for (int e = 0; e < E; ++e) r[e] = i + e >= 0 && i + e < V ? row[i + e] : static_cast<T>(-INFINITY);
    return r;
  }
};

// NCH pieces a thread in registers; NCH = 0: any number, read again for every pass.
template <typename T, int NT, int NCH>
__global__ __launch_bounds__(NT) void logprob_kernel(LogprobArgs a) {
  constexpr int NW = NT / 64;
  typedef RowPieces<T> Row;
  constexpr int E = Row::E;
  typedef typename Row::vec vec;
  __shared__ float red[2][16];
  __shared__ unsigned thr_w[16];
  __shared__ unsigned long long best_w[16];
  __shared__ unsigned long long cand[kCandidates];
  __shared__ int ncand;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
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
  vec reg[NCH > 0 ? NCH : 1];
  const int per = NCH > 0 ? NCH : (row.n + NT - 1) / NT;
  if (NCH > 0) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = tid + NT * k;
      if (c < row.n) {
        reg[k] = row.load(c);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) reg[k][e] = static_cast<T>(-INFINITY);
      }
    }
  }
  // f(piece's first element, its values) for each of this thread's pieces
  auto each = [&](auto f) {
    if (NCH > 0) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) f(row.first(tid + NT * k), reg[k]);
    } else {
      for (int k = 0; k < per; ++k)
        if (tid + NT * k < row.n) f(row.first(tid + NT * k), row.load(tid + NT * k));
    }
  };
  float mine = -INFINITY;
  each([&](int, const vec& v) {
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, static_cast<float>(v[e]));
  });
  float mx = wave_max(mine);
  if (lane == 0) red[0][w] = mx;
  __syncthreads();
  mx = red[0][0];
#pragma unroll
  for (int i = 1; i < NW; ++i) mx = fmaxf(mx, red[0][i]);
  __syncthreads();
  float z = 0.f, zt = 0.f;
  each([&](int, const vec& v) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = static_cast<float>(v[e]) - mx, p = exp_of(t);
      z += p;
      zt += p * fmaxf(t, -1e4f);  // (p is 0 there)
    }
  });
  z = wave_sum(z);
  zt = wave_sum(zt);
  if (lane == 0) red[0][w] = z, red[1][w] = zt;
  __syncthreads();
  z = 0.f, zt = 0.f;
#pragma unroll
  for (int i = 0; i < NW; ++i) z += red[0][i], zt += red[1][i];
  const float lz = logf(z);
  if (tid == 0) {
    const bool bad = a.targets && (y < 0 || y >= a.V);
    if (bad && a.err) __hip_atomic_fetch_or(a.err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (a.logp) a.logp[r] = bad ? __builtin_nanf("") : (static_cast<float>(l[y]) - mx) - lz;
    if (a.entropy) a.entropy[r] = lz - zt / z;
    if (a.m) a.m[r] = mx;
    if (a.l) a.l[r] = z;
  }
  if (a.top_k == 0) return;

  // A word that at least top_k logits reach: in each wave whose lanes all hold some of the row,
  // the q-th largest of the lanes' maxima, the least of them over those waves.
  const int full = min(NW, row.n / 64);
  if (tid == 0) ncand = 0;
  unsigned thr = 0;
  if (full > 0) {
    unsigned top = 0;
    each([&](int i, const vec& v) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= 0 && i + e < a.V) {
          const unsigned o = order_of(static_cast<float>(v[e]));
          top = top > o ? top : o;
        }
    });
    const int q = (a.top_k + full - 1) / full;
    unsigned m = 0;
    for (int i = 0; i < q; ++i) {
      m = wave_umax(top);
      const unsigned long long at = __ballot(top == m);
      if (lane == __ffsll(at) - 1) top = 0;
    }
    if (lane == 0) thr_w[w] = m;
    __syncthreads();
    thr = thr_w[0];
    for (int i = 1; i < full; ++i) thr = min(thr, thr_w[i]);
  }
  __syncthreads();
  auto key = [](float x, int i) { return static_cast<unsigned long long>(order_of(x)) << 32 | ~static_cast<unsigned>(i); };
  each([&](int i, const vec& v) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (i + e >= 0 && i + e < a.V && order_of(static_cast<float>(v[e])) >= thr) {
        const int at = atomicAdd(&ncand, 1);
        if (at < kCandidates) cand[at] = key(static_cast<float>(v[e]), i + e);
      }
  });
  __syncthreads();
  int64_t* ids = a.top_ids + static_cast<size_t>(r) * a.top_k;
  float* lps = a.top_logp + static_cast<size_t>(r) * a.top_k;
  auto put = [&](int at, unsigned long long k) {
    const unsigned id = ~static_cast<unsigned>(k);
    ids[at] = id;
    lps[at] = (static_cast<float>(l[id]) - mx) - lz;
  };
  const int n = ncand;
  if (n <= kCandidates) {  // each candidate's place: how many come before it
    for (int i = tid; i < n; i += NT) {
      const unsigned long long k = cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += cand[j] > k;
      if (before < a.top_k) put(before, k);
    }
    return;
  }
  // Many equal logits (masked vocabularies): the next one in order, top_k times.
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
      float g = -p * (dl + dh * (fmaxf(lp, -1e4f) + h));  // (p is 0 below)
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
#define NML_LOGPROB(NT, NCH) logprob_kernel<T, NT, NCH><<<a.rows, NT, 0, st>>>(a)
  if (pieces <= 256 * 4) NML_LOGPROB(256, 4);
  else if (pieces <= 512 * 8) NML_LOGPROB(512, 8);
  else if (pieces <= 512 * 16) NML_LOGPROB(512, 16);
  else if (pieces <= 1024 * 16) NML_LOGPROB(1024, 16);
  else NML_LOGPROB(1024, 0);
#undef NML_LOGPROB
  NML_LAUNCHED();
  return 0;
}

template <typename T>
int logprobs_bwd_launch(const LogprobBwdArgs& a, hipStream_t st) {
  constexpr int E = RowPieces<T>::E;
  const int pieces = (a.V + 2 * (E - 1)) / E;
  for (int r0 = 0; r0 < a.rows; r0 += 65535) {  // rows of one launch
    LogprobBwdArgs b = a;
    b.rows = a.rows - r0 < 65535 ? a.rows - r0 : 65535;
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
