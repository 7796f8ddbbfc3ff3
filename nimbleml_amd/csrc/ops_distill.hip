// Distillation from a teacher's top logits: the divergence of a model's distribution from the
// teacher's over the K tokens that the teacher's logits y are known of, row by row, and its
// gradient. With a temperature T,
//   q_k = exp(y_k/T) / Σ_j exp(y_j/T) over the K entries,  p_v = exp(x_v/T) / Σ exp(x/T) over the vocabulary
//   loss = Σ_k q_k·(log q_k − log p[id_k])
//   d x_v = dloss/T · (p_v − Σ_{k: id_k = v} q_k)
// An entry of id −1 or of y = −inf is absent; a row with no other has no teacher: its logits are not
// read, its loss and its gradient are 0. m = max x and l = Σ exp((x − m)/T) go from the forward to the
// gradient. Sums and statistics are float32 for either dtype.
//
// A workgroup goes over a row once (the forward as ops_logprob.hip: a reference of each thread's own,
// moved when a logit passes it by 8 powers of e); the teacher's entries, one a thread, are read beside
// the first pieces of the row, their logits gathered by id. The gradient writes p·dloss/T to the
// whole row first and then, behind a barrier, the elements that the teacher has entries of:
// entries of one id meet in the lowest of them, added in their order, so nothing depends on the
// order of atomics.
//
// Both are bound by HBM where rows are many. With inputs that change from call to call, 4096 rows of 32000 float16
// logits, 64 entries each: the loss 54 µs, 4.9 TB/s of reads; the gradient 120 µs, 4.4 TB/s of reads and
// writes. 2048 rows of 4096 float32 logits: 9.9 and 13.0 µs. A single row of 50304: 7.4 and 6.4 µs with its launch.
#include "kernels.hpp"
#include "row_pieces.hpp"

namespace nml {

namespace {

// Rows that leave CUs idle with four waves each: up to here sixteen waves take one.
constexpr int kFewRows = 512;
constexpr int kLaunchRows = 1 << 21;  // of one launch: its threads are counted in 32 bits
constexpr int kTeachers = kMaxDistillTop;
constexpr float kLog2e = 1.44269504088896341f;
// Differences of logits times a power of two, exactly: those of float32's largest, and their sums, stay finite
// where the temperature brings the loss back into its range.
constexpr float kFar = 0x1p-10f;

// A thread's entry of the teacher's.
struct Entry {
  int id;  // −1: absent
  float y;
};

// Entry `k` of row r. An id out of range is told, and is an entry of NaN, as which it makes the row NaN.
__device__ __forceinline__ Entry entry_of(const int64_t* ids, const float* ys, int r, int K, int k, int V, int* err) {
  Entry e{-1, -INFINITY};
  if (k < K) {
    const size_t at = static_cast<size_t>(r) * K + k;
    const int64_t id = ids[at];
    const float y = ys[at];
    if (id < -1 || id >= V) {
      if (err) __hip_atomic_fetch_or(err, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      e = Entry{0, __builtin_nanf("")};
    } else if (id >= 0 && y != -INFINITY) {
      e = Entry{static_cast<int>(id), y};
    }
  }
  return e;
}

struct Part {  // of Σ exp((x − ref)/T): the largest x seen, the reference, the sum
  float top, ref, z;
  __device__ __forceinline__ void move(float r, float c) {
    z *= __builtin_amdgcn_exp2f((ref - r) * c);
    ref = r;
  }
};

// F pieces of 16 bytes a thread in flight.
template <typename T, int NT, int F>
__global__ __launch_bounds__(NT) void distill_kernel(DistillArgs a) {
  constexpr int NW = NT / 64, KW = kTeachers / 64;
  typedef RowPieces<T> Row;
  constexpr int E = Row::E;
  typedef typename Row::vec vec;
  __shared__ Part parts[NW];
  __shared__ float top_w[KW], z_w[KW], s_w[KW];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  const Entry e = entry_of(a.top_ids, a.top_logits, r, a.K, tid, a.V, a.err);
  if (!__syncthreads_or(e.id >= 0)) {
    if (tid == 0) {
      a.loss[r] = 0.f;
      if (a.m) a.m[r] = 0.f;
      if (a.l) a.l[r] = 0.f;
    }
    return;
  }
  const float mine = e.id >= 0 ? static_cast<float>(x[e.id]) : 0.f;
  const Row row(x, a.V);
  const float c = a.c;
  const float slack = 8.f * kLog2e / c;  // in logits
  Part s{-INFINITY, kNone, 0.f};
  for (int i = tid; i - lane < row.n; i += F * NT) {
    vec v[F];
#pragma unroll
    for (int k = 0; k < F; ++k) {
      if (i + NT * k < row.n) {
        v[k] = row.load(i + NT * k);
      } else {
#pragma unroll
        for (int j = 0; j < E; ++j) v[k][j] = static_cast<T>(-INFINITY);
      }
    }
#pragma unroll
    for (int k = 0; k < F; ++k) {
      if (i - lane + NT * k >= row.n) break;
      const float top = piece_max<T>(v[k]);  // (NaN is not seen here; it reaches the sum)
      s.top = fmaxf(s.top, top);
      if (__ballot(top > s.ref + slack)) s.move(fmaxf(s.ref, top), c);
#pragma unroll
      for (int j = 0; j < E; ++j) s.z += __builtin_amdgcn_exp2f((static_cast<float>(v[k][j]) - s.ref) * c);
    }
  }
  // the wave's sum and the largest of its teacher's logits, then the workgroup's
  {
    const float top = wave_max_dpp(s.top);
    s.move(fmaxf(wave_max_dpp(s.ref), top), c);
    s.z = wave_sum_dpp(s.z);
    s.top = top;
    if (lane == 0) parts[w] = s;
    if (w < KW) {
      const float t = wave_max_dpp(e.y);
      if (lane == 0) top_w[w] = t;
    }
  }
  __syncthreads();
  Part p = lane < NW ? parts[lane] : Part{-INFINITY, kNone, 0.f};
  const float m = wave_max_dpp(p.top);
  p.move(fmaxf(m, kNone), c);
  float z = wave_sum_dpp(p.z);
  if (m == -INFINITY) z = __builtin_nanf("");
  if (w < KW) {
    float y = top_w[0];
#pragma unroll
    for (int i = 1; i < KW; ++i) y = fmaxf(y, top_w[i]);
    float q = 0.f, t = 0.f;
    if (e.id >= 0) {
      q = __builtin_amdgcn_exp2f((e.y - y) * c);
      // (the teacher's and the model's logits each from their own largest: an offset costs nothing)
      if (q != 0.f) t = q * ((e.y - y) * kFar - (mine * kFar - m * kFar));
    }
    q = wave_sum_dpp(q);
    t = wave_sum_dpp(t);
    if (lane == 0) z_w[w] = q, s_w[w] = t;
  }
  __syncthreads();
  if (tid == 0) {
    float q = 0.f, t = 0.f;
#pragma unroll
    for (int i = 0; i < KW; ++i) q += z_w[i], t += s_w[i];
    a.loss[r] = t / q * (a.inv_t / kFar) + (logf(z) - logf(q));
    if (a.m) a.m[r] = m;
    if (a.l) a.l[r] = z;
  }
}

// A workgroup takes `steps` times 256·F pieces of row blockIdx.y.
template <typename T, int F>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillBwdArgs a, int steps) {
  constexpr int NT = 256, KW = kTeachers / 64;
  static_assert(kTeachers <= NT, "an entry a thread");
  typedef RowPieces<T> Row;
  constexpr int E = Row::E;
  typedef typename Row::vec vec;
  __shared__ float top_w[KW], z_w[KW];
  __shared__ Entry entries[kTeachers];
  const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const T* x = static_cast<const T*>(a.logits) + static_cast<size_t>(r) * a.ld;
  T* out = static_cast<T*>(a.dlogits) + static_cast<size_t>(r) * a.ld_d;
  const Row row(x, a.V);
  const int c0 = blockIdx.x * steps * F * NT, c1 = min(row.n, c0 + steps * F * NT);
  if (c0 >= c1) return;
  const Entry e = entry_of(a.top_ids, a.top_logits, r, a.K, tid, a.V, blockIdx.x == 0 ? a.err : nullptr);
  const bool taught = __syncthreads_or(e.id >= 0);
  const float m = a.m[r], c = a.c;
  float s = a.dloss[r] * a.inv_t;  // of q; s / l: of exp((x − m)/T)
  const bool here = e.id >= row.first(c0) && e.id < row.first(c1) && e.id >= 0;
  float mine = 0.f;
  if (here) mine = static_cast<float>(x[e.id]);
  // the first pieces, in flight beside the teacher's entries
  vec v[F];
  auto load = [&](int i) {
#pragma unroll
    for (int k = 0; k < F; ++k)
      if (i + NT * k < c1) v[k] = row.load(i + NT * k);
  };
  if (taught) load(c0 + tid);
  float z = 0.f;  // of the teacher's exponentials
  if (taught) {
    const float t = wave_max_dpp(e.y);
    if (lane == 0) top_w[w] = t;
    __syncthreads();
    float y = top_w[0];
#pragma unroll
    for (int i = 1; i < KW; ++i) y = fmaxf(y, top_w[i]);
    const float q = e.id >= 0 ? __builtin_amdgcn_exp2f((e.y - y) * c) : 0.f;
    entries[tid] = Entry{e.id, q};
    const float sum = wave_sum_dpp(q);
    if (lane == 0) z_w[w] = sum;
    asm volatile("" : "+v"(mine));  // (it is there before the row may be overwritten)
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KW; ++i) z += z_w[i];
    if (!(z < INFINITY)) s = __builtin_nanf("");  // a NaN or +inf among them
  }
  const float sp = s / a.l[r];
  auto put = [&](int i0, const vec& d) {
    if (i0 >= 0 && i0 + E <= a.V && (reinterpret_cast<uintptr_t>(out + i0) & 15) == 0) {
      __builtin_nontemporal_store(d, reinterpret_cast<vec*>(out + i0));  // (4096 rows of 32000: 120 µs, 133 with stores kept in the caches)
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i0 + j >= 0 && i0 + j < a.V) out[i0 + j] = d[j];
    }
  };
  for (int i = c0 + tid; i < c1; i += F * NT) {
    if (taught && i >= c0 + F * NT) load(i);
#pragma unroll
    for (int k = 0; k < F; ++k) {
      if (i + NT * k >= c1) break;
      vec d;
#pragma unroll
      for (int j = 0; j < E; ++j)
        d[j] = static_cast<T>(taught ? sp * __builtin_amdgcn_exp2f((static_cast<float>(v[k][j]) - m) * c) : 0.f);
      put(row.first(i + NT * k), d);
    }
  }
  if (!taught) return;
  // the row's stores have arrived
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (here) {
    float q = 0.f;
    bool lowest = true;
    for (int k = 0; k < a.K; ++k) {
      const Entry o = entries[k];
      if (o.id == e.id) {
        q += o.y;
        lowest &= k >= tid;
      }
    }
    if (lowest) out[e.id] = static_cast<T>(sp * __builtin_amdgcn_exp2f((mine - m) * c) - s * (q / z));
  }
}

template <typename T>
int distill_launch(const DistillArgs& a, hipStream_t st) {
  for (long long r0 = 0; r0 < a.rows; r0 += kLaunchRows) {  // (r0 passes the largest int)
    DistillArgs b = a;
    b.rows = static_cast<int>(a.rows - r0 < kLaunchRows ? a.rows - r0 : kLaunchRows);
    b.logits = static_cast<const T*>(a.logits) + static_cast<size_t>(r0) * a.ld;
    b.top_ids = a.top_ids + static_cast<size_t>(r0) * a.K;
    b.top_logits = a.top_logits + static_cast<size_t>(r0) * a.K;
    b.loss = a.loss + r0;
    if (a.m) b.m = a.m + r0;
    if (a.l) b.l = a.l + r0;
    if (b.rows > kFewRows) distill_kernel<T, 256, 4><<<b.rows, 256, 0, st>>>(b);
    else distill_kernel<T, 1024, 4><<<b.rows, 1024, 0, st>>>(b);
    NML_LAUNCHED();
  }
  return 0;
}

template <typename T>
int distill_bwd_launch(const DistillBwdArgs& a, hipStream_t st) {
  constexpr int E = RowPieces<T>::E, F = 4, NT = 256;
  const int pieces = (a.V + 2 * (E - 1)) / E;  // at most, wherever a row starts
  for (long long r0 = 0; r0 < a.rows; r0 += 65535) {
    DistillBwdArgs b = a;
    b.rows = static_cast<int>(a.rows - r0 < 65535 ? a.rows - r0 : 65535);
    b.logits = static_cast<const T*>(a.logits) + static_cast<size_t>(r0) * a.ld;
    b.dlogits = static_cast<T*>(a.dlogits) + static_cast<size_t>(r0) * a.ld_d;
    b.top_ids = a.top_ids + static_cast<size_t>(r0) * a.K;
    b.top_logits = a.top_logits + static_cast<size_t>(r0) * a.K;
    b.m = a.m + r0;
    b.l = a.l + r0;
    b.dloss = a.dloss + r0;
    // whole rows where they are enough to fill the card, else parts of them
    const int all = (pieces + F * NT - 1) / (F * NT);
    const int parts = b.rows >= 2048 ? 1 : (2048 + b.rows - 1) / b.rows;
    const int steps = (all + parts - 1) / parts;
    distill_bwd_kernel<T, F><<<dim3((all + steps - 1) / steps, b.rows), NT, 0, st>>>(b, steps);
    NML_LAUNCHED();
  }
  return 0;
}

}  // namespace

int launch_distill(int dt, const DistillArgs& a, hipStream_t st) {
  if (a.rows == 0) return 0;
  return dt == F16 ? distill_launch<half_t>(a, st) : distill_launch<float>(a, st);
}

int launch_distill_backward(int dt, const DistillBwdArgs& a, hipStream_t st) {
  if (a.rows == 0) return 0;
  return dt == F16 ? distill_bwd_launch<half_t>(a, st) : distill_bwd_launch<float>(a, st);
}

}  // namespace nml
