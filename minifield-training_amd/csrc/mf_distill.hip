// Distillation from a teacher's top logits on gfx950: the loss of every row, its
// gradient with respect to the student's logits, or both in one pass.
//
// Row of V logits z, temperature T, teacher entries (i_k, t_k), k < K:
//   q = softmax(z / T),   p_k = exp(t_k / T) / sum over k of exp(t_k / T),   r = 0,
// or, where the logarithm L of the teacher's whole sum is known,
//   p_k = exp(t_k / T - L),   r = max(0, 1 - sum p_k),
// and with P = sum p_k, s = sum of q_j over the j that no entry names:
//   loss = w T^2 [ sum p_k (log p_k - log q_{i_k}) + r (log r - log s) ]
//   d loss / d z_j = w T [ q_j (P + r) - sum of p_k with i_k = j - r q_j / s [j not named] ].
// With L known, the logits that no entry names (the rest; one bit per logit in LDS tells) are
// summed beside a maximum of their own: with m' = max of them, e'_j = exp((z_j - m') / T),
// S' = sum e', f = exp((m' - max z) / T) and S = S' f + sum of exp((z_i - max z) / T) over the
// named i, the dense elements are e'_j times one factor of their row,
//   w T (f (P + r) / S - r / S'),
// and the K named ones are written anew, w T (exp((z_i - max z) / T) (P + r) / S - p);
// log s = (m' - max z) / T + log S' - log S.  A student whose logits of the entries are far
// above all others leaves a mass beyond them that is no number in fp32 (f is zero from 87 T
// on); its logarithm, and what its gradient says to the rest, do not need it.  Without L all
// logits are the rest: m' = max z, f = 1, S = S'.
//
// Exponentials of logits and their sums are fp32 (each thread adds at most 768: 512 of
// them, 393216 logits); the K masses, 1 - P and the few logarithms of a row are 64-bit, since
// they cancel: at log q = -20 and a loss of 1 the fp32 terms alone would cost 1e-6.
//
// Bound: memory, one read of the logits and one write of the gradient.  A workgroup
// of 256, 512 or 1024 takes a row.  Rows of up to 16 vectors of 16 bytes a thread stay in
// registers between the maximum, the sum and the gradient; longer ones are read again.
//
// Measured, 4096 x 65536 bf16 (512 MiB), 64 entries a row: loss 95-104 us (5.2-5.7
// TB/s), gradient from what it saved 173 (6.2 TB/s, a part of the logits still in the
// cache), both in one pass 207, with the teacher's total too (5.2 TB/s; a copy of the logits
// takes 206); 2048 x 65536 fp32 (512 MiB): loss 90 us, and its gradient 199.  64 rows of 65536
// bf16: loss 8.5 us.  24 rows of 131077: loss 13.8 us (one CU a row, its
// exponentials), gradient 6.4.
#include <algorithm>

#include "mf_distill.h"
#include "mf_rows.h"

namespace mf {

struct DistillArgs {
  const void* logits;
  const void* teacher;
  const void* ids;
  const float* total;     // or null
  const float* weights;   // or null: ones
  const float* upstream;  // backward: d sum / d loss of every row
  void* grad;
  float* loss;
  float* stats;
  long long stride, grad_stride;
  int vocabulary, top;
  float scale;  // log2(e) / T
  double temperature, per;  // T and 1 / T
  bool teacher_f32, ids64;
};

__device__ __forceinline__ int teacher_id(const DistillArgs& a, size_t at) {
  const long long id = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[at]
                               : (long long)reinterpret_cast<const int32_t*>(a.ids)[at];
  return id >= 0 && id < a.vocabulary ? (int)id : -1;
}

// exp((z - top) / T).  The difference first: a product of the type's lowest value
// with `scale` would be infinite, and a row of nothing else not uniform.
__device__ __forceinline__ float weight_of(float z, float top, float scale) {
  return fast_exp2((z - top) * scale);
}

// A named element of a row's gradient: after the dense ones.  mass: weighted by w T.
template <typename T>
__device__ __forceinline__ void store_named(T* grad, int id, float z, float mass, float top,
                                            float scale, float factor) {
  grad[id] = (T)fmaf(weight_of(z, top, scale), factor, -mass);
}

template <typename T, bool STREAM>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  const auto* u = reinterpret_cast<const typename RowVec<T>::U*>(p);
  return (Vec<T>)(STREAM ? __builtin_nontemporal_load(u) : *u);
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[kVec<T>]) {
  typename RowVec<T>::U u;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) u[i] = (T)x[i];
  __builtin_nontemporal_store(u, reinterpret_cast<typename RowVec<T>::U*>(p));
}

// A row's entries in LDS, and what wave 0 makes of them in 64 bits.
struct Teacher {
  int id[kDistillMostTop];  // -1: not there, nor behind the last up to a multiple of 8
  float z[kDistillMostTop];
  double mass[kDistillMostTop];
  float whole, rest;  // P + r and r
  int none, bad;      // no entry at all; one that is NaN or +infinity
  float top;          // the largest named logit, where the total is known
  int twice;          // and whether an id is named more than once
};

// Wave 0, while the row is on its way: masses, P, and the part of the loss that knows the
// teacher alone, sum p_k log p_k.  u0: entry `lane` of the teacher.
__device__ __forceinline__ void weigh_teacher(const DistillArgs& a, size_t row, int lane,
                                              float u0, Teacher& t, double& P, double& kl) {
  const int K = a.top;
  const bool tail = a.total != nullptr;
  bool there = false, bad = false;
  auto entry = [&](int k) {
    if (k >= K || t.id[k] < 0) return kNegInf;
    const float u = element(a.teacher, a.teacher_f32, row * K + k);
    bad |= !(u < kPosInf);
    there |= u != kNegInf;
    return u;
  };
  float first = kNegInf;
  if (lane < K && t.id[lane] >= 0) {
    first = u0;
    bad |= !(u0 < kPosInf);
    there |= u0 != kNegInf;
  }
  double shift, total;  // what the entries are taken beside, and the logarithm of their sum there
  if (tail) {
    shift = 0;
    total = a.total[row];
    bad |= !(a.total[row] < kPosInf);
  } else {
    float most = first;
    for (int k = lane + 64; k < K; k += 64) most = fmaxf(most, entry(k));
    most = max64(most);
    // (entries that are all -infinity have no mass, like none at all)
    shift = most == kNegInf ? 0.0 : (double)most;
    double s = exp((first - shift) * a.per);
    for (int k = lane + 64; k < K; k += 64) s += exp((entry(k) - shift) * a.per);
    s = sum64(s);
    total = s > 0 ? log(s) : 0.0;
  }
  P = kl = 0;
  for (int k = lane; k < K; k += 64) {
    const double logp = ((k == lane ? first : entry(k)) - shift) * a.per - total;
    const double mass = exp(logp);
    if (mass > 0) kl += mass * logp;
    t.mass[k] = mass;
    P += mass;
  }
  P = sum64(P);
  // without an entry there is no loss and no gradient, whatever the row holds; otherwise
  // an entry or a total that is NaN or +infinity makes the row NaN
  const bool none = !tail && !__any(there);
  bad = !none && __any(bad);
  if (lane == 0) {
    const double r = tail ? fmax(0.0, 1.0 - P) : 0.0;
    t.whole = (float)(P + r);
    t.rest = (float)r;
    t.none = none;
    t.bad = bad;
  }
}

// The loss, with `stats` what the backward needs, and with GRAD the gradient of the
// weighted loss.  U: vectors a thread has in flight; RESIDENT: they are the row.
template <typename T, bool GRAD, int THREADS, int U, bool RESIDENT>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(4)))
void distill_kernel(DistillArgs a) {
  constexpr int N = kVec<T>, W = THREADS / 64;
  extern __shared__ uint32_t named[];  // a bit per logit, where the total is known
  __shared__ Teacher t;
  __shared__ float part[3][W];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const size_t row = blockIdx.x;
  const int V = a.vocabulary, K = a.top;
  // (by a scalar load: the row's own wait for nothing else)
  typedef const __attribute__((address_space(4))) float* Scalars;
  const float w = a.weights ? ((Scalars)a.weights)[row] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  T* grad = GRAD ? reinterpret_cast<T*>(a.grad) + row * a.grad_stride : nullptr;
  // whole vectors; what is left of the row is one more value of each of the first threads
  const int vectors = V / N, odd = vectors * N + tid;
  auto no_gradient = [&] {
    const float zero[N] = {};
    for (int v = tid; v < vectors; v += THREADS) store_vec<T>(grad + (size_t)v * N, zero);
    if (odd < V) grad[odd] = (T)0.f;
  };
  if (w == 0.f) {  // whatever the row holds
    if (tid == 0) a.loss[row] = 0.f;
    if constexpr (GRAD) no_gradient();
    return;
  }
  const bool tail = a.total != nullptr;
  constexpr int STEP = U * THREADS;
  Vec<T> raw[U];
  // (loads have no condition: vectors beyond the row are its last.  The loss alone leaves
  // the logits in the last-level cache for the backward pass: read as a stream, its 4096 x
  // 65536 bf16 take 184 us, so 172)
  auto fetch = [&](Vec<T> (&to)[U], int first) {
    if (vectors == 0) return;
#pragma unroll
    for (int u = 0; u < U; ++u)
      to[u] = load_vec<T, GRAD>(z + (size_t)min(first + u * THREADS + tid, vectors - 1) * N);
  };
  auto blank = [&](int first) {
    if (first + STEP <= vectors) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const u32x4 x = __builtin_bit_cast(u32x4, raw[u]);
      constexpr uint32_t low = N == 8 ? 0xff80ff80u : 0xff800000u;  // -infinity
      const bool in = first + u * THREADS + tid < vectors;
      raw[u] = __builtin_bit_cast(Vec<T>, u32x4{in ? x[0] : low, in ? x[1] : low, in ? x[2] : low,
                                                in ? x[3] : low});
    }
  };
  // wave 0 asks for the entries in front of the row, and for their logits behind it: loads
  // return in order, and what is needed first comes first
  const int K8 = (K + 7) & ~7;
  int id0 = -1;
  float u0 = 0.f;
  if (wave == 0 && lane < K) {
    id0 = teacher_id(a, row * K + lane);
    u0 = element(a.teacher, a.teacher_f32, row * K + lane);
  }
  float extra = odd < V ? (float)z[odd] : kNegInf;
  fetch(raw, 0);
  float z0 = 0.f;
  if (wave == 0) {
    if (id0 >= 0) z0 = (float)z[id0];
    if (lane < K8) t.id[lane] = id0;
    for (int k = lane + 64; k < K8; k += 64) {
      const int id = k < K ? teacher_id(a, row * K + k) : -1;
      t.id[k] = id;
      t.z[k] = id >= 0 ? (float)z[id] : 0.f;
    }
  }
  if (tail) {
    for (int i = tid; i < (V + 31) / 32; i += THREADS) named[i] = 0;
    if (tid == 0) t.twice = 0;
  }
  // A vector of the row as it was loaded.  Each pass widens its values anew, one vector at
  // a time (left to itself the compiler keeps the first pass's, twice the registers in
  // bf16, and all exponentials of a pass: scratch).
  auto as_loaded = [&](int u) {
    u32x4 x = __builtin_bit_cast(u32x4, raw[u]);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(x));
    return __builtin_bit_cast(Vec<T>, x);
  };
  double P = 0, kl = 0;
  if (tail) {
    __syncthreads();
    for (int k = tid; k < K; k += THREADS) {
      if (t.id[k] < 0) continue;
      const uint32_t bit = 1u << (t.id[k] & 31);
      if (atomicOr(&named[t.id[k] >> 5], bit) & bit) t.twice = 1;
    }
    __syncthreads();
  }
  // (the other waves go on with the row; they meet wave 0 at its largest logit)
  if (wave == 0) {
    weigh_teacher(a, row, lane, u0, t, P, kl);
    if (lane < K) t.z[lane] = z0;
    if (tail) {
      float m = kNegInf;
      for (int k = lane; k < K; k += 64) m = t.id[k] >= 0 ? fmaxf(m, t.z[k]) : m;
      m = max64(m);
      if (lane == 0) t.top = m;
    }
  }
  // named logits are not the rest's
  auto hide = [&](int first) {
    if (!tail) return;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = first + u * THREADS + tid;
      const uint32_t bits =
          v < vectors ? (named[v * N >> 5] >> (v * N & 31)) & ((1u << N) - 1) : 0;
      if (bits) {
#pragma unroll
        for (int i = 0; i < N; ++i) raw[u][i] = bits >> i & 1 ? (T)kNegInf : raw[u][i];
      }
    }
  };
  if (tail && odd < V && named[odd >> 5] >> (odd & 31) & 1) extra = kNegInf;
  float top = kNegInf, rest = 0.f;  // the largest of the rest, and its sum beside that
  auto largest = [&] {
    float m = top;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, (float)raw[u][i]);
    return m;
  };
  auto add = [&](float base) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Vec<T> x = as_loaded(u);
#pragma unroll
      for (int i = 0; i < N; ++i) rest += weight_of((float)x[i], base, a.scale);
      asm volatile("" : "+v"(rest));  // (added here, not all behind the last vector)
    }
  };
  if constexpr (RESIDENT) {
    blank(0);
    hide(0);
    top = fmaxf(largest(), extra);
  } else {
    top = extra;
    rest = weight_of(extra, extra == kNegInf ? 0.f : extra, a.scale);
    for (int first = 0; first < vectors; first += STEP) {
      Vec<T> next[U];
      fetch(next, first + STEP);
      blank(first);
      hide(first);
      const float m = largest();
      // (a thread whose logits are all -infinity has a sum of zero, not NaN)
      const float base = m == kNegInf ? 0.f : m;
      rest *= weight_of(top, base, a.scale);
      top = m;
      add(base);
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
    }
  }
  const float wave_top = max64(top);
  if (lane == 0) part[0][wave] = wave_top;
  __syncthreads();
  float free = part[0][0];  // m'
#pragma unroll
  for (int i = 1; i < W; ++i) free = fmaxf(free, part[0][i]);
  float base = tail ? fmaxf(free, t.top) : free;  // the largest of all
  // (zero in the place of -infinity, so that differences to it are not NaN)
  free = free == kNegInf ? 0.f : free;
  base = base == kNegInf ? 0.f : base;
  if constexpr (RESIDENT) {
    add(free);
    rest += weight_of(extra, free, a.scale);
  } else {
    rest *= weight_of(top, free, a.scale);
  }
  float held = 0.f;  // the named ones' sum beside `base`, each id once
  if (tail) {
    for (int k = tid; k < K; k += THREADS) {
      const int id = t.id[k];
      bool once = id >= 0;
      if (t.twice) {  // (the first entry of an id counts)
        for (int j = 0; j < k; j += 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) once &= t.id[j + i] != id || j + i >= k;
        }
      }
      held += once ? weight_of(t.z[k], base, a.scale) : 0.f;
    }
    held = sum64(held);
  }
  rest = sum64(rest);
  if (lane == 0) {
    part[1][wave] = rest;
    part[2][wave] = held;
  }
  __syncthreads();
  rest = held = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    rest += part[1][i];
    held += part[2][i];
  }
  // f; zero where there is no rest
  const float factor = !tail ? 1.f : rest > 0.f ? weight_of(free, base, a.scale) : 0.f;
  const float sum = fmaf(rest, factor, held);
  // so does a logit that is NaN or +infinity, and a row of -infinity alone
  const bool none = t.none, bad = !none && (t.bad || !(sum > 0.f && sum < kPosInf));
  const float wt = (float)(w * a.temperature);
  const float one = none ? 0.f : bad ? __builtin_nanf("") : wt * (t.whole / sum);
  const float dense = fmaf(one, factor, rest > 0.f ? -wt * (t.rest / rest) : 0.f);
  if constexpr (GRAD) {
    if (none) {
      no_gradient();
    } else {
      for (int first = 0; first < vectors; first += STEP) {
        if (!RESIDENT) fetch(raw, first);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = first + u * THREADS + tid;
          const Vec<T> x = as_loaded(u);
          float g[N];
#pragma unroll
          for (int i = 0; i < N; ++i) g[i] = weight_of((float)x[i], free, a.scale) * dense;
          if (v < vectors) store_vec<T>(grad + (size_t)v * N, g);
        }
      }
      if (odd < V) grad[odd] = (T)(weight_of(extra, free, a.scale) * dense);
    }
  }
  // an element that several entries name has the mass of all of them.  (Where the bits tell that
  // none is, its own: 4096 x 65536 bf16, 64 entries, 225 us -> 207.)
  auto mass_of = [&](int k) {
    if (tail && !t.twice) return (float)t.mass[k];
    const int id = t.id[k];
    double m = 0;
    for (int j = 0; j < K8; j += 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (t.id[j + i] == id) m += t.mass[j + i];
    }
    return (float)m;
  };
  if (GRAD && !none) {
    // (the first entries' masses while the stores are on their way)
    const float mass0 = tid < K && t.id[tid] >= 0 ? mass_of(tid) : 0.f;
    // the dense stores have arrived before a named element is written anew
    drain_memory();
    __syncthreads();
    for (int k = tid; k < K; k += THREADS)
      if (t.id[k] >= 0)
        store_named(grad, t.id[k], t.z[k], wt * (k == tid ? mass0 : mass_of(k)), base, a.scale, one);
  }
  if (a.stats) {
    float* st = a.stats + row * (kDistillStats + K);
    for (int k = tid; k < K; k += THREADS)
      st[kDistillStats + k] = t.id[k] >= 0 ? wt * mass_of(k) : 0.f;
    if (tid == 0) {
      st[0] = base;
      st[1] = one;
      st[2] = free;
      st[3] = dense;
    }
  }
  if (wave == 0) {
    // the student's part of the loss: sum p_k (z_k - base) / T, and its sums' logarithms
    for (int k = lane; k < K; k += 64)
      if (t.mass[k] > 0) kl -= t.mass[k] * (((double)t.z[k] - base) * a.per);
    kl = sum64(kl);
    if (lane == 0) {
      const double lower = tail ? ((double)free - base) * a.per : 0.0;  // (m' - max z) / T
      const double all = (double)rest * factor + held;                  // S
      const double r = tail ? fmax(0.0, 1.0 - P) : 0.0;
      kl += P * log(all);
      if (r > 0) kl += r * (log(r) - (lower + log((double)rest)) + log(all));
      a.loss[row] = none ? 0.f
                    : bad ? __builtin_nanf("")
                          : (float)(w * a.temperature * a.temperature * kl);
    }
  }
}

// The gradient from what the forward pass saved: a workgroup takes a part of a row.
template <typename T, int U>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a, int parts) {
  constexpr int N = kVec<T>, SPAN = U * 256;
  const int tid = threadIdx.x;
  // (the last rows first: the forward pass has just read them)
  const size_t row = (gridDim.x - 1 - blockIdx.x) / parts;
  const int part = (int)(blockIdx.x % parts), first = part * SPAN;
  const int V = a.vocabulary, K = a.top;
  // the last part has the odd values behind the row's whole vectors
  const int vectors = V / N, odd = part == parts - 1 ? vectors * N + tid : V;
  const float up = a.upstream[row];
  const float* st = a.stats + row * (kDistillStats + K);
  // (the stats of a row without weight are not there; one without a teacher has no factors)
  bool live = up != 0.f && (!a.weights || a.weights[row] != 0.f);
  if (live) live = st[1] != 0.f;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  T* grad = reinterpret_cast<T*>(a.grad) + row * a.grad_stride;
  auto store = [&](int u, const float (&g)[N]) {
    const int v = first + u * 256 + tid;
    if (v < vectors) store_vec<T>(grad + (size_t)v * N, g);
  };
  if (!live) {
    const float zero[N] = {};
#pragma unroll
    for (int u = 0; u < U; ++u) store(u, zero);
    if (odd < V) grad[odd] = (T)0.f;
    return;
  }
  Vec<T> raw[U];
  if (vectors > 0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      raw[u] = load_vec<T, true>(z + (size_t)min(first + u * 256 + tid, vectors - 1) * N);
  }
  const float base = st[0], one = st[1] * up, free = st[2], dense = st[3] * up;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = weight_of((float)raw[u][i], free, a.scale) * dense;
    store(u, g);
  }
  if (odd < V) grad[odd] = (T)(weight_of((float)z[odd], free, a.scale) * dense);
  drain_memory();
  __syncthreads();
  const int last = part == parts - 1 ? V : (first + SPAN) * N;
  for (int k = tid; k < K; k += 256) {
    const int id = teacher_id(a, row * K + k);
    if (id >= first * N && id < last)
      store_named(grad, id, (float)z[id], st[kDistillStats + k] * up, base, a.scale, one);
  }
}

template <typename T, bool GRAD, int THREADS, int U, bool RESIDENT>
static void launch_row(const DistillArgs& a, int rows, hipStream_t stream) {
  const size_t lds = a.total ? ((size_t)a.vocabulary + 31) / 32 * 4 : 0;
  hipLaunchKernelGGL((distill_kernel<T, GRAD, THREADS, U, RESIDENT>), dim3(rows), dim3(THREADS), lds,
                     stream, a);
}

// With the gradient, rows that fit are kept in registers.  The loss alone streams its rows: it
// needs each logit once, and rows kept in registers took 17.3 us instead of 14.2 at 64 x
// 131077 bf16, 175 instead of 122 at 2000 x 131077, 5.6 instead of 5.4 at 64 x 8192.
//
// Threads: a row's start and end (its first loads, the teacher, the sums over its waves) take
// what a row of any length takes, so short rows are taken by fewer threads and more of them
// at once; but not where all rows are in flight by then (512: two of 512 threads a CU).
// us, 512 threads -> 256, loss and gradient:
//   bf16 4096 x  8192  59.7 ->  39.4   1024 x  8192  20.9 -> 15.1    256 x 8192  10.1 -> 10.0
//        4096 x 32003 143.1 -> 123.9   1024 x 32003  39.7 -> 35.0    512 x 32003 21.7 -> 23.4
//        4096 x 65536 201.5 -> 221.4
//   fp32 4096 x 16384 112.7 -> 106.5   4096 x 32003 209.9 -> 221.7
// and the loss alone: bf16 4096 x 8192 37.6 -> 25.0, 4096 x 32003 81.9 -> 72.0, 4096 x 65536
// 100.6 -> 103.0.  The longest rows that fit, and longer ones, take 1024 threads: 512 -> 1024,
// bf16 4096 x 131077 591 -> 562, 64 x 131077 31.8 -> 28.8, 64 x 200000 50.9 -> 41.0, 512 x 200000
// 115 -> 119, fp32 2048 x 131077 682 -> 643; the loss alone 237 -> 301 at bf16 4096 x 131077.
template <typename T>
static hipError_t launch_distill_t(const DistillArgs& a, int rows, hipStream_t stream) {
  const int vectors = a.vocabulary / kVec<T>;
  const bool narrow = vectors <= 16 * 256 && rows > 512;
  if (!a.grad && narrow)
    launch_row<T, false, 256, 4, false>(a, rows, stream);
  else if (!a.grad)
    launch_row<T, false, 512, 4, false>(a, rows, stream);
  else if (narrow && vectors <= 4 * 256)
    launch_row<T, true, 256, 4, true>(a, rows, stream);
  else if (narrow && vectors <= 8 * 256)
    launch_row<T, true, 256, 8, true>(a, rows, stream);
  else if (narrow)
    launch_row<T, true, 256, 16, true>(a, rows, stream);
  else if (vectors <= 4 * 512)
    launch_row<T, true, 512, 4, true>(a, rows, stream);
  else if (vectors <= 8 * 512)
    launch_row<T, true, 512, 8, true>(a, rows, stream);
  else if (vectors <= 16 * 512)
    launch_row<T, true, 512, 16, true>(a, rows, stream);
  else if (vectors <= 16 * 1024)
    launch_row<T, true, 1024, 16, true>(a, rows, stream);
  else
    launch_row<T, true, 1024, 4, false>(a, rows, stream);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_distill_bwd_t(const DistillArgs& a, int rows, hipStream_t stream) {
  constexpr int U = 4, SPAN = U * 256;
  const int parts = std::max(1, (a.vocabulary / kVec<T> + SPAN - 1) / SPAN);
  hipLaunchKernelGGL((distill_bwd_kernel<T, U>), dim3((unsigned)rows * parts), dim3(256), 0, stream,
                     a, parts);
  return hipGetLastError();
}

hipError_t launch_distill(const void* logits, long long stride, const void* teacher,
                          bool teacher_f32, const void* ids, bool ids64, const float* total,
                          const float* weights, bool f32, int rows, int vocabulary, int top,
                          double temperature, float* loss, float* stats, void* grad,
                          long long grad_stride, hipStream_t stream) {
  const DistillArgs a{logits, teacher, ids, total, weights, nullptr, grad, loss, stats, stride,
                      grad_stride, vocabulary, top, (float)(1.4426950408889634 / temperature),
                      temperature, 1.0 / temperature, teacher_f32, ids64};
  return f32 ? launch_distill_t<float>(a, rows, stream) : launch_distill_t<bf16>(a, rows, stream);
}

hipError_t launch_distill_bwd(const void* logits, long long stride, const void* ids, bool ids64,
                              const float* weights, const float* stats, const float* upstream,
                              bool f32, int rows, int vocabulary, int top, double temperature,
                              void* grad, long long grad_stride, hipStream_t stream) {
  const DistillArgs a{logits, nullptr, ids, nullptr, weights, upstream, grad, nullptr,
                      const_cast<float*>(stats), stride, grad_stride, vocabulary, top,
                      (float)(1.4426950408889634 / temperature), temperature,
                      1.0 / temperature, false, ids64};
  return f32 ? launch_distill_bwd_t<float>(a, rows, stream)
             : launch_distill_bwd_t<bf16>(a, rows, stream);
}

}  // namespace mf
