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
// With e_j = exp((z_j - max z) / T), S = sum e and S' = sum of e over the j that are
// not named, every dense element is e_j times one factor of its row,
//   w T ((P + r) / S - r / S'),
// and the K named ones are written anew, w T (e_j (P + r) / S - p).  S' is summed by
// itself, through one bit per logit in LDS: as a difference S - sum of named e it
// would lose what a confident student leaves beyond the teacher's entries.
//
// Exponentials of logits and their sums are fp32 (each thread adds at most a few
// hundred); the K masses, 1 - P and the few logarithms of a row are 64-bit, since
// they cancel: at log q = -20 and a loss of 1 the fp32 terms alone would cost 1e-6.
//
// Bound: memory, one read of the logits and one write of the gradient.  A workgroup
// of 1024 takes a row.  Rows of up to 16 vectors a thread stay in registers between
// the maximum, the sum and the gradient; longer ones are read again.
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
  double temperature;
  bool teacher_f32, ids64;
};

constexpr int kDistillThreads = 1024;

__device__ __forceinline__ int teacher_id(const DistillArgs& a, size_t at) {
  const long long id = a.ids64 ? reinterpret_cast<const long long*>(a.ids)[at]
                               : (long long)reinterpret_cast<const int32_t*>(a.ids)[at];
  return id >= 0 && id < a.vocabulary ? (int)id : -1;
}

__device__ __forceinline__ double sum64d(double x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
  return x;
}

// exp((z - top) / T).  The difference first: a product of the type's lowest value
// with `scale` would be infinite, and a row of nothing else not uniform.
__device__ __forceinline__ float weight_of(float z, float top, float scale) {
  return fast_exp2((z - top) * scale);
}

// The named elements of a row's gradient: one thread each, after the dense ones.
template <typename T>
__device__ __forceinline__ void store_named(T* grad, int id, float z, float mass, float top,
                                            float scale, float factor, float w) {
  grad[id] = (T)fmaf(weight_of(z, top, scale), factor, -w * mass);
}

// LOSS: the loss (and with `stats` what the backward needs); GRAD: the gradient of
// the weighted loss.  U: vectors a thread has in flight; RESIDENT: they are the row.
template <typename T, bool GRAD, int U, bool RESIDENT, bool TAIL>
__global__ __launch_bounds__(kDistillThreads) void distill_kernel(DistillArgs a) {
  constexpr int N = kVec<T>, W = kDistillThreads / 64;
  extern __shared__ uint32_t named[];  // a bit per logit, where the total is known
  __shared__ int id_of[kDistillMostTop];
  __shared__ float z_of[kDistillMostTop], mass_of[kDistillMostTop];
  __shared__ float part[3][W];
  __shared__ float row_factors[3];  // w T (P + r) / S, the dense factor, w T
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x;
  const int V = a.vocabulary, K = a.top;
  const float w = a.weights ? a.weights[row] : 1.f;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  T* grad = GRAD ? reinterpret_cast<T*>(a.grad) + row * a.grad_stride : nullptr;
  const int vectors = (V + N - 1) / N;
  if (w == 0.f) {  // whatever the row holds
    if (tid == 0) a.loss[row] = 0.f;
    if constexpr (GRAD) {
      const float zero[N] = {};
      for (int v = tid; v < vectors; v += kDistillThreads)
        store_row<T, TAIL, true>(grad, v * N, V, zero);
    }
    return;
  }
  const bool tail = a.total != nullptr;
  // the first vectors are on their way while the teacher's entries are looked at
  Vec<T> raw[U];
  auto fetch = [&](int first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = first + u * kDistillThreads + tid;
      raw[u] = load_row<T, TAIL, true>(z, v * N, V, kNegInf);
    }
  };
  fetch(0);
  if (tail)
    for (int i = tid; i < (V + 31) / 32; i += kDistillThreads) named[i] = 0;
  if (tid < K) {
    const int id = teacher_id(a, row * K + tid);
    id_of[tid] = id;
    z_of[tid] = id >= 0 ? (float)z[id] : 0.f;
  }
  __syncthreads();
  if (tail) {
    if (tid < K && id_of[tid] >= 0) atomicOr(&named[id_of[tid] >> 5], 1u << (id_of[tid] & 31));
    __syncthreads();
  }
  // maximum and sums
  float top = kNegInf, rest = 0.f, held = 0.f;  // sums beside `top`, not named and named
  for (int first = 0; first < vectors; first += U * kDistillThreads) {
    if (!RESIDENT && first) fetch(first);
    float m = top;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, (float)raw[u][i]);
    // (a thread whose logits are all -infinity has a sum of zero, not NaN)
    const float base = m == kNegInf ? 0.f : m;
    const float old = weight_of(top, base, a.scale);
    rest *= old;
    held *= old;
    top = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = first + u * kDistillThreads + tid;
      uint32_t bits = 0;
      if (tail && v < vectors)
        bits = (named[v * N >> 5] >> (v * N & 31)) & ((1u << N) - 1);
      float e[N];
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = weight_of((float)raw[u][i], base, a.scale);
      if (bits) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          held += bits >> i & 1 ? e[i] : 0.f;
          rest += bits >> i & 1 ? 0.f : e[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) rest += e[i];
      }
    }
  }
  const float wave_top = max64(top);
  if (lane == 0) part[0][wave] = wave_top;
  __syncthreads();
  float all = part[0][0];
#pragma unroll
  for (int i = 1; i < W; ++i) all = fmaxf(all, part[0][i]);
  const float base = all == kNegInf ? 0.f : all;
  const float mine = weight_of(top, base, a.scale);
  rest = sum64(rest * mine);
  held = sum64(held * mine);
  if (lane == 0) {
    part[1][wave] = rest;
    part[2][wave] = held;
  }
  __syncthreads();
  // the row's few numbers in 64 bits, by one wave
  if (wave == 0) {
    float srest = 0.f, sheld = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      srest += part[1][i];
      sheld += part[2][i];
    }
    const double sum = (double)srest + (double)sheld;
    const double per = 1.0 / a.temperature;
    const double log_sum = log(sum);  // beside the largest logit
    double whole, P = 0, kl = 0;
    bool there = false, bad = !(sum > 0 && sum < __builtin_huge_val());
    auto entry = [&](int k) {
      if (id_of[k] < 0) return -__builtin_huge_val();
      const float t = element(a.teacher, a.teacher_f32, row * K + k);
      bad |= !(t < kPosInf);
      there |= t != kNegInf;
      return (double)t * per;
    };
    if (tail) {
      bad |= !(a.total[row] < kPosInf);
      whole = a.total[row];
    } else {
      double most = -__builtin_huge_val(), s = 0;
      for (int k = lane; k < K; k += 64) most = fmax(most, entry(k));
#pragma unroll
      for (int m = 1; m < 64; m <<= 1) most = fmax(most, __shfl_xor(most, m));
      for (int k = lane; k < K; k += 64)
        s += exp(entry(k) - most);
      // (entries that are all -infinity have no mass, like none at all)
      whole = most == -__builtin_huge_val() ? 0.0 : most + log(sum64d(s));
    }
    for (int k = lane; k < K; k += 64) {
      double mass = 0;
      if (id_of[k] >= 0) {
        const double logp = entry(k) - whole;
        mass = exp(logp);
        if (mass > 0) kl += mass * (logp + log_sum - ((double)z_of[k] - base) * per);
      }
      mass_of[k] = (float)mass;
      P += mass;
    }
    P = sum64d(P);
    kl = sum64d(kl);
    const double r = tail ? fmax(0.0, 1.0 - P) : 0.0;
    if (r > 0) kl += r * (log(r) - log((double)srest / sum));
    // without a teacher's entry no loss and no gradient, whatever the row holds; otherwise a
    // logit, an entry or a total that is NaN or +infinity makes the row NaN, and so does a
    // row of -infinity alone
    const bool none = !tail && !__any(there);
    bad = !none && __any(bad);
    if (lane == 0) {
      const double keep = bad ? __builtin_nan("") : 1.0;
      a.loss[row] = none ? 0.f : (float)(w * a.temperature * a.temperature * kl * keep);
      const double one = none ? 0.0 : (P + r) / sum;
      const double dense = one - (srest > 0.f ? r / srest : 0.0);
      const double wt = w * a.temperature;
      row_factors[0] = (float)(wt * one * keep);
      row_factors[1] = (float)(wt * dense * keep);
      row_factors[2] = (float)wt;
      if (a.stats) {
        float* st = a.stats + row * (kDistillStats + K);
        st[0] = base;
#pragma unroll
        for (int i = 0; i < 3; ++i) st[1 + i] = row_factors[i];
      }
    }
  }
  if (!GRAD && !a.stats) return;
  __syncthreads();
  // an element that several entries name has the mass of all of them
  float mass = 0.f;
  const int id = tid < K ? id_of[tid] : -1;
  if (id >= 0)
    for (int k = 0; k < K; ++k) mass += id_of[k] == id ? mass_of[k] : 0.f;
  if constexpr (!GRAD) {
    if (tid < K) a.stats[row * (kDistillStats + K) + kDistillStats + tid] = mass;
    return;
  }
  const float dense = row_factors[1];
  if (row_factors[0] == 0.f) {  // no teacher: no gradient, whatever the row holds
    const float zero[N] = {};
    for (int v = tid; v < vectors; v += kDistillThreads)
      store_row<T, TAIL, true>(grad, v * N, V, zero);
    return;
  }
  for (int first = 0; first < vectors; first += U * kDistillThreads) {
    if (!RESIDENT) fetch(first);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = first + u * kDistillThreads + tid;
      float g[N];
#pragma unroll
      for (int i = 0; i < N; ++i) g[i] = weight_of((float)raw[u][i], base, a.scale) * dense;
      store_row<T, TAIL, true>(grad, v * N, V, g);
    }
  }
  // the dense stores have arrived before a named element is written anew
  drain_memory();
  __syncthreads();
  if (id >= 0)
    store_named(grad, id, z_of[tid], mass, base, a.scale, row_factors[0], row_factors[2]);
}

// The gradient from what the forward pass saved: a workgroup takes a part of a row.
template <typename T, int U, bool TAIL>
__global__ __launch_bounds__(256) void distill_bwd_kernel(DistillArgs a, int parts) {
  constexpr int N = kVec<T>, span = U * 256 * N;
  const int tid = threadIdx.x;
  const size_t row = blockIdx.x / parts;
  const int first = (int)(blockIdx.x % parts) * span;
  const int V = a.vocabulary, K = a.top;
  const float up = a.upstream[row];
  const float* st = a.stats + row * (kDistillStats + K);
  // (the stats of a row without weight are not there; one without a teacher has no factors)
  bool live = up != 0.f && (!a.weights || a.weights[row] != 0.f);
  if (live) live = st[1] != 0.f;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  T* grad = reinterpret_cast<T*>(a.grad) + row * a.grad_stride;
  if (!live) {
    const float zero[N] = {};
#pragma unroll
    for (int u = 0; u < U; ++u)
      store_row<T, TAIL, true>(grad, first + (u * 256 + tid) * N, V, zero);
    return;
  }
  Vec<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
    raw[u] = load_row<T, TAIL, true>(z, first + (u * 256 + tid) * N, V, kNegInf);
  const float base = st[0], one = st[1] * up, dense = st[2] * up, wt = st[3] * up;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float g[N];
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = weight_of((float)raw[u][i], base, a.scale) * dense;
    store_row<T, TAIL, true>(grad, first + (u * 256 + tid) * N, V, g);
  }
  drain_memory();
  __syncthreads();
  for (int k = tid; k < K; k += 256) {
    const int id = teacher_id(a, row * K + k);
    if (id >= first && id < first + span)
      store_named(grad, id, (float)z[id], st[kDistillStats + k], base, a.scale, one, wt);
  }
}

template <typename T, bool GRAD, int U, bool RESIDENT>
static void launch_row(const DistillArgs& a, int rows, hipStream_t stream) {
  const size_t lds = a.total ? ((size_t)a.vocabulary + 31) / 32 * 4 : 0;
  if (a.vocabulary % kVec<T>)
    hipLaunchKernelGGL((distill_kernel<T, GRAD, U, RESIDENT, true>), dim3(rows),
                       dim3(kDistillThreads), lds, stream, a);
  else
    hipLaunchKernelGGL((distill_kernel<T, GRAD, U, RESIDENT, false>), dim3(rows),
                       dim3(kDistillThreads), lds, stream, a);
}

template <typename T>
static hipError_t launch_distill_t(const DistillArgs& a, int rows, hipStream_t stream) {
  const int per = (a.vocabulary + kVec<T> * kDistillThreads - 1) / (kVec<T> * kDistillThreads);
  if (!a.grad) {
    launch_row<T, false, 4, false>(a, rows, stream);
  } else if (per <= 2) {
    launch_row<T, true, 2, true>(a, rows, stream);
  } else if (per <= 4) {
    launch_row<T, true, 4, true>(a, rows, stream);
  } else if (per <= 8) {
    launch_row<T, true, 8, true>(a, rows, stream);
  } else if (per <= 16) {
    launch_row<T, true, 16, true>(a, rows, stream);
  } else {
    launch_row<T, true, 4, false>(a, rows, stream);
  }
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_distill_bwd_t(const DistillArgs& a, int rows, hipStream_t stream) {
  constexpr int U = 4, span = U * 256 * kVec<T>;
  const int parts = (a.vocabulary + span - 1) / span;
  if (a.vocabulary % kVec<T>)
    hipLaunchKernelGGL((distill_bwd_kernel<T, U, true>), dim3((unsigned)rows * parts), dim3(256), 0,
                       stream, a, parts);
  else
    hipLaunchKernelGGL((distill_bwd_kernel<T, U, false>), dim3((unsigned)rows * parts), dim3(256),
                       0, stream, a, parts);
  return hipGetLastError();
}

hipError_t launch_distill(const void* logits, long long stride, const void* teacher,
                          bool teacher_f32, const void* ids, bool ids64, const float* total,
                          const float* weights, bool f32, int rows, int vocabulary, int top,
                          double temperature, float* loss, float* stats, void* grad,
                          long long grad_stride, hipStream_t stream) {
  const DistillArgs a{logits, teacher, ids, total, weights, nullptr, grad, loss, stats, stride,
                      grad_stride, vocabulary, top, (float)(1.4426950408889634 / temperature),
                      temperature, teacher_f32, ids64};
  return f32 ? launch_distill_t<float>(a, rows, stream) : launch_distill_t<bf16>(a, rows, stream);
}

hipError_t launch_distill_bwd(const void* logits, long long stride, const void* ids, bool ids64,
                              const float* weights, const float* stats, const float* upstream,
                              bool f32, int rows, int vocabulary, int top, double temperature,
                              void* grad, long long grad_stride, hipStream_t stream) {
  const DistillArgs a{logits, nullptr, ids, nullptr, weights, upstream, grad, nullptr,
                      const_cast<float*>(stats), stride, grad_stride, vocabulary, top,
                      (float)(1.4426950408889634 / temperature), temperature, false, ids64};
  return f32 ? launch_distill_bwd_t<float>(a, rows, stream)
             : launch_distill_bwd_t<bf16>(a, rows, stream);
}

}  // namespace mf
