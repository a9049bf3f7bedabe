// Layer norm and RMS norm over the last dimension, forward and backward, on gfx950.
//
// Per row of D values, with mu = mean(x) (0 for the RMS norm) and
// rstd = (mean((x - mu)^2) + eps)^-1/2:
//   h = (x - mu) rstd,   y = h w + b.
// The row stays in registers, so the spread is summed from the differences to
// the mean themselves, not from squares less a square, which would lose rows
// whose mean is large beside their spread.  Backward, with g = dy w:
//   dx = rstd (g - mean(g) - h mean(g h))     (mean(g) only for the layer norm)
//   dw = sum over rows of dy h,   db = sum over rows of dy.
// All in fp32, each output rounded once.  (The prologue's per-head norm rounds the
// normalised value before the gain, as the reference's declared types do.)
//
// Bound: memory.  A row belongs to 16 lanes, a wave or a workgroup of 512, by its
// width, each lane holding up to kMostVectors vectors of 16 bytes of it.  The
// backward's workgroups take rows in a grid-wide stride and keep the sums of dw and
// db for their own columns in registers; what each workgroup has at the end is
// written once and added by a second launch in workgroup order: no atomics, the
// same bits every time.
#include <algorithm>

#include "mf_norm.h"
#include "mf_rows.h"

namespace mf {

struct NormArgs {
  const void* x;
  const void* weight;
  const void* bias;  // or null
  void* y;
  float2* stats;     // mean and rstd of every row, or null
  long long x_stride;
  int rows, dim;
  float eps, inv_dim;
  bool center, param_f32;
};

// Sum over the L lanes that share a row; `part` is LDS for one value a wave.
template <int L>
__device__ __forceinline__ float row_sum(float x, float* part) {
  if constexpr (L == 16) return sum16(x);
  x = sum64(x);
  if constexpr (L == 64) return x;
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < L / 64; ++i) s += part[i];
  return s;
}

// The lane's share of a parameter, in its own dtype (uniform branch).
template <typename T, int C, int L, bool TAIL>
__device__ __forceinline__ void load_params(const void* p, bool f32, int lane, int dim,
                                            float (&w)[C][kVec<T>]) {
  constexpr int N = kVec<T>;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const int col = (c * L + lane) * N;
    if (f32 == (N == 4)) {
      const Vec<T> v = load_row<T, TAIL>(reinterpret_cast<const T*>(p), col, dim);
#pragma unroll
      for (int i = 0; i < N; ++i) w[c][i] = (float)v[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) w[c][i] = col + i < dim ? element(p, f32, col + i) : 0.f;
    }
  }
}

template <typename T, int L, int C, bool TAIL>
__global__ __launch_bounds__(L > 64 ? L : 256) void norm_kernel(NormArgs a) {
  constexpr int N = kVec<T>, R = L > 64 ? 1 : 256 / L;
  __shared__ float part[2][L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x % L;
  const int row = blockIdx.x * R + threadIdx.x / L;
  if (L <= 64 && row >= a.rows) return;
  const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.x_stride;
  Vec<T> raw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) raw[c] = load_row<T, TAIL>(x, (c * L + lane) * N, a.dim);
  float w[C][N], b[C][N];
  load_params<T, C, L, TAIL>(a.weight, a.param_f32, lane, a.dim, w);
  if (a.bias) load_params<T, C, L, TAIL>(a.bias, a.param_f32, lane, a.dim, b);
  float mean = 0.f;
  if (a.center) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) s += (float)raw[c][i];
    mean = row_sum<L>(s, part[0]) * a.inv_dim;
  }
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = (float)raw[c][i] - mean;
      if (!TAIL && (c * L + lane) * N >= a.dim) continue;
      if (TAIL && (c * L + lane) * N + i >= a.dim) continue;
      s = fmaf(d, d, s);
    }
  const float rstd = rsqrtf(fmaf(row_sum<L>(s, part[1]), a.inv_dim, a.eps));
  T* y = reinterpret_cast<T*>(a.y) + (size_t)row * a.dim;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i] = ((float)raw[c][i] - mean) * rstd * w[c][i];
      if (a.bias) o[i] += b[c][i];
    }
    store_row<T, TAIL>(y, (c * L + lane) * N, a.dim, o);
  }
  if (a.stats && lane == 0) a.stats[row] = float2{mean, rstd};
}

// ---------------------------------------------------------------------------

struct NormBwdArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const float2* stats;
  void* dx;         // or null
  float* partials;  // [gridDim.x][2][dim], or null
  long long x_stride, dy_stride;
  int rows, dim;
  float inv_dim;
  bool center, param_f32;
};

template <typename T, int L, int C, bool TAIL>
__global__ __launch_bounds__(512) void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int N = kVec<T>, R = 512 / L;
  extern __shared__ float lds[];  // the workgroup's sums [2][dim]
  __shared__ float part[2][2][8];
  const int lane = threadIdx.x % L;
  float w[C][N], dw[C][N], db[C][N];
  load_params<T, C, L, TAIL>(a.weight, a.param_f32, lane, a.dim, w);
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = 0.f;
  // rows of the workgroup: the next one is fetched while one is computed
  const int step = gridDim.x * R;
  int row = blockIdx.x * R + threadIdx.x / L;
  Vec<T> xr[C], gr[C];
  float2 st = {0.f, 0.f};
  auto fetch = [&](int r) {
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)r * a.x_stride;
    const T* g = reinterpret_cast<const T*>(a.dy) + (size_t)r * a.dy_stride;
#pragma unroll
    for (int c = 0; c < C; ++c) xr[c] = load_row<T, TAIL>(x, (c * L + lane) * N, a.dim);
#pragma unroll
    for (int c = 0; c < C; ++c) gr[c] = load_row<T, TAIL>(g, (c * L + lane) * N, a.dim);
    st = a.stats[r];
  };
  if (row < a.rows) fetch(row);
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    float h[C][N], g[C][N], sg = 0.f, sgh = 0.f;
    const float rstd = st.y;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float dy = (float)gr[c][i];
        h[c][i] = ((float)xr[c][i] - st.x) * rstd;
        dw[c][i] = fmaf(dy, h[c][i], dw[c][i]);
        db[c][i] += dy;
        g[c][i] = dy * w[c][i];  // zero past the row's end
        sg += g[c][i];
        sgh = fmaf(g[c][i], h[c][i], sgh);
      }
    const int next = row + step;
    if (next < a.rows) fetch(next);
    if (!a.dx) continue;
    if constexpr (L > 64) {
      sg = sum64(sg);
      sgh = sum64(sgh);
      if ((threadIdx.x & 63) == 0) {
        part[turn][0][threadIdx.x >> 6] = sg;
        part[turn][1][threadIdx.x >> 6] = sgh;
      }
      __syncthreads();
      sg = sgh = 0.f;
#pragma unroll
      for (int i = 0; i < L / 64; ++i) {
        sg += part[turn][0][i];
        sgh += part[turn][1][i];
      }
    } else {
      sg = row_sum<L>(sg, nullptr);
      sgh = row_sum<L>(sgh, nullptr);
    }
    sg = a.center ? sg * a.inv_dim : 0.f;
    sgh *= a.inv_dim;
    T* dx = reinterpret_cast<T*>(a.dx) + (size_t)row * a.dim;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float o[N];
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] = rstd * (g[c][i] - fmaf(h[c][i], sgh, sg));
      store_row<T, TAIL>(dx, (c * L + lane) * N, a.dim, o);
    }
  }
  if (!a.partials) return;
  // the workgroup's rows, added in the order of its waves
  if constexpr (L == 16) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dw[c][i] = halves_sum(rows16_sum(dw[c][i]));
        db[c][i] = halves_sum(rows16_sum(db[c][i]));
      }
  }
  float* out = a.partials + (size_t)blockIdx.x * 2 * a.dim;
  constexpr int W = L > 64 ? 1 : 8;
  for (int wave = 0; wave < W; ++wave) {
    if (W == 1 || (int)(threadIdx.x >> 6) == wave) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int col = (c * L + lane) * N + i;
          if (col >= a.dim || (L == 16 && (threadIdx.x & 63) >= 16)) continue;
          float* to = W == 1 ? out : lds;
          to[col] = (wave ? lds[col] : 0.f) + dw[c][i];
          to[a.dim + col] = (wave ? lds[a.dim + col] : 0.f) + db[c][i];
        }
    }
    if (W > 1) __syncthreads();
  }
  if (W > 1)
    for (int i = threadIdx.x; i < 2 * a.dim; i += 512) out[i] = lds[i];
}

// dweight and dbias from the workgroups' sums: 64 columns a workgroup, its 16
// waves take 1/16 of the partials each, in order.
__global__ __launch_bounds__(1024) void norm_reduce_kernel(const float* partials, int count,
                                                           int dim, void* dweight, void* dbias,
                                                           bool f32) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = blockIdx.x * 64 + lane;  // of 2 dim
  const int per = (count + 15) / 16, first = wave * per, last = min(count, first + per);
  float s = 0.f;
  if (col < 2 * dim) {
#pragma unroll 8
    for (int i = first; i < last; ++i) s += partials[(size_t)i * 2 * dim + col];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave || col >= 2 * dim) return;
#pragma unroll
  for (int i = 1; i < 16; ++i) s += sums[i][lane];
  void* out = col < dim ? dweight : dbias;
  const int at = col < dim ? col : col - dim;
  if (!out) return;
  if (f32)
    reinterpret_cast<float*>(out)[at] = s;
  else
    reinterpret_cast<bf16*>(out)[at] = (bf16)s;
}

// Lanes and vectors a row by its width (in vectors).
struct NormShape {
  int lanes, vectors;
};
static NormShape norm_shape(int vectors) {
  if (vectors <= 16) return {16, 1};
  for (int c = 1; c <= 4; c *= 2)
    if (vectors <= 64 * c) return {64, c};
  for (int c = 1; c < kNormMostVectors; c *= 2)
    if (vectors <= 512 * c) return {512, c};
  return {512, kNormMostVectors};
}

// Workgroups of the backward: two for each of 256 CUs, fewer where that leaves
// them less than two rows a wave.
static int norm_bwd_blocks(int rows, int dim, bool f32) {
  const int n = f32 ? 4 : 8;
  const NormShape s = norm_shape((dim + n - 1) / n);
  const long long per = 2ll * (512 / s.lanes);
  return (int)std::min<long long>(512, std::max<long long>(1, (rows + per - 1) / per));
}

size_t norm_bwd_workspace_bytes(int rows, int dim, bool f32) {
  return sizeof(float) * 2 * (size_t)norm_bwd_blocks(rows, dim, f32) * dim;
}

template <typename T, typename F>
static void with_shape(int dim, F&& f) {
  constexpr int N = kVec<T>;
  const NormShape s = norm_shape((dim + N - 1) / N);
  const bool tail = dim % N != 0;
  auto go = [&](auto l, auto c) {
    if (tail)
      f(l, c, std::true_type{});
    else
      f(l, c, std::false_type{});
  };
  using std::integral_constant;
  if (s.lanes == 16) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  if (s.lanes == 64) {
    if (s.vectors == 1) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (s.vectors == 2) return go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    return go(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  }
  if (s.vectors == 1) return go(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  if (s.vectors == 2) return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
  if (s.vectors == 4) return go(integral_constant<int, 512>{}, integral_constant<int, 4>{});
  // (a bf16 row of kNormMostDim has four)
  if constexpr (N == 4) go(integral_constant<int, 512>{}, integral_constant<int, 8>{});
}

template <typename T>
static hipError_t launch_norm_t(const NormArgs& a, hipStream_t stream) {
  with_shape<T>(a.dim, [&](auto l, auto c, auto tail) {
    constexpr int L = decltype(l)::value;
    constexpr int R = L > 64 ? 1 : 256 / L;
    hipLaunchKernelGGL((norm_kernel<T, L, decltype(c)::value, decltype(tail)::value>),
                       dim3((a.rows + R - 1) / R), dim3(L > 64 ? L : 256), 0, stream, a);
  });
  return hipGetLastError();
}

hipError_t launch_norm(const void* x, long long x_stride, const void* weight, const void* bias,
                       bool f32, bool param_f32, int rows, int dim, bool center, float eps, void* y,
                       float* stats, hipStream_t stream) {
  const NormArgs a{x, weight, bias, y, reinterpret_cast<float2*>(stats), x_stride, rows, dim, eps,
                   (float)(1.0 / dim), center, param_f32};
  return f32 ? launch_norm_t<float>(a, stream) : launch_norm_t<bf16>(a, stream);
}

template <typename T>
static hipError_t launch_norm_bwd_t(const NormBwdArgs& a, int blocks, hipStream_t stream) {
  with_shape<T>(a.dim, [&](auto l, auto c, auto tail) {
    constexpr int L = decltype(l)::value;
    const size_t lds = L > 64 || !a.partials ? 0 : sizeof(float) * 2 * a.dim;
    hipLaunchKernelGGL((norm_bwd_kernel<T, L, decltype(c)::value, decltype(tail)::value>),
                       dim3(blocks), dim3(512), lds, stream, a);
  });
  return hipGetLastError();
}

hipError_t launch_norm_bwd(const void* x, long long x_stride, const void* weight,
                           const float* stats, const void* dy, long long dy_stride, bool f32,
                           bool param_f32, int rows, int dim, bool center, void* dx, void* dweight,
                           void* dbias, void* workspace, hipStream_t stream) {
  const bool sums = dweight || dbias;
  const int blocks = norm_bwd_blocks(rows, dim, f32);
  const NormBwdArgs a{x, dy, weight, reinterpret_cast<const float2*>(stats), dx,
                      sums ? reinterpret_cast<float*>(workspace) : nullptr, x_stride, dy_stride,
                      rows, dim, (float)(1.0 / dim), center, param_f32};
  hipError_t e = f32 ? launch_norm_bwd_t<float>(a, blocks, stream)
                     : launch_norm_bwd_t<bf16>(a, blocks, stream);
  if (e != hipSuccess || !sums) return e;
  hipLaunchKernelGGL(norm_reduce_kernel, dim3((2 * dim + 63) / 64), dim3(1024), 0, stream,
                     a.partials, blocks, dim, dweight, dbias, param_f32);
  return hipGetLastError();
}

}  // namespace mf
