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
// Bound: memory.  A row belongs to 16, 64, 256 or 512 lanes by its width, each lane holding
// up to kNormMostVectors vectors of 16 bytes of it.  The backward's workgroups take rows in
// a grid-wide stride and keep the sums of dw and db for their own columns in registers, with
// the next two rows in flight; what each workgroup has at the end is written once and added
// by a second launch in workgroup order.  Of few rows the sums are taken by workgroups of
// the same launch, which read the rows again by columns.  No atomics: the same bits every
// time.
//
// Measured, 32768 x 1024 bf16 (64 MiB a tensor, what the last pass left in the cache
// included): forward 30 us (4.5 TB/s read and written), backward 36 (5.6), its second launch
// 4.0; 8192 x 4096 bf16: 28, 36 and 4.1; 999 x 771 fp32: 3.8 and 10.8 (one launch).
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
template <typename T, Edge E>
__device__ __forceinline__ void load_param(const void* p, bool f32, const RowPlace<T, E>& at,
                                           float (&w)[kVec<T>]) {
  constexpr int N = kVec<T>;
  if (f32 == (N == 4)) {
    const Vec<T> v = at.load(reinterpret_cast<const T*>(p));
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = (float)v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      w[i] = reinterpret_cast<const float*>(p)[E == EDGE_SHORT ? min(i, at.dim - 1) : at.at + i];
  }
}
template <typename T, Edge E, int C>
__device__ __forceinline__ void load_params(const void* p, bool f32, const RowPlace<T, E> (&at)[C],
                                            float (&w)[C][kVec<T>]) {
#pragma unroll
  for (int c = 0; c < C; ++c) load_param<T, E>(p, f32, at[c], w[c]);
}

// (Two rows a group of lanes, for more loads in flight, measured 30 us against 30 at 32768 x
// 1024 bf16 and 3.8 against 3.0 at 64 x 1024.)
template <typename T, int L, int C, Edge E>
__global__ __launch_bounds__(L > 64 ? L : 256) void norm_kernel(NormArgs a) {
  constexpr int N = kVec<T>, R = L > 64 ? 1 : 256 / L;
  __shared__ float part[2][L > 64 ? L / 64 : 1];
  const int lane = threadIdx.x % L;
  const int row = blockIdx.x * R + threadIdx.x / L;
  if (R > 1 && row >= a.rows) return;
  const T* x = reinterpret_cast<const T*>(a.x) + (size_t)row * a.x_stride;
  RowPlace<T, E> at[C];
  Vec<T> raw[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    at[c] = RowPlace<T, E>(c * L + lane, a.dim);
    raw[c] = at[c].load(x);
  }
  float w[C][N], b[C][N];
  load_params<T, E, C>(a.weight, a.param_f32, at, w);
  if (a.bias) load_params<T, E, C>(a.bias, a.param_f32, at, b);
  // sum over the row of f(value)
  auto sum = [&](auto f, float* lds) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float y = f((float)raw[c][i]);
        v += at[c].mine(i) ? y : 0.f;
      }
      s += at[c].any() ? v : 0.f;
    }
    return row_sum<L>(s, lds);
  };
  const float mean = a.center ? sum([](float v) { return v; }, part[0]) * a.inv_dim : 0.f;
  const float square = sum([mean](float v) { return (v - mean) * (v - mean); }, part[1]);
  const float rstd = rsqrtf(fmaf(square, a.inv_dim, a.eps));
  T* y = reinterpret_cast<T*>(a.y) + (size_t)row * a.dim;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      o[i] = ((float)raw[c][i] - mean) * rstd * w[c][i];
      if (a.bias) o[i] += b[c][i];
    }
    at[c].store(y, o);
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
  float* partials;  // [row_blocks][2][dim], or null
  void* dweight;    // of a launch that sums over the rows itself, or null
  void* dbias;
  long long x_stride, dy_stride;
  int rows, dim, row_blocks;
  float inv_dim;
  bool center, param_f32;
};

__device__ __forceinline__ void store_param(void* p, bool f32, int i, float x) {
  if (f32)
    reinterpret_cast<float*>(p)[i] = x;
  else
    reinterpret_cast<bf16*>(p)[i] = (bf16)x;
}

// dweight and dbias of 8 vectors of columns, by a workgroup that goes through all rows: 64
// groups of 8 lanes with every 64th row each.  `lds`: [8][8 N][2].
constexpr int kColumnLanes = 8;

template <typename T, Edge E>
__device__ __forceinline__ void sum_columns(const NormBwdArgs& a, int block, float* lds) {
  constexpr int N = kVec<T>, L = kColumnLanes, G = 512 / L, AHEAD = 4;
  const int lane = threadIdx.x % L, group = threadIdx.x / L, wave = threadIdx.x >> 6;
  const bool first = (threadIdx.x & 63) < L;  // of the wave's groups
  const RowPlace<T, E> at(block * L + lane, a.dim);
  float dw[N] = {}, db[N] = {};
  for (int r0 = group; r0 < a.rows; r0 += G * AHEAD) {
    Vec<T> x[AHEAD], dy[AHEAD];
    float2 st[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const int r = min(r0 + G * j, a.rows - 1);
      st[j] = a.stats[r];
      x[j] = at.load(reinterpret_cast<const T*>(a.x) + (size_t)r * a.x_stride);
      dy[j] = at.load(reinterpret_cast<const T*>(a.dy) + (size_t)r * a.dy_stride);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (r0 + G * j >= a.rows) break;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (float)dy[j][i];
        dw[i] = fmaf(d, ((float)x[j][i] - st[j].x) * st[j].y, dw[i]);
        db[i] += d;
      }
    }
  }
  float* mine = lds + (wave * L + lane) * N * 2;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    // the wave's groups: lanes 8, 16 and 32 apart
    dw[i] += dpp<0x128>(dw[i]);
    db[i] += dpp<0x128>(db[i]);
    dw[i] = halves_sum(rows16_sum(dw[i]));
    db[i] = halves_sum(rows16_sum(db[i]));
    if (first) {
      mine[2 * i] = dw[i];
      mine[2 * i + 1] = db[i];
    }
  }
  __syncthreads();
  if (wave > 0 || !first || !at.any()) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float w = 0.f, b = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      w += lds[((k * L + lane) * N + i) * 2];
      b += lds[((k * L + lane) * N + i) * 2 + 1];
    }
    if (!at.mine(i)) continue;
    if (a.dweight) store_param(a.dweight, a.param_f32, at.at + i, w);
    if (a.dbias) store_param(a.dbias, a.param_f32, at.at + i, b);
  }
}

// Waves a SIMD that the registers are held to: two workgroups a CU, one for the rows of most
// registers a lane.
template <typename T, int L, int C>
constexpr int kNormBwdWaves = C * kVec<T> > (L < 512 ? 16 : 8) ? 2 : 4;

template <typename T, int L, int C, Edge E>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(kNormBwdWaves<T, L, C>)))
void norm_bwd_kernel(NormBwdArgs a) {
  constexpr int N = kVec<T>, R = 512 / L, W = L > 64 ? L / 64 : 1;
  // rows in flight beside the one that is computed, as the registers have room
  constexpr int AHEAD = C * N <= 16 ? 2 : 0, SLOTS = AHEAD ? AHEAD : 1;
  extern __shared__ float lds[];  // the workgroup's sums, or sum_columns'
  __shared__ float part[2][2][8];
  if ((int)blockIdx.x >= a.row_blocks) return sum_columns<T, E>(a, blockIdx.x - a.row_blocks, lds);
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  RowPlace<T, E> at[C];
#pragma unroll
  for (int c = 0; c < C; ++c) at[c] = RowPlace<T, E>(c * L + lane, a.dim);
  // the weights stay in registers, but for the rows of most registers a lane: from the cache
  constexpr bool HOLD = C * N <= 16;
  float held[HOLD ? C : 1][N], dw[C][N], db[C][N];
  if constexpr (HOLD) load_params<T, E, C>(a.weight, a.param_f32, at, held);
  auto weights = [&](int c, float (&w)[N]) {
    if constexpr (HOLD) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = held[c][i];
    } else {
      load_param<T, E>(a.weight, a.param_f32, at[c], w);
    }
  };
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) dw[c][i] = db[c][i] = 0.f;
  const int step = a.row_blocks * R;
  Vec<T> xr[SLOTS][C], gr[SLOTS][C];
  float2 st[SLOTS];
  auto fetch = [&](int n, int first) {  // (a row beyond the last is read again, not used)
    const int r = min(first + group, a.rows - 1);
    const T* x = reinterpret_cast<const T*>(a.x) + (size_t)r * a.x_stride;
    const T* g = reinterpret_cast<const T*>(a.dy) + (size_t)r * a.dy_stride;
    st[n] = a.stats[r];
#pragma unroll
    for (int c = 0; c < C; ++c) xr[n][c] = at[c].load(x);
#pragma unroll
    for (int c = 0; c < C; ++c) gr[n][c] = at[c].load(g);
  };
  int turn = 0;
  auto compute = [&](int n, int first) {
    if (!AHEAD) fetch(n, first);
    const int row = first + group;
    const bool live = R == 1 || row < a.rows;
    const float mean = st[n].x, rstd = st[n].y;
    Vec<T> x[C], dy[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      x[c] = xr[n][c];
      dy[c] = gr[n][c];
    }
    if (AHEAD) fetch(n, first + AHEAD * step);
    turn ^= 1;
    float sg = 0.f, sgh = 0.f;
    if (live) {
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float vg = 0.f, vgh = 0.f, w[N];
        weights(c, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float d = (float)dy[c][i], h = ((float)x[c][i] - mean) * rstd;
          dw[c][i] = fmaf(d, h, dw[c][i]);
          db[c][i] += d;
          const float g = at[c].mine(i) ? d * w[i] : 0.f;
          vg += g;
          vgh = fmaf(g, h, vgh);
        }
        sg += at[c].any() ? vg : 0.f;
        sgh += at[c].any() ? vgh : 0.f;
      }
    }
    if (!a.dx) return;
    if constexpr (L == 16) {
      sg = sum16(sg);
      sgh = sum16(sgh);
    } else {
      sg = sum64(sg);
      sgh = sum64(sgh);
    }
    if constexpr (W > 1) {
      // (two sets of sums in turn: one barrier a row)
      if ((threadIdx.x & 63) == 0) {
        part[turn][0][threadIdx.x >> 6] = sg;
        part[turn][1][threadIdx.x >> 6] = sgh;
      }
      __syncthreads();
      sg = sgh = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        sg += part[turn][0][group * W + i];
        sgh += part[turn][1][group * W + i];
      }
    }
    if (!live) return;
    sg = a.center ? sg * a.inv_dim : 0.f;
    sgh *= a.inv_dim;
    T* dx = reinterpret_cast<T*>(a.dx) + (size_t)row * a.dim;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      // (the row as it was loaded: what the first pass made of it would take twice its registers)
      u32x4 xs = __builtin_bit_cast(u32x4, x[c]), ds = __builtin_bit_cast(u32x4, dy[c]);
      asm volatile("" : "+v"(xs), "+v"(ds));
      const Vec<T> xv = __builtin_bit_cast(Vec<T>, xs), dv = __builtin_bit_cast(Vec<T>, ds);
      float o[N], w[N];
      weights(c, w);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float h = ((float)xv[i] - mean) * rstd;
        o[i] = rstd * fmaf((float)dv[i], w[i], -fmaf(h, sgh, sg));
      }
      at[c].store(dx, o);
    }
  };
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) fetch(n, blockIdx.x * R + n * step);
  for (int first = blockIdx.x * R; first < a.rows; first += SLOTS * step) {
#pragma unroll
    for (int n = 0; n < SLOTS; ++n)
      if (first + n * step < a.rows) compute(n, first + n * step);
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
  auto store_sums = [&](float* to, const RowPlace<T, E>& at, const float (&x)[N]) {
    if (!at.any()) return;
    if constexpr (E == EDGE_WHOLE) {
#pragma unroll
      for (int i = 0; i < N; i += 4)
        *reinterpret_cast<RowVec<float>::U*>(to + at.at + i) =
            RowVec<float>::U{x[i], x[i + 1], x[i + 2], x[i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at.mine(i)) to[at.at + i] = x[i];
    }
  };
  constexpr int G = R > 8 ? 8 : R;  // groups of lanes with sums of their own
  if constexpr (G == 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      store_sums(out, at[c], dw[c]);
      store_sums(out + a.dim, at[c], db[c]);
    }
    return;
  }
  // (a value's lanes side by side: by columns, lanes would be N values apart and meet in a
  // bank eight at a time)
  auto slot = [&](int c, int i, int lane) { return (c * N + i) * L + lane; };
  constexpr int HALF = C * N * L;
  for (int g = 0; g < G; ++g) {
    if ((int)(L == 16 ? threadIdx.x >> 6 : group) == g && (L > 16 || (threadIdx.x & 63) < 16)) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int k = slot(c, i, lane);
          lds[k] = (g ? lds[k] : 0.f) + dw[c][i];
          lds[HALF + k] = (g ? lds[HALF + k] : 0.f) + db[c][i];
        }
    }
    __syncthreads();
  }
  for (int v = threadIdx.x; v < C * L; v += 512) {
    const RowPlace<T, E> place(v, a.dim);
    float w[N], b[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w[i] = lds[slot(v / L, i, v % L)];
      b[i] = lds[HALF + slot(v / L, i, v % L)];
    }
    store_sums(out, place, w);
    store_sums(out + a.dim, place, b);
  }
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
  if (out) store_param(out, f32, at, s);
}

// Lanes and vectors a row by its width (in vectors): the fewest lanes, so that sums cross the
// fewest, as long as a lane's vectors leave the registers for enough rows.  32768 rows of
// bf16, forward + backward us, taken and with the next more lanes: 128 wide, 16 lanes 6.2 + 12.8,
// 64 lanes 11.3 + 19.8; 1024 wide, 64 lanes 25.3 + 40.3, 256 lanes 35.2 + 50.6; 2048 wide, 256
// lanes 43.3 + 82.8, 512 lanes 67.7 + 87.0.  Up to 4096 rows they differ by 3 us at most.
struct NormShape {
  int lanes, vectors;
};
static NormShape norm_shape(int vectors) {
  if (vectors <= 16) return {16, 1};
  if (vectors <= 64) return {64, 1};
  if (vectors <= 128) return {64, 2};
  if (vectors <= 256) return {256, 1};
  for (int c = 1; c < kNormMostVectors; c *= 2)
    if (vectors <= 512 * c) return {512, c};
  return {512, kNormMostVectors};
}

// Workgroups of the backward: as many as 256 CUs hold at once (two each, or one of the most
// registers), fewer where that leaves them less than two rows a group of lanes.
static int norm_bwd_blocks(int rows, int dim, bool f32) {
  const int n = f32 ? 4 : 8;
  const NormShape s = norm_shape((dim + n - 1) / n);
  const long long per = 2ll * (512 / s.lanes);
  const int most = s.vectors * n > (s.lanes < 512 ? 16 : 8) ? 256 : 512;
  return (int)std::min<long long>(most, std::max<long long>(1, (rows + per - 1) / per));
}

// Rows that are few enough for the workgroups of sum_columns to read again instead of a
// second launch over the others' sums.  A workgroup of theirs goes through all rows, so their
// time grows with the rows; a second launch and its workspace cost the host 5 to 7 us a pass
// (forward and backward through autograd, 999 x 771 fp32: 70 us, with one launch 64; in the
// caller's thread 34 and 29; every size up to 1024 rows is as much below).  On the card, the
// backward pass alone, us, two launches -> one:
//              bf16 256 rows   768 rows       1024 rows      1536 rows       fp32 1024 rows
//    256 wide    7.2 ->  4.9    7.9 ->  6.9    8.1 ->  7.8    8.8 ->  9.8     6.8 ->  5.9
//   1024 wide    9.7 ->  5.1   10.5 ->  7.1   10.7 ->  8.1   11.5 -> 15.8     8.1 -> 10.7
//   2048 wide    7.6 ->  5.1    9.7 -> 10.3   10.2 -> 13.9   13.2 -> 18.1    13.4 -> 12.8
//   8192 wide   13.5 ->  7.2   18.1 -> 18.1   19.4 -> 21.5   22.7 -> 28.3    25.9 -> 28.2
// Up to 1024 rows one launch loses at most 3.7 us there, less than it saves the host; beyond,
// it loses more with every row.
static bool norm_small(int rows) { return rows <= kNormFewRows; }

size_t norm_bwd_workspace_bytes(int rows, int dim, bool f32) {
  return norm_small(rows) ? 0 : sizeof(float) * 2 * (size_t)norm_bwd_blocks(rows, dim, f32) * dim;
}

template <typename T, typename F>
static void with_shape(int dim, F&& f) {
  constexpr int N = kVec<T>;
  const NormShape s = norm_shape((dim + N - 1) / N);
  using std::integral_constant;
  auto go = [&](auto l, auto c) {
    if (edge_of<T>(dim) == EDGE_WHOLE)
      f(l, c, integral_constant<Edge, EDGE_WHOLE>{});
    else
      f(l, c, integral_constant<Edge, EDGE_CUT>{});
  };
  auto wide = [&](auto c) { go(integral_constant<int, 512>{}, c); };
  if (edge_of<T>(dim) == EDGE_SHORT)
    f(integral_constant<int, 16>{}, integral_constant<int, 1>{},
      integral_constant<Edge, EDGE_SHORT>{});
  else if (s.lanes == 16)
    go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (s.lanes == 64 && s.vectors == 1)
    go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (s.lanes == 64)
    go(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (s.lanes == 256)
    go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (s.vectors == 1)
    wide(integral_constant<int, 1>{});
  else if (s.vectors == 2)
    wide(integral_constant<int, 2>{});
  else if (s.vectors == 4)
    wide(integral_constant<int, 4>{});
  else if constexpr (N == 4)  // (a bf16 row of kNormMostDim has four)
    wide(integral_constant<int, 8>{});
}

template <typename T>
static hipError_t launch_norm_t(const NormArgs& a, hipStream_t stream) {
  with_shape<T>(a.dim, [&](auto l, auto c, auto edge) {
    constexpr int L = decltype(l)::value;
    constexpr int R = L > 64 ? 1 : 256 / L;
    hipLaunchKernelGGL((norm_kernel<T, L, decltype(c)::value, decltype(edge)::value>),
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
static hipError_t launch_norm_bwd_t(const NormBwdArgs& a, hipStream_t stream) {
  constexpr int N = kVec<T>;
  const bool columns = a.dweight || a.dbias;
  constexpr int S = kColumnLanes * N;  // columns of a workgroup that sums them
  const int blocks = a.row_blocks + (columns ? (a.dim + S - 1) / S : 0);
  with_shape<T>(a.dim, [&](auto l, auto c, auto edge) {
    constexpr int L = decltype(l)::value;
    const size_t lds = columns ? sizeof(float) * 2 * 8 * S
                       : L > 256 || !a.partials ? 0 : sizeof(float) * 2 * decltype(c)::value * N * L;
    hipLaunchKernelGGL((norm_bwd_kernel<T, L, decltype(c)::value, decltype(edge)::value>),
                       dim3(blocks), dim3(512), lds, stream, a);
  });
  return hipGetLastError();
}

hipError_t launch_norm_bwd(const void* x, long long x_stride, const void* weight,
                           const float* stats, const void* dy, long long dy_stride, bool f32,
                           bool param_f32, int rows, int dim, bool center, void* dx, void* dweight,
                           void* dbias, void* workspace, hipStream_t stream) {
  const bool sums = dweight || dbias, small = norm_small(rows);
  const bool partials = sums && !small;
  const int blocks = dx || partials ? norm_bwd_blocks(rows, dim, f32) : 0;
  NormBwdArgs a{x, dy, weight, reinterpret_cast<const float2*>(stats), dx,
                partials ? reinterpret_cast<float*>(workspace) : nullptr,
                small ? dweight : nullptr, small ? dbias : nullptr, x_stride, dy_stride,
                rows, dim, blocks, (float)(1.0 / dim), center, param_f32};
  auto launch = [&] {
    return f32 ? launch_norm_bwd_t<float>(a, stream) : launch_norm_bwd_t<bf16>(a, stream);
  };
  hipError_t e;
  if (small && sums && dx == dy) {  // the columns are read before dx takes dy's place
    a.row_blocks = 0;
    if ((e = launch()) != hipSuccess) return e;
    a.row_blocks = blocks;
    a.dweight = a.dbias = nullptr;
  }
  e = launch();
  if (e != hipSuccess || !partials) return e;
  hipLaunchKernelGGL(norm_reduce_kernel, dim3((2 * dim + 63) / 64), dim3(1024), 0, stream,
                     a.partials, blocks, dim, dweight, dbias, param_f32);
  return hipGetLastError();
}

}  // namespace mf
