// Rotary position embeddings in their general form, and the append of new keys
// and values to a paged cache, on gfx950.
//
// Pair i of a head's `rotary_dim` rotated dims -- dims (i, i + rotary_dim / 2) in
// the half layout, (2 i, 2 i + 1) in the interleaved one -- turns by the angle
// a = position * f_i:
//   u' = mu (u cos a - w sin a),   w' = mu (w cos a + u sin a)
// and the other dims pass.  The backward is the transpose: the same with -sin.
// All in fp32 from the tensor dtype, rounded once at the end.  (The prologue of
// mf_prologue.hip rounds every step to the tensor dtype, as the reference's
// declared types do: kernels/rotary.py:7-39.)
//
// Angles.  f_i / 2 pi modulo one turn is a 64-bit fraction, made on the host in
// extended precision (mf_rotary_turns); position * fraction modulo 2^64 drops whole turns exactly,
// so the fraction is good to position * 2^-65 turns at any int32 position.  What is left
// of it beside the nearest quarter turn is rounded to fp32, by at most 2.4e-8 radians
// (pi 2^-27).  Rounded as a fraction of a whole turn, by up to 9.4e-8, it left unit-normal
// values 4.7e-8 off in the mean square instead of 3.6e-8; cos and sin rounded from 64-bit
// angles and separate fp32 operations leave 4.1e-8.
// (An fp32 product is off by position * 2^-24 radians: 0.008 at 131072, twice a
// bf16 rounding.)
//
// The append adds, for every new token of a step's plan, the optional RMS norm
// of each query and key head over its 64 dims (before the rotation), the
// rotation at the token's position, and the store of key and value into the
// token's page and slot.
//
// Bound: memory, one read and one write of every value.  A thread takes units of
// V pairs (two loads of up to 16 bytes): in the half layout both halves of its
// pairs, so no exchange between lanes is needed but the norm's sum, which runs
// over the 32 / V lanes of a head.  A workgroup takes whole tokens, and its
// threads make the tokens' cos and sin in LDS once, for all heads, while the
// first rows are in flight.  8 x 4096 tokens of 16/8 heads of 64 in bf16 (201 MB a
// direction) 35 to 38 us, 5.3 to 5.7 TB/s; the append of 20912 tokens (171 MB) 29 us,
// 5.9; of 64 tokens 4 us, a launch.
#include "mf_paged.h"

namespace mf {

constexpr int kMaxPairs = 128;   // rotary_dim up to 256
constexpr int kTurnTokens = 16;  // tokens of a workgroup at most

struct TurnArgs {
  const void* src[3];             // q, k, v
  void* dst[3];                   // q, k dense; k, v pages when paged
  long long src_stride[3];        // elements between tokens
  PagedStrides pages[2];          // of k, v
  const void* gain[2];
  const int32_t* positions;       // [tokens] or null (token % seq_len)
  const PagedToken* records;      // paged: the plan's tokens
  int tokens, D, half;            // half: pairs that rotate
  int page_size, page_count;
  int heads[3], uph, units, tpb;  // units per head, per token; tokens per workgroup
  int interleaved;
  float eps, magnitude, sign;
  FastDiv div_units, div_uph, div_half, div_len;
  uint64_t turn[kMaxPairs];       // turns per position, 2^-64ths
};

template <typename T, int V> struct TurnVec;
template <> struct TurnVec<bf16, 8> { typedef bf16x8 type; };
template <> struct TurnVec<bf16, 4> { typedef bf16x4 type; };
template <> struct TurnVec<bf16, 1> { typedef bf16 type; };
template <> struct TurnVec<float, 4> { typedef f32x4 type; };
template <> struct TurnVec<float, 1> { typedef float type; };

template <typename T, int V>
__device__ __forceinline__ void widen(const typename TurnVec<T, V>::type& v, float (&x)[V]) {
  if constexpr (V == 1) {
    x[0] = (float)v;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = (float)v[i];
  }
}

template <typename T, int V>
__device__ __forceinline__ typename TurnVec<T, V>::type narrow(const float (&x)[V]) {
  typename TurnVec<T, V>::type v;
  if constexpr (V == 1) {
    v = (T)x[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)x[i];
  }
  return v;
}

// Sum over the 32 / V lanes of a 64-dim head.
template <int V>
__device__ __forceinline__ float head_sum(float x) {
  if constexpr (V == 1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor(x, o);
  } else {
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, false));
    x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, false));
    if constexpr (V == 4)
      x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x141, 0xF, 0xF, false));
  }
  return x;
}

// sin and cos of an angle in 2^-64ths of a turn: the nearest quarter turn is taken out
// in integers, so that what is converted to a float, and rounded, is an angle of at most
// pi / 4 whichever quadrant the angle lies in.
__device__ __forceinline__ void sincos_turns(uint64_t turns, float& s, float& c) {
  const int64_t rest = (int64_t)(turns << 2) >> 2;  // [-2^61, 2^61)
  const uint32_t quarter = (uint32_t)((turns - (uint64_t)rest) >> 62);
  float s0, c0;
  sincospif((float)rest * 0x1p-63f, &s0, &c0);      // (half turns)
  const float x = quarter & 1 ? s0 : c0, y = quarter & 1 ? c0 : s0;
  c = quarter == 1 || quarter == 2 ? -x : x;
  s = quarter >= 2 ? -y : y;
}

template <typename T, int V, int U, bool PAGED>
__global__ __launch_bounds__(256) void turn_rows_kernel(TurnArgs a) {
  typedef typename TurnVec<T, V>::type Vec;
  __shared__ float2 table[kTurnTokens * kMaxPairs];  // [token][pair] (cos, sin) * magnitude
  const int tok0 = blockIdx.x * a.tpb;
  const int total = a.tpb * a.units;
  for (int first = 0; first < total; first += 256 * U) {
    Vec x0[U], x1[U];
    int kind[U], head[U], tl[U], o0[U], o1[U], pair[U];  // pair: first pair, -1 when the unit passes
    bool live[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int idx = first + 256 * j + threadIdx.x;
      tl[j] = fast_div(idx, a.div_units);
      const int rem = idx - tl[j] * a.units;
      int h = fast_div(rem, a.div_uph);
      const int c = rem - h * a.uph;
      live[j] = idx < total && tok0 + tl[j] < a.tokens;
      kind[j] = h < a.heads[0] ? 0 : h < a.heads[0] + a.heads[1] ? 1 : 2;
      h -= kind[j] > 0 ? a.heads[0] : 0;
      h -= kind[j] > 1 ? a.heads[1] : 0;
      head[j] = h;
      const bool turns = kind[j] < 2 && c * V < a.half;
      pair[j] = turns ? c * V : -1;
      o0[j] = turns && !a.interleaved ? c * V : 2 * c * V;
      o1[j] = o0[j] + (turns && !a.interleaved ? a.half : V);
      if (live[j]) {
        const void* base = kind[j] == 0 ? a.src[0] : kind[j] == 1 ? a.src[1] : a.src[2];
        const long long stride = kind[j] == 0 ? a.src_stride[0]
                                              : kind[j] == 1 ? a.src_stride[1] : a.src_stride[2];
        const T* p = reinterpret_cast<const T*>(base) + (long long)(tok0 + tl[j]) * stride +
                     (long long)h * a.D;
        x0[j] = *reinterpret_cast<const Vec*>(p + o0[j]);
        x1[j] = *reinterpret_cast<const Vec*>(p + o1[j]);
      } else {
        x0[j] = Vec{};
        x1[j] = Vec{};
      }
    }
    if (first == 0) {
      __builtin_amdgcn_sched_barrier(0);  // the rows are in flight before the angles are made
      for (int i = threadIdx.x; i < a.tpb * a.half; i += 256) {
        const int t = fast_div(i, a.div_half);
        const int p = i - t * a.half;
        const int tok = min(tok0 + t, a.tokens - 1);
        int pos;
        if constexpr (PAGED) {
          pos = a.records[tok].position;
        } else {
          pos = a.positions ? a.positions[tok] : tok - fast_div(tok, a.div_len) * (int)a.div_len.d;
        }
        float s, c;
        sincos_turns((uint64_t)(int64_t)pos * a.turn[p], s, c);
        table[i] = make_float2(c * a.magnitude, s * a.magnitude * a.sign);
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
      float u[V], w[V];
      widen<T, V>(x0[j], u);
      widen<T, V>(x1[j], w);
      Vec y0 = x0[j], y1 = x1[j];
      if constexpr (PAGED) {
        const void* gain = kind[j] == 0 ? a.gain[0] : a.gain[1];
        if (gain) {  // (the same for a head's lanes)
          float ss = 0.f;
#pragma unroll
          for (int i = 0; i < V; ++i) ss = fmaf(u[i], u[i], fmaf(w[i], w[i], ss));
          const float inv = rsqrtf(head_sum<V>(ss) * (1.f / kD) + a.eps);
          float g0[V], g1[V];
          widen<T, V>(*reinterpret_cast<const Vec*>(reinterpret_cast<const T*>(gain) + o0[j]), g0);
          widen<T, V>(*reinterpret_cast<const Vec*>(reinterpret_cast<const T*>(gain) + o1[j]), g1);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            u[i] *= inv * g0[i];
            w[i] *= inv * g1[i];
          }
          if (kind[j] < 2) {
            y0 = narrow<T, V>(u);
            y1 = narrow<T, V>(w);
          }
        }
      }
      if (pair[j] >= 0) {
        const float2* cs = table + tl[j] * a.half + pair[j];
        float r0[V], r1[V];
        if (V > 1 && a.interleaved) {
          // pairs of neighbours: V / 2 in each vector
#pragma unroll
          for (int i = 0; i + 1 < V; i += 2) {
            const float2 m = cs[i / 2], n = cs[V / 2 + i / 2];
            r0[i] = fmaf(u[i], m.x, -u[i + 1] * m.y);
            r0[i + 1] = fmaf(u[i + 1], m.x, u[i] * m.y);
            r1[i] = fmaf(w[i], n.x, -w[i + 1] * n.y);
            r1[i + 1] = fmaf(w[i + 1], n.x, w[i] * n.y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            r0[i] = fmaf(u[i], cs[i].x, -w[i] * cs[i].y);
            r1[i] = fmaf(w[i], cs[i].x, u[i] * cs[i].y);
          }
        }
        y0 = narrow<T, V>(r0);
        y1 = narrow<T, V>(r1);
      }
      if (!live[j]) continue;
      const int tok = tok0 + tl[j];
      T* dst;
      if (!PAGED || kind[j] == 0) {
        dst = reinterpret_cast<T*>(kind[j] == 0 ? a.dst[0] : a.dst[1]) +
              ((long long)tok * (kind[j] == 0 ? a.heads[0] : a.heads[1]) + head[j]) * a.D;
      } else {
        const PagedToken rec = a.records[tok];
        // (the plan's pages and slots are within its pool; this one may be smaller)
        if ((unsigned)rec.page >= (unsigned)a.page_count || rec.slot >= a.page_size) continue;
        const PagedStrides st = kind[j] == 1 ? a.pages[0] : a.pages[1];
        dst = reinterpret_cast<T*>(kind[j] == 1 ? a.dst[1] : a.dst[2]) + rec.page * st.page +
              rec.slot * st.slot + head[j] * st.head;
      }
      *reinterpret_cast<Vec*>(dst + o0[j]) = y0;
      *reinterpret_cast<Vec*>(dst + o1[j]) = y1;
    }
  }
}

template <typename T, int V, bool PAGED>
static hipError_t launch_turn_v(TurnArgs& a, hipStream_t stream) {
  a.uph = a.D / (2 * V);
  a.units = (a.heads[0] + a.heads[1] + a.heads[2]) * a.uph;
  // One unit a thread, two where a token has more units than a workgroup has threads:
  // the rows in flight come from many workgroups, not from deep loops.  us for one,
  // two and four units: 8 x 4096 tokens of 16/8 heads 35.6, 35.7 and 40.8 (5.7 TB/s;
  // a copy of 1 GiB runs at 5.2), the append of 20912 tokens 34.1, 35.9 and 40.2;
  // 8 x 2048 of 24 heads of 96, 24 rotated (288 units) 34.7, 30.3 and 31.1.
  const int per = a.units > 256 ? 512 : 256;
  a.tpb = per / a.units < 1 ? 1 : per / a.units > kTurnTokens ? kTurnTokens : per / a.units;
  a.div_units = make_fastdiv(a.units);
  a.div_uph = make_fastdiv(a.uph);
  a.div_half = make_fastdiv(a.half < 1 ? 1 : a.half);
  const long long grid = ((long long)a.tokens + a.tpb - 1) / a.tpb;
  if (grid >= (1 << 24)) return hipErrorInvalidConfiguration;  // 2^32 threads
  if (per > 256)
    hipLaunchKernelGGL((turn_rows_kernel<T, V, 2, PAGED>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((turn_rows_kernel<T, V, 1, PAGED>), dim3((unsigned)grid), dim3(256), 0, stream, a);
  return hipGetLastError();
}

// The widest vectors that rotated dims, head dim, strides and addresses allow.
template <bool PAGED>
static hipError_t launch_turn(TurnArgs& a, bool f32, uint64_t addresses, uint64_t strides,
                              hipStream_t stream) {
  const int r = 2 * a.half;
  const int size = f32 ? 4 : 2;
  auto fits = [&](int v) {
    return r % (2 * v) == 0 && a.D % (2 * v) == 0 && strides % v == 0 && addresses % (v * size) == 0;
  };
  if (f32) return fits(4) ? launch_turn_v<float, 4, PAGED>(a, stream)
                          : launch_turn_v<float, 1, PAGED>(a, stream);
  return fits(8)   ? launch_turn_v<bf16, 8, PAGED>(a, stream)
         : fits(4) ? launch_turn_v<bf16, 4, PAGED>(a, stream)
                   : launch_turn_v<bf16, 1, PAGED>(a, stream);
}

static void set_turns(TurnArgs& a, const uint64_t* turns, int rotary_dim, int interleaved,
                      float magnitude) {
  a.half = turns ? rotary_dim / 2 : 0;
  a.interleaved = interleaved;
  a.magnitude = magnitude;
  for (int i = 0; i < a.half; ++i) a.turn[i] = turns[i];
}

hipError_t launch_rotate(const void* q, long long q_stride, const void* k, long long k_stride,
                         const int32_t* positions, const uint64_t* turns, bool f32, int tokens,
                         int seq_len, int Hq, int Hkv, int D, int rotary_dim, int interleaved,
                         float magnitude, bool backward, void* q_out, void* k_out,
                         hipStream_t stream) {
  TurnArgs a = {};
  a.src[0] = q;
  a.src[1] = k;
  a.dst[0] = q_out;
  a.dst[1] = k_out;
  a.src_stride[0] = q_stride;
  a.src_stride[1] = k_stride;
  a.positions = positions;
  a.tokens = tokens;
  a.D = D;
  a.heads[0] = Hq;
  a.heads[1] = Hkv;
  a.sign = backward ? -1.f : 1.f;
  a.div_len = make_fastdiv(seq_len);
  set_turns(a, turns, rotary_dim, interleaved, magnitude);
  return launch_turn<false>(a, f32, (uint64_t)q | (uint64_t)k | (uint64_t)q_out | (uint64_t)k_out,
                            (uint64_t)(q_stride | k_stride), stream);
}

hipError_t launch_paged_append(const void* q, long long q_stride, const void* k,
                               long long k_stride, const void* v, long long v_stride,
                               const void* q_gain, const void* k_gain, float eps,
                               const uint64_t* turns, int rotary_dim, int interleaved,
                               float magnitude, bool f32, int tokens, int Hq, int Hkv,
                               int page_size, int pages, const PagedToken* records, void* k_pages,
                               void* v_pages, const PagedStrides& k_strides,
                               const PagedStrides& v_strides, void* q_out, hipStream_t stream) {
  TurnArgs a = {};
  a.src[0] = q;
  a.src[1] = k;
  a.src[2] = v;
  a.dst[0] = q_out;
  a.dst[1] = k_pages;
  a.dst[2] = v_pages;
  a.src_stride[0] = q_stride;
  a.src_stride[1] = k_stride;
  a.src_stride[2] = v_stride;
  a.pages[0] = k_strides;
  a.pages[1] = v_strides;
  a.gain[0] = q_gain;
  a.gain[1] = k_gain;
  a.eps = eps;
  a.records = records;
  a.page_size = page_size;
  a.page_count = pages;
  a.tokens = tokens;
  a.D = kD;
  a.heads[0] = Hq;
  a.heads[1] = Hkv;
  a.heads[2] = Hkv;
  a.sign = 1.f;
  a.div_len = make_fastdiv(1);
  set_turns(a, turns, rotary_dim, interleaved, magnitude);
  const uint64_t addresses = (uint64_t)q | (uint64_t)k | (uint64_t)v | (uint64_t)q_out |
                             (uint64_t)k_pages | (uint64_t)v_pages | (uint64_t)q_gain |
                             (uint64_t)k_gain;
  const uint64_t strides = (uint64_t)(q_stride | k_stride | v_stride | k_strides.page |
                                      k_strides.slot | k_strides.head | v_strides.page |
                                      v_strides.slot | v_strides.head);
  return launch_turn<true>(a, f32, addresses, strides, stream);
}

}  // namespace mf
