// Causal attention of a step's new tokens over a paged cache on gfx950.
//
// For each KV head the rows of a sequence are its (token, head of the group)
// pairs; row i * G + g at position p sees keys 0 .. p.  The plan (mf_paged.h)
// cut rows into tiles and a tile's keys into items; one workgroup of four waves
// takes an item of one KV head, in one of two ways:
//
//   up to 32 rows (decode, drafts): every wave holds all rows and takes every
//     fourth 32-key block, with a K and a V buffer of its own in LDS: no barrier
//     until the waves' softmax states are merged.  Bound: HBM, each cached key
//     and value is read once for all rows of its head.
//   up to 128 rows (chunks): every wave holds 32 rows, all share 64-key stages in
//     a ring of two.  Bound: MFMA and the LDS reads that feed it.
//
// Both use S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs: an accumulator
// column is a row of the batch, so its maximum and sum are in-lane reductions and
// one exchange between the halves, and the probabilities are already the operand
// of the second product.  Probabilities are rounded to bf16 for it (half a step,
// 2^-9 of each, of either sign); the sum adds the same rounded values, so that
// the weights still add to one.
//
// Items of a split tile write (max, sum, unnormalised output); a second launch
// joins them in item order.  No atomics: the same inputs give the same bits.
//
// Pages.  Page sizes are multiples of 8 and blocks start at multiples of 32, so
// eight keys of a block lie in one page: their page number is a scalar load, and
// their rows are moved by one LDS DMA from a scalar base.  Keys that are not
// there (behind the context, in a page outside the pool) are read from a row of
// zeros in the plan, so that nothing a masked slot holds, infinities and NaN
// included, meets a product.
#include "mf_f32.h"
#include "mf_lds.h"
#include "mf_paged.h"

namespace mf {

struct PagedArgs {
  const char* q;
  const char* k;
  const char* v;
  const int* table;
  const int* head;
  const char* zeros;
  const int* items;
  const int* tiles;
  char* out;
  float2* ml;               // partial results: (max in log2 units, sum) per row and KV head
  float* acc;               // and 64 outputs
  long long q_stride;       // bytes between tokens
  PagedStrides ks, vs;      // bytes
  long long table_stride;
  long long out_bytes;
  int page_size, pages, Hq, Hkv, G, zero_rest, tile_blocks;
  float scale_log2;
  FastDiv div_g, div_page, div_hkv;
};

struct ItemView {
  int start, row0, nrows, base, key0, key1, partial, sequence;
};

__device__ __forceinline__ ItemView load_item(const PagedArgs& a, int item) {
  const i32x8u r = ld_const8(a.items, 8 * item);
  return {r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};
}

// The page of key `key` of a table row (key wave-uniform, below the context).
__device__ __forceinline__ int page_of(const PagedArgs& a, const int* row, int key) {
  return ld_const(row, fast_div(key, a.div_page));
}

// Byte offset of key `key`'s row of KV head `kvh` in a pool, its page being `page`.
__device__ __forceinline__ long long row_offset(const PagedArgs& a, const PagedStrides& s, int page,
                                                int key, int kvh) {
  const int slot = key - fast_div(key, a.div_page) * a.page_size;
  return page * s.page + slot * s.slot + kvh * s.head;
}

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// dma16 with a 64-bit address per lane.
__device__ __forceinline__ void dma16_lane(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(src), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

template <int N>
__device__ __forceinline__ void wait_vm_lds() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Rows of keys key0 .. key0 + 7 (one page, `page` already checked or -1) into
// rows r0 .. r0 + 7 of an LDS tile; rows of keys from `end` on, and of no page,
// are zeros.  lane_off: the lane's byte offset from the first row.
__device__ __forceinline__ void dma_keys8(const PagedArgs& a, const char* pool,
                                          const PagedStrides& s, uint32_t lane_off, int chunk_off16,
                                          int page, int key0, int end, int kvh, char* tile, int r0) {
  const uint32_t dst = uniform((int)lds_offset(tile + r0 * kRowBytes));
  const char* base = pool + row_offset(a, s, max(page, 0), key0, kvh);
  if (page >= 0 && key0 + 8 <= end) {
    dma16(base, lane_off, dst);
  } else {
    const int row = __lane_id() >> 3;
    const char* src = page >= 0 && key0 + row < end ? base + lane_off : a.zeros + chunk_off16;
    dma16_lane(src, dst);
  }
}

// One row's running softmax: probabilities are 2^(s c - shift); shift is the
// running maximum in log2 units once a key was seen, and moves only when a new
// one exceeds it by more than lag (8 then, -inf before).
struct RowState {
  float shift, lag, l0, l1;
};

__device__ __forceinline__ void grow(RowState& st, float mx, f32x16 (&acc)[2]) {
  const bool up = mx > st.lag;
  if (__any(up)) {
    const float d = up ? mx : 0.f;
    // (a row that has seen no key holds zeros: 2^-d of its first maximum may
    // not be finite)
    const float alpha = st.lag > 0.f ? fast_exp2(-d) : 1.f;
    st.shift += d;
    st.lag = up ? 8.f : st.lag;
    st.l0 *= alpha;
    st.l1 *= alpha;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      acc[0][r] *= alpha;
      acc[1][r] *= alpha;
    }
  }
}

// Probabilities, their sums, and O += P V of one 32-key block whose V rows are
// rows v0 .. v0 + 31 of an LDS tile.
__device__ __forceinline__ void block_pv(f32x16& s, RowState& st, float c, const char* vt, int v0,
                                         int lane, f32x16 (&acc)[2]) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], c, -st.shift));
  const bf16x8 p0 = pack8(s, 0), p1 = pack8(s, 8);
  const u32x4 w0 = __builtin_bit_cast(u32x4, p0), w1 = __builtin_bit_cast(u32x4, p1);
  const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a0 = w0[j], a1 = w1[j];
    st.l0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a0), ones, st.l0, false);
    st.l1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a1), ones, st.l1, false);
  }
  const int tr_row = tr_row_of(lane), tr_col = tr_col_of(lane);
#pragma unroll
  for (int db = 0; db < 2; ++db) {
    const bf16x8 va = tile_tr_operand(vt, v0 + tr_row, db * 32 + tr_col);
    const bf16x8 vb = tile_tr_operand(vt, v0 + 16 + tr_row, db * 32 + tr_col);
    acc[db] = mfma32x32x16(va, p0, acc[db]);
    acc[db] = mfma32x32x16(vb, p1, acc[db]);
  }
}

__device__ __forceinline__ f32x16 block_scores(const char* kt, int k0, int lane,
                                               const bf16x8 (&qf)[4]) {
  f32x16 s = zero16();
#pragma unroll
  for (int ks = 0; ks < 4; ++ks)
    s = mfma32x32x16(tile_chunk(kt, k0 + (lane & 31), 2 * ks + (lane >> 5)), qf[ks], s);
  return s;
}

// Scores of keys from the lane's limit on (block of 32 keys from kb) and of the
// 8-key groups in `gone` become -inf; returns the column's maximum in the lane.
__device__ __forceinline__ float mask_scores(f32x16& s, int kb, int lim, bool diag, int gone,
                                             int lane) {
  if (diag) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = kb + acc_row(r, lane) < lim ? s[r] : kNegInf;
  }
  if (gone) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (gone >> g & 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g + i] = kNegInf;
      }
  }
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
  return mx;
}

// The lane's row of an item, and its output row.
struct RowOf {
  int token, head;
};
__device__ __forceinline__ RowOf row_of(const PagedArgs& a, const ItemView& it, int row, int kvh) {
  const int i = fast_div(it.row0 + row, a.div_g);
  return {it.start + i, kvh * a.G + (it.row0 + row - i * a.G)};
}

__device__ __forceinline__ void load_query(const PagedArgs& a, const RowOf& r, int lane,
                                           bf16x8 (&qf)[4]) {
  const char* src = a.q + r.token * a.q_stride + (long long)r.head * (kD * 2) + 16 * (lane >> 5);
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) qf[ks] = ld_bf16x8(src + 32 * ks);
}

// Keys that row `row` of the item sees, none from the item's end on.
__device__ __forceinline__ int row_limit(const PagedArgs& a, const ItemView& it, int row) {
  return min(max(it.base + fast_div(it.row0 + row, a.div_g) + 1, 0), it.key1);
}

// --------------------------------------------------------------------------
// Up to 32 rows: the waves split the keys.
// --------------------------------------------------------------------------
constexpr int kWaveLds = 2 * 32 * kRowBytes;  // a wave's K and V block

__device__ __forceinline__ void few_rows(const PagedArgs& a, const ItemView& it, int kvh, char* lds,
                                         float (*lm)[kFewRows], float (*ll)[kFewRows]) {
  const int lane = fresh_lane_id();  // (not kept alive across the other path's loop)
  const int wave = uniform(threadIdx.x >> 6);
  char* kt = lds + wave * kWaveLds;
  char* vt = kt + 32 * kRowBytes;
  const int row = min(lane & 31, it.nrows - 1);
  bf16x8 qf[4];
  load_query(a, row_of(a, it, row, kvh), lane, qf);
  const int lim = row_limit(a, it, row);
  const int least = uniform(row_limit(a, it, 0));
  drain_memory();

  const int chunk16 = ((lane & 7) ^ swz(lane >> 3)) * 16;
  const uint32_t k_off = (uint32_t)((lane >> 3) * a.ks.slot) + chunk16;
  const uint32_t v_off = (uint32_t)((lane >> 3) * a.vs.slot) + chunk16;
  const int* trow = a.table + it.sequence * a.table_stride;
  const int blocks = (it.key1 - it.key0 + 31) >> 5;

  f32x16 acc[2] = {zero16(), zero16()};
  RowState st = {0.f, kNegInf, 0.f, 0.f};
  const float c = a.scale_log2;
  int page[4];  // of the block that is fetched next
  auto pages_of = [&](int b) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int id = page_of(a, trow, min(it.key0 + 32 * b + 8 * g, it.key1 - 1));
      page[g] = (unsigned)id < (unsigned)a.pages ? id : -1;
    }
  };
  auto fetch = [&](const char* pool, const PagedStrides& s, uint32_t off, int b, char* tile) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      dma_keys8(a, pool, s, off, chunk16, page[g], it.key0 + 32 * b + 8 * g, it.key1, kvh, tile,
                8 * g);
  };
  int gone = 0, gone_next = 0;
  auto gone_of = [&]() {
    int m = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) m |= page[g] < 0 ? 1 << g : 0;
    return m;
  };
  int b = wave;
  if (b < blocks) {
    pages_of(b);
    gone_next = gone_of();
    fetch(a.k, a.ks, k_off, b, kt);
    fetch(a.v, a.vs, v_off, b, vt);
  }
  for (; b < blocks; b += 4) {
    const int kb = it.key0 + 32 * b;
    const bool more = b + 4 < blocks;
    gone = gone_next;
    if (more) {
      pages_of(b + 4);
      gone_next = gone_of();
    }
    wait_vm_lds<4>();  // K is there; V's four may be on their way
    f32x16 s = block_scores(kt, 0, lane, qf);
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    if (more) fetch(a.k, a.ks, k_off, b + 4, kt);
    const float mx = mask_scores(s, kb, lim, kb + 32 > least, gone, lane);
    grow(st, fmaf(halves_max(mx), c, -st.shift), acc);
    if (more) wait_vm_lds<4>(); else wait_vm_lds<0>();
    block_pv(s, st, c, vt, 0, lane, acc);
    wait_lds();
    __builtin_amdgcn_sched_barrier(0);
    if (more) fetch(a.v, a.vs, v_off, b + 4, vt);
  }
  wait_vm_lds<0>();

  // merge the waves: states to LDS (16-byte pieces of a row swizzled by the row)
  const float l = halves_sum(st.l0 + st.l1);
  if (lane < 32) {
    lm[wave][lane] = st.lag > 0.f ? st.shift : kNegInf;
    ll[wave][lane] = l;
  }
  if ((lane & 31) < it.nrows) {
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int piece = 8 * db + 2 * g + (lane >> 5);
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[db][4 * g + i];
        *reinterpret_cast<f32x4*>(kt + (lane & 31) * 256 + ((piece ^ (lane & 15)) << 4)) = x;
      }
  }
  __syncthreads();
  const int r = threadIdx.x >> 3, d8 = threadIdx.x & 7;
  if (r >= it.nrows) return;
  float top = lm[0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, lm[w][r]);
  float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float wt = lm[w][r] == kNegInf ? 0.f : fast_exp2(lm[w][r] - top);
    sum = fmaf(wt, ll[w][r], sum);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(lds + w * kWaveLds + r * 256 +
                                                      (((2 * d8 + h) ^ (r & 15)) << 4));
#pragma unroll
      for (int i = 0; i < 4; ++i) o[4 * h + i] = fmaf(wt, x[i], o[4 * h + i]);
    }
  }
  if (it.partial < 0) {
    const RowOf ro = row_of(a, it, r, kvh);
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    bf16x8 y;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = (bf16)(sum > 0.f ? o[i] * inv : 0.f);
    *reinterpret_cast<bf16x8*>(a.out + ((long long)ro.token * a.Hq + ro.head) * (kD * 2) + 16 * d8) = y;
  } else {
    const size_t at = ((size_t)it.partial + r) * a.Hkv + kvh;
    f32x4 x, y;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = o[i], y[i] = o[4 + i];
    *reinterpret_cast<f32x4*>(a.acc + at * kD + 8 * d8) = x;
    *reinterpret_cast<f32x4*>(a.acc + at * kD + 8 * d8 + 4) = y;
    if (d8 == 0) a.ml[at] = make_float2(top, sum);
  }
}

// --------------------------------------------------------------------------
// Up to 128 rows: the waves split the rows.
// --------------------------------------------------------------------------
constexpr int kSlotBytes = 2 * kTileBytes;  // 64 keys of K and of V

__device__ __forceinline__ void many_rows(const PagedArgs& a, const ItemView& it, int kvh,
                                          char* lds, int (*lost)[4]) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const bool idle = 32 * wave >= it.nrows;
  const int row = min(32 * wave + (lane & 31), it.nrows - 1);
  bf16x8 qf[4];
  load_query(a, row_of(a, it, row, kvh), lane, qf);
  const int lim = idle ? 0 : row_limit(a, it, row);
  // the rows' limits ascend
  const int least = uniform(__builtin_amdgcn_readlane(lim, 0));
  const int most = uniform(__builtin_amdgcn_readlane(lim, 31));
  drain_memory();

  const int chunk16 = ((lane & 7) ^ swz(lane >> 3)) * 16;
  const uint32_t k_off = (uint32_t)((lane >> 3) * a.ks.slot) + chunk16;
  const uint32_t v_off = (uint32_t)((lane >> 3) * a.vs.slot) + chunk16;
  const int* trow = a.table + it.sequence * a.table_stride;
  const int stages = (it.key1 - it.key0 + 63) >> 6;

  f32x16 acc[2] = {zero16(), zero16()};
  RowState st = {0.f, kNegInf, 0.f, 0.f};
  const float c = a.scale_log2;
  int page[2];  // of this wave's two groups of the stage that is fetched next
  auto pages_of = [&](int s) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int id = page_of(a, trow, min(it.key0 + 64 * s + 8 * (wave + 4 * j), it.key1 - 1));
      page[j] = (unsigned)id < (unsigned)a.pages ? id : -1;
    }
  };
  auto fetch = [&](int s) {
    char* slot = lds + (s & 1) * kSlotBytes;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int g = wave + 4 * j, key = it.key0 + 64 * s + 8 * g;
      dma_keys8(a, a.k, a.ks, k_off, chunk16, page[j], key, it.key1, kvh, slot, 8 * g);
      dma_keys8(a, a.v, a.vs, v_off, chunk16, page[j], key, it.key1, kvh, slot + kTileBytes, 8 * g);
    }
    // groups of this wave without a page: bit wave + 4 j
    lost[s & 1][wave] = (page[0] < 0 ? 1 << wave : 0) | (page[1] < 0 ? 16 << wave : 0);
  };
  if (stages > 0) {
    pages_of(0);
    fetch(0);
    if (stages > 1) pages_of(1);
  }
  for (int s = 0; s < stages; ++s) {
    wait_vm_lds<0>();
    barrier();
    if (s + 1 < stages) {
      fetch(s + 1);
      if (s + 2 < stages) pages_of(s + 2);
    }
    const int4 lo = *reinterpret_cast<const int4*>(lost[s & 1]);
    const int gone = uniform(lo.x | lo.y | lo.z | lo.w);
    const char* kt = lds + (s & 1) * kSlotBytes;
    const char* vt = kt + kTileBytes;
    const int kb = it.key0 + 64 * s;
    const bool run0 = kb < most, run1 = kb + 32 < most;
    if (!run0) continue;
    f32x16 s0 = block_scores(kt, 0, lane, qf), s1;
    if (run1) s1 = block_scores(kt, 32, lane, qf);
    float mx = mask_scores(s0, kb, lim, kb + 32 > least, gone & 15, lane);
    if (run1) mx = fmaxf(mx, mask_scores(s1, kb + 32, lim, kb + 64 > least, gone >> 4, lane));
    grow(st, fmaf(halves_max(mx), c, -st.shift), acc);
    block_pv(s0, st, c, vt, 0, lane, acc);
    if (run1) block_pv(s1, st, c, vt, 32, lane, acc);
  }
  wait_vm_lds<0>();  // no DMA may still target this workgroup's LDS at exit

  const int elane = fresh_lane_id();
  const int half = elane >> 5, erow = 32 * wave + (elane & 31);
  const float l = halves_sum(st.l0 + st.l1);
  if (erow >= it.nrows) return;
  if (it.partial < 0) {
    const RowOf ro = row_of(a, it, erow, kvh);
    const bool has = l > 0.f;
    store_bf16_rows(reinterpret_cast<bf16*>(a.out + ((long long)ro.token * a.Hq + ro.head) * (kD * 2)),
                    acc, has ? 1.f / l : 0.f, has, half);
  } else {
    const size_t at = ((size_t)it.partial + erow) * a.Hkv + kvh;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[db][4 * g + i];
        *reinterpret_cast<f32x4*>(a.acc + at * kD + 32 * db + 8 * g + 4 * half) = x;
      }
    if (half == 0) a.ml[at] = make_float2(st.lag > 0.f ? st.shift : kNegInf, l);
  }
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(4)))
void paged_attn_bf16_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[2 * kSlotBytes];
  __shared__ __attribute__((aligned(16))) float small[2][4][kFewRows];
  static_assert(4 * kWaveLds <= sizeof(lds), "the waves' blocks fit the ring");
  const int item = uniform(fast_div(blockIdx.x, a.div_hkv));
  if (item >= ld_const(a.head, kHeadItems)) return;
  const int kvh = uniform(blockIdx.x - item * a.Hkv);
  const ItemView it = load_item(a, item);
  if (it.nrows < 1) return;
  if (it.nrows <= kFewRows)
    few_rows(a, it, kvh, lds, small[0], small[1]);
  else
    many_rows(a, it, kvh, lds, reinterpret_cast<int(*)[4]>(small));
}

// --------------------------------------------------------------------------
// fp32: always up to 32 rows; the waves split the keys (32x32x2 MFMAs, rows staged
// through registers, as the packed fp32 forward).
// --------------------------------------------------------------------------
struct F32Keys {
  f32x4 x[8];
};

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void paged_attn_f32_kernel(PagedArgs a) {
  __shared__ F32Tile kt[4], vt[4], qt;
  __shared__ float lm[4][32], ll[4][32];
  const int item = uniform(fast_div(blockIdx.x, a.div_hkv));
  if (item >= ld_const(a.head, kHeadItems)) return;
  const int kvh = uniform(blockIdx.x - item * a.Hkv);
  const ItemView it = load_item(a, item);
  if (it.nrows < 1) return;
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  const int row = min(lane & 31, it.nrows - 1);
  const int lim = row_limit(a, it, row);
  const int least = uniform(row_limit(a, it, 0));
  constexpr int kRow = kD * 4;
  if (wave == 0) {
    f32x4 x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const RowOf ro = row_of(a, it, min(4 * i + (lane >> 4), it.nrows - 1), kvh);
      x[i] = *reinterpret_cast<const f32x4*>(a.q + ro.token * a.q_stride +
                                             (long long)ro.head * kRow + 16 * (lane & 15));
    }
    f32_store(qt, lane, x);
  }
  const int* trow = a.table + it.sequence * a.table_stride;
  const int blocks = (it.key1 - it.key0 + 31) >> 5;
  f32x4 kx[8], vx[8];
  int fetched_gone = 0;
  auto fetch = [&](int b) {
    fetched_gone = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int key = it.key0 + 32 * b + 8 * g;
      const int at = min(key, it.key1 - 1);
      const int id = page_of(a, trow, at);
      const bool there = (unsigned)id < (unsigned)a.pages;
      if (!there) fetched_gone |= 1 << g;
      // keys of the group before the item's end: all in this page
      const char* kp = a.k + row_offset(a, a.ks, there ? id : 0, min(key, at), kvh);
      const char* vp = a.v + row_offset(a, a.vs, there ? id : 0, min(key, at), kvh);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = min(4 * h + (lane >> 4), max(it.key1 - 1 - key, 0));
        kx[2 * g + h] = *reinterpret_cast<const f32x4*>(kp + r * a.ks.slot + 16 * (lane & 15));
        vx[2 * g + h] = *reinterpret_cast<const f32x4*>(vp + r * a.vs.slot + 16 * (lane & 15));
      }
    }
  };
  // rows that are not there are stored as zeros
  auto drop = [&](f32x4 (&x)[8], int gone) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      if (gone >> g & 1) x[2 * g] = x[2 * g + 1] = f32x4{0.f, 0.f, 0.f, 0.f};
  };

  f32x16 acc[2] = {zero16(), zero16()};
  float m = kNegInf, l = 0.f;
  const float c = a.scale_log2;
  int b = wave;
  if (b < blocks) fetch(b);
  __syncthreads();
  for (; b < blocks; b += 4) {
    const int kb = it.key0 + 32 * b;
    const int gone = fetched_gone;
    if (gone) {
      drop(kx, gone);
      drop(vx, gone);
    }
    wave_lds_fence();
    f32_store(kt[wave], lane, kx, it.key1 - kb);
    f32_store(vt[wave], lane, vx, it.key1 - kb);
    wave_lds_fence();
    if (b + 4 < blocks) fetch(b + 4);
    f32x16 s = zero16();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const f32x4 kr = kt[wave].row4(lane, j), qr = qt.row4(lane, j);
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mfma32x32x2(kr[e], qr[e], s);
    }
    const float mx = halves_max(mask_scores(s, kb, lim, kb + 32 > least, gone, lane));
    if (__any(mx > m)) {
      const float mnew = fmaxf(m, mx);
      const float alpha = mnew == kNegInf ? 1.f : fast_exp2((m - mnew) * c);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        acc[0][r] *= alpha;
        acc[1][r] *= alpha;
      }
    }
    const float mc = m == kNegInf ? 0.f : m * c;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = fast_exp2(fmaf(s[r], c, -mc));
      l += s[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      acc[0] = mfma32x32x2(vt[wave].col(lane, 0, r), s[r], acc[0]);
      acc[1] = mfma32x32x2(vt[wave].col(lane, 1, r), s[r], acc[1]);
    }
  }
  l = halves_sum(l);
  if (lane < 32) {
    lm[wave][lane] = m == kNegInf ? kNegInf : m * c;
    ll[wave][lane] = l;
  }
  wave_lds_fence();
  f32_put(kt[wave], lane, acc);
  __syncthreads();
  const int r = threadIdx.x >> 3, d0 = 8 * (threadIdx.x & 7);
  if (r >= it.nrows) return;
  float top = lm[0][r];
#pragma unroll
  for (int w = 1; w < 4; ++w) top = fmaxf(top, lm[w][r]);
  float wt[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    wt[w] = lm[w][r] == kNegInf ? 0.f : fast_exp2(lm[w][r] - top);
    sum = fmaf(wt[w], ll[w][r], sum);
  }
  const size_t at = ((size_t)max(it.partial, 0) + r) * a.Hkv + kvh;
  const RowOf ro = row_of(a, it, r, kvh);
  const float inv = it.partial >= 0 ? 1.f : sum > 0.f ? 1.f / sum : 0.f;
  float* dst = it.partial >= 0 ? a.acc + at * kD + d0
                               : reinterpret_cast<float*>(a.out) +
                                     ((long long)ro.token * a.Hq + ro.head) * kD + d0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) o += f32_at(kt[w], r, d0 + 4 * h) * wt[w];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = sum > 0.f ? o[e] * inv : 0.f;
    *reinterpret_cast<f32x4*>(dst + 4 * h) = o;
  }
  if (it.partial >= 0 && d0 == 0) a.ml[at] = make_float2(top, sum);
}

// --------------------------------------------------------------------------
// Joins the items of split tiles, in item order: o = sum_i 2^(m_i - M) acc_i / sum_i
// 2^(m_i - M) l_i.  A workgroup takes a tile of one KV head; eight threads of a
// row take eight dims each, and where there are few rows, the rest of the
// threads share the items.  Workgroups past the tiles zero the output rows that
// belong to no sequence, where that is asked for.
// --------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  __shared__ float part[32][64];
  __shared__ float2 pml[32];
  if ((int)blockIdx.x >= a.tile_blocks) {
    const long long row = (long long)a.Hq * kD * (F32 ? 4 : 2);
    const long long end = ld_const(a.head, kHeadEnd) * row;
    const long long at = (long long)(blockIdx.x - a.tile_blocks) * 16384;
    for (long long x = at + 16 * threadIdx.x; x < min(at + 16384, a.out_bytes); x += 16 * 256)
      if (x >= end) st_u32x4(a.out + x, u32x4{0, 0, 0, 0});
    return;
  }
  const int t = uniform(fast_div(blockIdx.x, a.div_hkv));
  if (t >= ld_const(a.head, kHeadTiles)) return;
  const int kvh = uniform(blockIdx.x - t * a.Hkv);
  const i32x8u tr = ld_const8(a.tiles, 8 * t);
  ItemView it = {};
  it.start = tr[0];
  it.row0 = tr[1];
  it.nrows = tr[2];
  const int partial = tr[3], splits = tr[4];
  int rp = 1;  // rows a round takes
  while (rp < it.nrows && rp < 32) rp <<= 1;
  const int sp = 32 / rp;  // threads' groups that share a row's items
  const int slot = threadIdx.x >> 3, d0 = 8 * (threadIdx.x & 7);
  const int r = slot & (rp - 1), share = slot / rp;
  for (int row0 = 0; row0 < it.nrows; row0 += rp) {
    const int row = min(row0 + r, it.nrows - 1);
    float m = kNegInf, l = 0.f, o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = 0.f;
    for (int s = share; s < splits; s += sp) {
      const size_t at = ((size_t)partial + (size_t)s * it.nrows + row) * a.Hkv + kvh;
      const float2 ml = a.ml[at];
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.acc + at * kD + d0);
      const f32x4 y = *reinterpret_cast<const f32x4*>(a.acc + at * kD + d0 + 4);
      const float top = fmaxf(m, ml.x);
      const float wa = m == kNegInf ? 0.f : fast_exp2(m - top);
      const float wb = ml.x == kNegInf ? 0.f : fast_exp2(ml.x - top);
      l = l * wa + ml.y * wb;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        o[i] = o[i] * wa + x[i] * wb;
        o[4 + i] = o[4 + i] * wa + y[i] * wb;
      }
      m = top;
    }
    __syncthreads();  // the previous round's readers are done
#pragma unroll
    for (int i = 0; i < 8; ++i) part[slot][d0 + i] = o[i];
    if (d0 == 0) pml[slot] = make_float2(m, l);
    __syncthreads();
    if (share == 0 && row0 + r < it.nrows) {
      float top = m;
      for (int x = 1; x < sp; ++x) top = fmaxf(top, pml[x * rp + r].x);
      float sum = 0.f, z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      for (int x = 0; x < sp; ++x) {
        const float2 ml = pml[x * rp + r];
        const float w = ml.x == kNegInf ? 0.f : fast_exp2(ml.x - top);
        sum = fmaf(w, ml.y, sum);
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = fmaf(w, part[x * rp + r][d0 + i], z[i]);
      }
      const RowOf ro = row_of(a, it, row, kvh);
      const float inv = sum > 0.f ? 1.f / sum : 0.f;
      const long long at = ((long long)ro.token * a.Hq + ro.head) * kD + d0;
      if constexpr (F32) {
        float* dst = reinterpret_cast<float*>(a.out) + at;
#pragma unroll
        for (int i = 0; i < 8; ++i) dst[i] = sum > 0.f ? z[i] * inv : 0.f;
      } else {
        bf16x8 y;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (bf16)(sum > 0.f ? z[i] * inv : 0.f);
        *reinterpret_cast<bf16x8*>(reinterpret_cast<bf16*>(a.out) + at) = y;
      }
    }
  }
}

hipError_t launch_paged_attn(const void* q, long long q_stride, const void* k_pages,
                             const void* v_pages, const PagedStrides& k_strides,
                             const PagedStrides& v_strides, const int32_t* page_table,
                             long long table_stride, bool f32, int tokens, int sequences,
                             int page_size, int pages, int Hq, int Hkv, float scale,
                             const void* plan, bool zero_rest, void* out, void* workspace,
                             hipStream_t stream) {
  const int size = f32 ? 4 : 2;
  const PagedLayout lay = paged_layout(sequences, tokens, Hq / Hkv, Hkv, f32);
  const char* p = reinterpret_cast<const char*>(plan);
  PagedArgs a = {};
  a.q = reinterpret_cast<const char*>(q);
  a.k = reinterpret_cast<const char*>(k_pages);
  a.v = reinterpret_cast<const char*>(v_pages);
  a.table = page_table;
  a.head = reinterpret_cast<const int*>(p);
  a.zeros = p + lay.zeros;
  a.items = reinterpret_cast<const int*>(p + lay.items);
  a.tiles = reinterpret_cast<const int*>(p + lay.tiles);
  a.out = reinterpret_cast<char*>(out);
  a.ml = reinterpret_cast<float2*>(workspace);
  a.acc = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) +
                                   align256(lay.cap_rows * Hkv * (2 * sizeof(float))));
  a.q_stride = q_stride * size;
  a.ks = {k_strides.page * size, k_strides.slot * size, k_strides.head * size};
  a.vs = {v_strides.page * size, v_strides.slot * size, v_strides.head * size};
  a.table_stride = table_stride;
  a.out_bytes = (long long)tokens * Hq * kD * size;
  a.page_size = page_size;
  a.pages = pages;
  a.Hq = Hq;
  a.Hkv = Hkv;
  a.G = Hq / Hkv;
  a.zero_rest = zero_rest;
  a.tile_blocks = lay.cap_tiles * Hkv;
  a.scale_log2 = scale * kLog2e;
  a.div_g = make_fastdiv(a.G);
  a.div_page = make_fastdiv(page_size);
  a.div_hkv = make_fastdiv(Hkv);
  const dim3 grid((unsigned)lay.cap_items * Hkv);
  const long long rest = zero_rest ? (a.out_bytes + 16383) / 16384 : 0;
  const dim3 join((unsigned)(a.tile_blocks + rest));
  if (f32) {
    hipLaunchKernelGGL(paged_attn_f32_kernel, grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(paged_join_kernel<true>, join, dim3(256), 0, stream, a);
  } else {
    hipLaunchKernelGGL(paged_attn_bf16_kernel, grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(paged_join_kernel<false>, join, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace mf
