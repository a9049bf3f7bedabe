// Causal attention of a step's new tokens over a paged cache on gfx950.
//
// For each KV head the rows of a sequence are its (token, head of the group)
// pairs; row i * G + g at position p sees keys 0 .. p.  The plan (mf_paged.h)
// cut rows into tiles and a tile's keys into items; a workgroup of four waves
// takes an item in one of two ways:
//
//   up to 32 rows (decode, drafts): every wave holds all rows of one or two KV
//     heads and takes 32-key blocks of its own, through a K and a V buffer of its
//     own in LDS: no barrier until the states of waves that share an item are
//     merged.  Bound: HBM, each cached key and value is read once for all rows of
//     its head.  One token for each of 64 sequences of 129 to 8192 keys, 16/8 heads
//     (494 MB): 84 us, 5.9 TB/s, and the join 5; 24 sequences of 3 to 8 drafts, 24/8
//     heads (391 MB): 70 and 5.  Half the workgroups a CU take 3 % longer.
//   up to 256 rows (chunks), one KV head: every wave holds 64 rows, all share
//     64-key stages in a ring of four, so an operand read from LDS feeds two MFMAs.
//     2048 tokens behind 28672, 16/8 heads: 275 to 300 us with the join, 830 to 900
//     TFLOP/s; 16384 behind none 605 (a large bf16 matrix product on the card: 1190
//     TFLOP/s).  MFMA busy 41 % of the cycles, VALU 58 %, and the clock: the same launch
//     over zeros takes 14 % less.  (8 maxima less a block changed nothing.)
//
// The same sequences with 24 rows on the second path: 101 us instead of 76, so few
// rows end at 32, what one MFMA holds.
//
// Both use S^T = K Q^T and O^T += V^T P^T with 32x32x16 MFMAs: an accumulator
// column is a row of the batch, so its maximum and sum are in-lane reductions and
// one exchange between the halves, and the probabilities are already the operand
// of the second product.  Of few rows they go into it as two bf16 parts, within 2^-16
// of each, so that an output is off by its own rounding alone (1.65e-3 in the mean
// square; with one part 2.3e-3).  The second part takes single tokens and drafts 2 %
// longer (64 tokens 92.7 us with the join instead of 90.6, drafts 76.1 instead of 75.0);
// made before the first part's products instead of under them, 3 %.  It would take many
// rows 35 % longer (a chunk over 28 K keys 414 us instead of 307, 16 K causal 853 instead
// of 610): theirs are rounded to bf16 once, by 2^-8 of each at most, of either sign, as
// in the packed forward that trains the model; the sum adds the same rounded values, so
// that the weights still add to one.
//
// Items of a split tile write (max, sum, unnormalised output); a second launch
// joins them in item order.  No atomics: the same inputs give the same bits.
//
// Rows.  A row that sees no key is zeros.  One that sees a key is what the definition
// gives, whatever its scores are: NaN where one is NaN or +infinity, or all are
// -infinity.  So "no key" is a state of its own: maximum -infinity and a sum whose bits
// are zero.  A NaN marks the sum (a maximum passes over it), +infinity does so with the
// subtraction of the shift, and a row that has only scores of -infinity gets the lowest
// finite maximum and a sum of one at its end (mark_low): beside any other maximum its
// weight is 0, and without one the row is NaN (row_factor).  What tells sums apart looks
// at their bits: the file is compiled as if no comparison saw a NaN.
//
// Pages.  Page sizes are multiples of 8 and blocks start at multiples of 32, so
// eight keys of a block lie in one page: their page number is a scalar load, and
// their rows are moved by LDS DMAs from a scalar base.  Keys that are not there
// (behind the context, in a page outside the pool) are read from a row of zeros
// in the plan, so that nothing a masked slot holds, infinities and NaN included,
// meets a product.
#include <type_traits>

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
  const int* shares[2];     // by kind
  const int* items[2];
  const int* joins;
  char* out;
  float2* ml;               // partial results: (max in log2 units, sum) per KV head and row
  float* acc;               // and 64 outputs
  long long q_stride;       // bytes between tokens
  PagedStrides ks, vs;      // bytes
  long long table_stride;
  long long out_bytes;
  long long cap_rows;       // partial rows of a KV head
  int page_size, pages, Hq, Hkv, G;
  int few_turns, many_turns;  // 256 workgroups each
  int join_blocks, head_pairs;
  float scale_log2;
  FastDiv div_g, div_page, div_hkv, div_pairs;
};

struct ItemView {
  int start, row0, nrows, base, key0, key1, partial, sequence;
};

__device__ __forceinline__ ItemView load_item(const int* items, int item) {
  const i32x8u r = ld_const8(items, 8 * item);
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
// LDS DMAs of 16 bytes a lane (mf_lds.h) that are not kept in cache: a few-rows
// item's keys and values are read once.  Kept, 64 single tokens take 101 us instead
// of 91, two over 128 K keys 101 instead of 89, drafts 86 instead of 76.
__device__ __forceinline__ void dma16_once(const void* sbase, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               :: "v"(voff), "s"(sbase), "s"(lds) : "memory", "m0");
}
// With a 64-bit address per lane.
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

// One row's running softmax: probabilities are 2^(s c - shift); shift is the
// running maximum in log2 units once a key was seen, and moves only when a new
// one exceeds it by more than lag (8 then, -inf before).
struct RowState {
  float shift, lag, l0, l1;
};

// Whether a sum of weights is that of a row without keys.
__device__ __forceinline__ bool no_weight(float l) { return __float_as_uint(l) == 0u; }

// The weight of a state (m, l) where states are joined under the maximum `top`.
__device__ __forceinline__ float state_weight(float m, float l, float top) {
  return no_weight(l) ? 0.f : fast_exp2(m - top);
}

// The maximum of a row with keys whose scores are all -infinity.  (With -infinity there
// too, and a weight of one chosen under a maximum of -infinity, the second select beside
// each weight cost attention and join of one token 11.1 us instead of 10.0.)
constexpr float kLowest = -0x1.fffffep127f;

// What a row's outputs are multiplied by: zero without keys, NaN where no score is above
// -infinity.
__device__ __forceinline__ float row_factor(float top, float sum) {
  float nan;
  asm("v_mov_b32 %0, 0x7fc00000" : "=v"(nan));  // (a constant NaN may be optimised away)
  return no_weight(sum) ? 0.f : top == kLowest ? nan : 1.f / sum;
}

// The first position from `from` (a page's or block's first key) up to `end` whose page
// is in the pool, 2^31 - 1 if there is none; all lanes of the wave take part.
__device__ __forceinline__ int first_key(const PagedArgs& a, const int* row, int from, int end) {
  const int lane = fresh_lane_id();
  const int last = fast_div(end - 1, a.div_page);
  for (int p0 = fast_div(from, a.div_page); p0 <= last; p0 += 64) {
    const bool there = p0 + lane <= last && (unsigned)row[min(p0 + lane, last)] < (unsigned)a.pages;
    const uint64_t any = __ballot(there);
    if (any) return max(from, (p0 + __ffsll((unsigned long long)any) - 1) * a.page_size);
  }
  return 0x7fffffff;
}

// The state of a row (maximum in log2 units, sum) at the end of its keys from `from` up to
// `end`, of which it sees `lim`: one without a maximum that sees a key has a score of
// -infinity there.  Rows mostly have a maximum, and no table is read.
__device__ __forceinline__ float2 mark_low(const PagedArgs& a, const int* row, int from, int end,
                                           int lim, float m, float l) {
  const bool open = no_weight(l) && lim > from;
  if (__any(open)) {
    const int first = first_key(a, row, from, end);
    if (open && first < lim) return make_float2(kLowest, 1.f);
  }
  return make_float2(m, l);
}

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

// Probabilities of one 32-key block in bf16 (the operands of its two 16-key
// steps), and their sums.
__device__ __forceinline__ void block_probs(f32x16& s, RowState& st, float c, bf16x8& p0, bf16x8& p1) {
#pragma unroll
  for (int r = 0; r < 16; ++r) s[r] = fast_exp2(fmaf(s[r], c, -st.shift));
  p0 = pack8(s, 0);
  p1 = pack8(s, 8);
  const u32x4 w0 = __builtin_bit_cast(u32x4, p0), w1 = __builtin_bit_cast(u32x4, p1);
  const bf16x2 ones = __builtin_bit_cast(bf16x2, 0x3F803F80u);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t a0 = w0[j], a1 = w1[j];
    st.l0 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a0), ones, st.l0, false);
    st.l1 = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, a1), ones, st.l1, false);
  }
}

// The same, the probabilities themselves kept for their second part.
__device__ __forceinline__ void block_probs_first(f32x16& s, const RowState& st, float c, bf16x8 (&p)[2]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = fast_exp2(fmaf(s[i], c, -st.shift));
  p[0] = pack8(s, 0);
  p[1] = pack8(s, 8);
}
// What p leaves of the probabilities, in bf16 too: together within 2^-16 of each.  The
// sum adds the probabilities.
__device__ __forceinline__ void block_probs_rest(const f32x16& s, RowState& st, bf16x8 (&p)[2]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const u32x4 w = __builtin_bit_cast(u32x4, p[j]);
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = s[8 * j + 2 * i], b = s[8 * j + 2 * i + 1];
      st.l0 += a;
      st.l1 += b;
      x[i] = round_bf16_pair(a - bf16_lo(w[i]), b - bf16_hi(w[i]));
    }
    p[j] = __builtin_bit_cast(bf16x8, x);
  }
}

// Scores of keys from the lane's limit on (block of 32 keys from kb) and of the
// 8-key groups in `gone` become -inf.
__device__ __forceinline__ void mask_scores(f32x16& s, int kb, int lim, int gone, int lane) {
#pragma unroll
  for (int r = 0; r < 16; ++r)
    s[r] = kb + acc_row(r, lane) < lim && !(gone >> (r >> 2) & 1) ? s[r] : kNegInf;
}

// A value the compiler cannot see through: what is computed from it stays in the
// branch it is made in.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+s"(x));
  return x;
}

// Maximum of a column's scores in the lane.
__device__ __forceinline__ float column_max(const f32x16& s) {
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
  return mx;
}

// Infinities and NaN among values that some rows of an item do not see.  Their
// probability is 0 there, and 0 times such a value is NaN.  Any leaves its mark in the
// sums, so the loops do not look for them: an item with causally masked keys whose
// sums are not all finite is done once more (Careful, 32 rows at a time), now with
// these values taken out of the operands of masked blocks (drop_wild) and added by
// themselves to the rows that do see them (add_wild, key by key).  Rows that see none
// come out with the same bits as without them.  (A check of every masked block as it
// comes cost chunks 4 %, in registers.)
typedef std::false_type Plain;
typedef std::true_type Careful;

// Bits 15 and 31 of the result: whether the low and the high half of a word are
// such values (an exponent of all ones carries into them).
__device__ __forceinline__ uint32_t wild_bits(uint32_t w) {
  return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
// Bit 31: whether one of the floats is one.
__device__ __forceinline__ uint32_t wild_bits(const f32x16& v) {
  uint32_t any = 0;
#pragma unroll
  for (int r = 0; r < 16; ++r) any |= (__float_as_uint(v[r]) & 0x7f800000u) + 0x00800000u;
  return any & 0x80000000u;
}
__device__ __forceinline__ uint32_t wild_bits(const bf16x8& v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  return wild_bits(w[0]) | wild_bits(w[1]) | wild_bits(w[2]) | wild_bits(w[3]);
}
__device__ __forceinline__ void drop_wild(bf16x8& v) {
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x = w[i];
    w[i] = x & ~((wild_bits(x) >> 15) * 0xffffu);
  }
  v = __builtin_bit_cast(bf16x8, w);
}
// The same of a float, as all ones or zero.  (Integers throughout: the file is compiled
// as if no value were NaN, and a comparison of floats may be simplified by that.)
__device__ __forceinline__ uint32_t wild_mask(float x) {
  return 0u - (((__float_as_uint(x) & 0x7f800000u) + 0x00800000u) >> 31);
}
// acc += x, whatever x is.
__device__ __forceinline__ float add_any(float acc, float x) {
  asm("v_add_f32 %0, %0, %1" : "+v"(acc) : "v"(x));
  return acc;
}
// quad(key, 4 db + g): dims 32 db + 8 g + 4 half .. + 3 of a key of the block; `seen`
// keys of it are the lane's row's.
template <typename Quad>
__device__ __forceinline__ void add_wild(f32x16 (&acc)[2], int seen, Quad quad) {
#pragma unroll 1
  for (int key = 0; key < 32; ++key) {
    const uint32_t mine = key < seen ? 0xffffffffu : 0u;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const u32x2 w = quad(key, 4 * db + g);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = w[i];
          const uint32_t y = x & ((wild_bits(x) >> 15) * 0xffffu) & mine;
          acc[db][4 * g + 2 * i] = add_any(acc[db][4 * g + 2 * i], bf16_lo(y));
          acc[db][4 * g + 2 * i + 1] = add_any(acc[db][4 * g + 2 * i + 1], bf16_hi(y));
        }
      }
  }
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
// Up to 32 rows of HW (1 or 2) adjacent KV heads a wave.
//
// A wave's K (and V) block in LDS is 32 tokens of HW 128-byte rows; a DMA moves
// 8 / HW tokens, HW * 128 consecutive bytes of each where heads lie next to each
// other.  (Two heads: 256-byte pieces of a token's row instead of 128; 64 single
// tokens 91 us instead of 96, drafts 76 instead of 82.)  The
// 16-byte pieces of a token are permuted by XOR with few_swz(token), so that the
// 16 tokens that an operand read covers fall on all banks, and the transposing
// reads of eight tokens too.
// --------------------------------------------------------------------------
template <int HW>
__device__ __forceinline__ int few_swz(int t) {
  return HW == 1 ? swz(t) : ((t & 7) << 1) | ((t >> 3) & 1);
}

template <int HW>
struct FewLds {
  static constexpr int kTok = HW * kRowBytes;      // bytes of a token
  static constexpr int kBlock = 32 * kTok;         // a K or V block
  static constexpr int kWave = 2 * kBlock;
};

// Keys of block kb .. kb + 31 of a pool into a wave's LDS block.  at: byte offsets of
// the first rows of its four groups; off: the lane's byte offsets from the first
// token of a DMA, by the DMA's number (mod 4 for two heads, where the permutation
// depends on it).
template <int HW>
__device__ __forceinline__ void few_fetch(const PagedArgs& a, const char* pool, long long slot,
                                          const long long (&at)[4], const uint32_t (&off)[2 * HW],
                                          int gone, int kb, int end, char* block) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int key = kb + 8 * g;
    const char* base = pool + at[g];
    if (!(gone >> g & 1) && key + 8 <= end) {
#pragma unroll
      for (int j = 0; j < HW; ++j)
        dma16_once(base + j * 4 * slot, off[HW == 1 ? 0 : (2 * g + j) & 3],
                   uniform((int)lds_offset(block + (HW * g + j) * 1024)));
    } else {
      const int lane = __lane_id();
#pragma unroll
      for (int j = 0; j < HW; ++j) {
        const bool there = !(gone >> g & 1) && key + j * 4 + lane / (8 * HW) < end;
        const char* src = there ? base + j * 4 * slot + off[HW == 1 ? 0 : (2 * g + j) & 3]
                                : a.zeros + 16 * (lane & 7);
        dma16_lane(src, uniform((int)lds_offset(block + (HW * g + j) * 1024)));
      }
    }
  }
}

// ALONE: the wave takes all keys of its rows, carefully, with the many-rows path's
// arithmetic (rows that do not see an infinity or NaN get that path's very bits).
template <int HW, bool ALIKE, bool ALONE>
__device__ __forceinline__ void few_rows(const PagedArgs& a, const ItemView& it, int pair,
                                         int key_wave, char* wave_lds, float* lm, float* ll) {
  typedef FewLds<HW> L;
  const int lane = fresh_lane_id();  // (not kept alive across the other path's loop)
  const int half = lane >> 5;
  const int head0 = HW * pair;
  char* kt = wave_lds;
  char* vt = wave_lds + L::kBlock;
  const int row = min(lane & 31, it.nrows - 1);
  bf16x8 qf[HW][4];
#pragma unroll
  for (int h = 0; h < HW; ++h) load_query(a, row_of(a, it, row, head0 + h), lane, qf[h]);
  const int lim = row_limit(a, it, row);
  const int least = uniform(row_limit(a, it, 0));
  drain_memory();

  // the lane's piece of a DMA: token tok, and the piece whose place is the lane's
  uint32_t k_off[2 * HW], v_off[2 * HW];
#pragma unroll
  for (int i = 0; i < 2 * HW; ++i) {
    const int tok = lane / (8 * HW);
    const int piece = (lane & (8 * HW - 1)) ^ few_swz<HW>(HW == 1 ? tok : 4 * i + tok);
    k_off[i] = (uint32_t)(tok * a.ks.slot) + (uint32_t)((piece >> 3) * a.ks.head) + 16 * (piece & 7);
    v_off[i] = ALIKE ? k_off[i] : (uint32_t)(tok * a.vs.slot) +
                                      (uint32_t)((piece >> 3) * a.vs.head) + 16 * (piece & 7);
  }
  // operand addresses: piece 8 h + 2 ks + half of token lane & 31, and for the
  // transposing reads piece 8 h + 4 db + tr_col / 8 of token tr_row (+ 8, + 16)
  const int tr_row = tr_row_of(lane), tr_col = tr_col_of(lane);
  const int k_at = (lane & 31) * L::kTok + ((half ^ few_swz<HW>(lane & 31)) << 4);
  const int v_at = tr_row * L::kTok + (((tr_col >> 3) ^ few_swz<HW>(tr_row)) << 4) + 2 * (tr_col & 7);

  const int* trow = a.table + it.sequence * a.table_stride;
  const int blocks = (it.key1 - it.key0 + 31) >> 5;
  f32x16 acc[HW][2];
  RowState st[HW];
  float top[HW];
  const float c = a.scale_log2;
  // The table's entries of the block that is fetched next, checked only when they are
  // used (a check is a wait for the load); where its rows are; the groups of eight
  // keys without a page.
  int entry[4], gone = 0, gone_next = 0;
  long long at[4];
  auto load_entries = [&](int b) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      entry[g] = page_of(a, trow, min(it.key0 + 32 * b + 8 * g, it.key1 - 1));
  };
  auto place = [&](const PagedStrides& s, int b) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at[g] = row_offset(a, s, gone_next >> g & 1 ? 0 : entry[g], it.key0 + 32 * b + 8 * g, head0);
  };
  auto fetch_keys = [&](int b) {
    gone_next = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) gone_next |= (unsigned)entry[g] < (unsigned)a.pages ? 0 : 1 << g;
    place(a.ks, b);
    few_fetch<HW>(a, a.k, a.ks.slot, at, k_off, gone_next, it.key0 + 32 * b, it.key1, kt);
  };
  auto fetch_values = [&](int b) {
    if (!ALIKE) place(a.vs, b);
    few_fetch<HW>(a, a.v, ALIKE ? a.ks.slot : a.vs.slot, at, v_off, gone_next, it.key0 + 32 * b,
                  it.key1, vt);
  };
  auto run = [&](auto how) {
    constexpr bool careful = decltype(how)::value;
#pragma unroll
    for (int h = 0; h < HW; ++h) {
      acc[h][0] = acc[h][1] = zero16();
      st[h] = {0.f, kNegInf, 0.f, 0.f};
      top[h] = kNegInf;
    }
    int b = ALONE ? 0 : key_wave;
    if (b < blocks) {
      load_entries(b);
      fetch_keys(b);
      fetch_values(b);
    }
    constexpr int kStep = ALONE ? 1 : kKeyWaves;
    for (; b < blocks; b += kStep) {
      const int kb = it.key0 + 32 * b, next = b + kStep;
      const bool more = next < blocks;
      gone = gone_next;
      if (more) load_entries(next);
      wait_vm_lds<4 * HW>();  // K is there; V's DMAs may be on their way
      f32x16 s[HW];
#pragma unroll
      for (int h = 0; h < HW; ++h) {
        s[h] = zero16();
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
          s[h] = mfma32x32x16(ld_bf16x8(kt + (k_at ^ ((8 * h + 2 * ks) << 4))), qf[h][ks], s[h]);
      }
      wait_lds();
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch_keys(next);
      const bool masked = kb + 32 > least || gone;
      bf16x8 p[HW][2];
#pragma unroll
      for (int h = 0; h < HW; ++h) {
        if (masked) mask_scores(s[h], opaque(kb), lim, gone, lane);
        const float mx = column_max(s[h]);
        if (!ALONE || __any(mx > top[h])) {
          grow(st[h], fmaf(halves_max(mx), c, -st[h].shift), acc[h]);
          if (ALONE) top[h] = (st[h].shift + st[h].lag) * (1.f / c);
        }
        if constexpr (ALONE) block_probs(s[h], st[h], c, p[h][0], p[h][1]);
        else block_probs_first(s[h], st[h], c, p[h]);
      }
      if (more) wait_vm_lds<4 * HW>(); else wait_vm_lds<0>();
#pragma unroll
      for (int h = 0; h < HW; ++h) {
        bf16x8 v[2][2];
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const char* from = vt + 16 * j * L::kTok;
            const int x = v_at ^ ((8 * h + 4 * db) << 4);
            const u32x2 lo = lds_read_tr16(from + x);
            // token + 8: the permutation of two heads differs in its lowest bit
            const u32x2 hi = lds_read_tr16(from + 8 * L::kTok + (HW == 1 ? x : x ^ 16));
            const u32x4 w = {lo[0], lo[1], hi[0], hi[1]};
            v[db][j] = __builtin_bit_cast(bf16x8, w);
          }
        if (careful && masked) {
          add_wild(acc[h], lim - kb, [&](int key, int piece) {
            return *reinterpret_cast<const u32x2*>(
                vt + key * L::kTok + (((8 * h + piece) ^ few_swz<HW>(key)) << 4) + 8 * half);
          });
#pragma unroll
          for (int db = 0; db < 2; ++db) {
            drop_wild(v[db][0]);
            drop_wild(v[db][1]);
          }
        }
#pragma unroll
        for (int part = 0; part < (ALONE ? 1 : 2); ++part) {
          // (the second part is made under the first one's products)
          if (part == 1) block_probs_rest(s[h], st[h], p[h]);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int db = 0; db < 2; ++db) acc[h][db] = mfma32x32x16(v[db][j], p[h][j], acc[h][db]);
        }
      }
      wait_lds();
      __builtin_amdgcn_sched_barrier(0);
      if (more) fetch_values(next);
    }
  };
  bool careful = ALONE;
  if constexpr (!ALONE) {
    run(Plain{});
    if (it.key1 > least) {
      uint32_t wild = 0;
#pragma unroll
      for (int h = 0; h < HW; ++h) wild |= wild_bits(acc[h][0]) | wild_bits(acc[h][1]);
      careful = __any(wild != 0);
    }
  }
  if (careful) run(Careful{});
  wait_vm_lds<0>();  // no DMA may still target this workgroup's LDS

  // the wave's states to LDS: row r of head h at (32 h + r) * 256 bytes, 16-byte
  // pieces permuted by the row
#pragma unroll
  for (int h = 0; h < HW; ++h) {
    const float2 ml = mark_low(a, trow, it.key0 + (ALONE ? 0 : 32 * key_wave), it.key1, lim,
                               st[h].lag > 0.f ? st[h].shift : kNegInf,
                               halves_sum(st[h].l0 + st[h].l1));
    if (lane < 32) {
      lm[32 * h + lane] = ml.x;
      ll[32 * h + lane] = ml.y;
    }
    if ((lane & 31) < it.nrows) {
#pragma unroll
      for (int db = 0; db < 2; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int piece = 8 * db + 2 * g + half;
          f32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = acc[h][db][4 * g + i];
          *reinterpret_cast<f32x4*>(wave_lds + (32 * h + (lane & 31)) * 256 +
                                    ((piece ^ (lane & 15)) << 4)) = x;
        }
    }
  }
}

// Merges the states of an item that waves first .. first + WAVES - 1 hold, and writes
// rows or partial results; eight threads of these waves a row.
template <int HW, int WAVES>
__device__ __forceinline__ void few_merge(const PagedArgs& a, const ItemView& it, int pair,
                                          int first, int thread, const char* lds,
                                          const float (*lm)[64], const float (*ll)[64]) {
  const int d8 = thread & 7;
  for (int x = thread >> 3; x < HW * it.nrows; x += 8 * WAVES) {
    const int h = x >= it.nrows ? 1 : 0, r = x - h * it.nrows, at = 32 * h + r;
    const int kvh = HW * pair + h;
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lm[first + w][at]);
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float m = lm[first + w][at], l = ll[first + w][at];
      const float wt = state_weight(m, l, top);
      sum = fmaf(wt, l, sum);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(
            lds + (first + w) * FewLds<HW>::kWave + at * 256 + (((2 * d8 + q) ^ (r & 15)) << 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) o[4 * q + i] = fmaf(wt, y[i], o[4 * q + i]);
      }
    }
    if (it.partial < 0) {
      const RowOf ro = row_of(a, it, r, kvh);
      const bool none = no_weight(sum);
      const float inv = row_factor(top, sum);
      bf16x8 y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (bf16)(none ? 0.f : o[i] * inv);
      *reinterpret_cast<bf16x8*>(a.out + ((long long)ro.token * a.Hq + ro.head) * (kD * 2) + 16 * d8) = y;
    } else {
      const size_t to = (size_t)(kvh * a.cap_rows) + it.partial + r;
      f32x4 y, z;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = o[i], z[i] = o[4 + i];
      *reinterpret_cast<f32x4*>(a.acc + to * kD + 8 * d8) = y;
      *reinterpret_cast<f32x4*>(a.acc + to * kD + 8 * d8 + 4) = z;
      if (d8 == 0) a.ml[to] = make_float2(top, sum);
    }
  }
}

// A many-rows item again: every wave its own 64 rows, 32 at a time.
template <bool ALIKE>
__device__ __forceinline__ void many_again(const PagedArgs& a, const ItemView& it, int kvh, char* lds,
                                           float (&lm)[4][64], float (&ll)[4][64]) {
  const int wave = uniform(threadIdx.x >> 6);
  __syncthreads();  // the waves are done with what LDS held
#pragma unroll 1
  for (int row = 64 * wave; row < min(64 * wave + 64, it.nrows); row += 32) {
    const ItemView part = {it.start, it.row0 + row, min(32, it.nrows - row), it.base, it.key0,
                           it.key1,  it.partial < 0 ? -1 : it.partial + row, it.sequence};
    few_rows<1, ALIKE, true>(a, part, kvh, wave, lds + wave * FewLds<1>::kWave, lm[wave], ll[wave]);
    wave_lds_fence();
    few_merge<1, 1>(a, part, kvh, wave, threadIdx.x & 63, lds, lm, ll);
    wave_lds_fence();
  }
}

// --------------------------------------------------------------------------
// Up to 256 rows: the waves split the rows, 64 (two 32-row blocks) each, so that
// every K and V operand read from LDS feeds two MFMAs.
// --------------------------------------------------------------------------
constexpr int kSlotBytes = 2 * kTileBytes;  // 64 keys of K and of V
constexpr int kSlots = 4;

// False if the item has to be done again, carefully.
template <bool ALIKE>
__device__ __forceinline__ bool many_rows(const PagedArgs& a, const ItemView& it, int kvh, char* lds,
                                          int (*lost)[4], int* flags) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  bf16x8 qf[2][4];
  int lim[2], least = 0, most = 0;
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int row0 = 64 * wave + 32 * rb;
    const int row = min(row0 + (lane & 31), it.nrows - 1);
    load_query(a, row_of(a, it, row, kvh), lane, qf[rb]);
    lim[rb] = row_limit(a, it, row);
    // the rows' limits ascend
    if (rb == 0) least = uniform(__builtin_amdgcn_readlane(lim[0], 0));
    if (row0 < it.nrows) most = uniform(__builtin_amdgcn_readlane(lim[rb], 31));
  }
  drain_memory();

  const int piece16 = ((lane & 7) ^ swz(lane >> 3)) * 16;
  const uint32_t k_off = (uint32_t)((lane >> 3) * a.ks.slot) + piece16;
  const uint32_t v_off = ALIKE ? k_off : (uint32_t)((lane >> 3) * a.vs.slot) + piece16;
  const int* trow = a.table + it.sequence * a.table_stride;
  const int stages = (it.key1 - it.key0 + 63) >> 6;
  f32x16 acc[2][2];
  RowState st[2];
  const float c = a.scale_log2, inv_c = 1.f / c;
  float top[2];  // scores from which a row's shift moves

  // A wave fetches keys 16 wave .. + 15 of a stage: two groups of eight, in one page
  // where the page size is a multiple of 16.  The table's entries of the stage that is
  // fetched next are loaded a stage ahead and checked when they are used (a check is
  // a wait for the load).
  const char* kbase = a.k + kvh * a.ks.head;
  const char* vbase = a.v + kvh * (ALIKE ? a.ks.head : a.vs.head);
  const bool one_page = a.page_size % 16 == 0;
  const PagedStrides& vs = ALIKE ? a.ks : a.vs;
  int entry[2];
  auto load_entries = [&](int s) {
    const int key = it.key0 + 64 * s + 16 * wave;
    entry[0] = page_of(a, trow, min(key, it.key1 - 1));
    if (!one_page) entry[1] = page_of(a, trow, min(key + 8, it.key1 - 1));
  };
  auto fetch = [&](int s) {
    char* slot = lds + (s & (kSlots - 1)) * kSlotBytes;
    const int key = it.key0 + 64 * s + 16 * wave;
    const int at = key - fast_div(key, a.div_page) * a.page_size;
    const uint32_t dst = uniform((int)lds_offset(slot + 16 * wave * kRowBytes));
    const bool whole = one_page && (unsigned)entry[0] < (unsigned)a.pages && key + 16 <= it.key1;
    if (whole) {
      const long long off = entry[0] * a.ks.page + at * a.ks.slot;
      const long long voff = ALIKE ? off : entry[0] * vs.page + at * vs.slot;
      dma16(kbase + off, k_off, dst);
      dma16(kbase + off + 8 * a.ks.slot, k_off, dst + 8 * kRowBytes);
      dma16(vbase + voff, v_off, dst + kTileBytes);
      dma16(vbase + voff + 8 * vs.slot, v_off, dst + kTileBytes + 8 * kRowBytes);
      lost[s & (kSlots - 1)][wave] = 0;
      return;
    }
    int gone = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int first = key + 8 * j;
      const int id = one_page ? entry[0] : entry[j];
      const bool page = (unsigned)id < (unsigned)a.pages;
      const bool there = page && first + (lane >> 3) < it.key1;
      const char* none = a.zeros + 16 * (lane & 7);
      dma16_lane(there ? a.k + row_offset(a, a.ks, page ? id : 0, first, kvh) + k_off : none,
                 dst + 8 * j * kRowBytes);
      dma16_lane(there ? a.v + row_offset(a, vs, page ? id : 0, first, kvh) + v_off : none,
                 dst + kTileBytes + 8 * j * kRowBytes);
      gone |= page ? 0 : 1 << (2 * wave + j);
    }
    lost[s & (kSlots - 1)][wave] = gone;  // bit g: keys 8 g .. of the stage have no page
  };
  const int tr_row = tr_row_of(lane), tr_col = tr_col_of(lane);
  auto read_keys = [&](const char* kt, int k0, bf16x8 (&k)[4]) {
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) k[ks] = tile_chunk(kt, k0 + (lane & 31), 2 * ks + (lane >> 5));
  };
  // scores of one 32-key block for both row blocks
  auto scores = [&](const bf16x8 (&k)[4], f32x16 (&out)[2]) {
    out[0] = out[1] = zero16();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      out[0] = mfma32x32x16(k[ks], qf[0][ks], out[0]);
      out[1] = mfma32x32x16(k[ks], qf[1][ks], out[1]);
    }
  };
  // One 32-key block: cur are its scores and mx their maxima; next and mx become
  // those of the block whose keys are rows k0 .. of kn.  The next block's first
  // product runs under this one's exponentials, its maxima under this one's second
  // product: a wave alone keeps both pipes in use.  The operands of both are read
  // first, under the check of the maxima.
  auto step = [&](int kb, int gone, f32x16 (&cur)[2], f32x16 (&next)[2], float (&mx)[2],
                  const char* kn, int k0, const char* vt, int v0) {
    bf16x8 k[4], v[2][2];
    read_keys(kn, k0, k);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < 2; ++db)
        v[j][db] = tile_tr_operand(vt, v0 + 16 * j + tr_row, db * 32 + tr_col);
    __builtin_amdgcn_sched_barrier(0);
    if (kb + 32 > least || gone) {
      const int at = opaque(kb);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        mask_scores(cur[rb], at, lim[rb], gone, lane);
        mx[rb] = column_max(cur[rb]);
      }
    }
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
      if (__any(mx[rb] > top[rb])) {
        grow(st[rb], fmaf(halves_max(mx[rb]), c, -st[rb].shift), acc[rb]);
        top[rb] = (st[rb].shift + st[rb].lag) * inv_c;
      }
    scores(k, next);
    bf16x8 p[2][2];
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) block_probs(cur[rb], st[rb], c, p[rb][0], p[rb][1]);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        acc[0][db] = mfma32x32x16(v[j][db], p[0][j], acc[0][db]);
        acc[1][db] = mfma32x32x16(v[j][db], p[1][j], acc[1][db]);
      }
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) mx[rb] = column_max(next[rb]);
  };

#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    acc[rb][0] = acc[rb][1] = zero16();
    st[rb] = {0.f, kNegInf, 0.f, 0.f};
    top[rb] = kNegInf;
  }
#pragma unroll
  for (int s = 0; s < kSlots - 1; ++s)
    if (s < stages) {
      load_entries(s);
      fetch(s);
    }
  if (kSlots - 1 < stages) load_entries(kSlots - 1);
  f32x16 sa[2], sb[2];
  float mx[2];
  for (int s = 0; s < stages; ++s) {
    // this wave's parts of stages s and s + 1 are there; the one behind may be on its way
    if (s + 2 < stages) wait_vm_lds<4>(); else wait_vm_lds<0>();
    barrier();
    if (s + kSlots - 1 < stages) {
      fetch(s + kSlots - 1);
      if (s + kSlots < stages) load_entries(s + kSlots);
    }
    const int4 lo = *reinterpret_cast<const int4*>(lost[s & (kSlots - 1)]);
    const int gone = uniform(lo.x | lo.y | lo.z | lo.w);
    const char* kt = lds + (s & (kSlots - 1)) * kSlotBytes;
    const char* vt = kt + kTileBytes;
    const char* kn = lds + ((s + 1) & (kSlots - 1)) * kSlotBytes;
    const int kb = it.key0 + 64 * s;
    if (kb >= most) continue;
    if (s == 0) {
      bf16x8 k[4];
      read_keys(kt, 0, k);
      scores(k, sa);
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) mx[rb] = column_max(sa[rb]);
    }
    // (behind the last stage the next block's scores are of whatever lies there, unused)
    step(kb, gone & 15, sa, sb, mx, kt, 32, vt, 0);
    step(kb + 32, gone >> 4, sb, sa, mx, kn, 0, vt, 32);
  }
  wait_vm_lds<0>();  // no DMA may still target this workgroup's LDS
  if (it.key1 > row_limit(a, it, 0)) {
    uint32_t wild = 0;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) wild |= wild_bits(acc[rb][0]) | wild_bits(acc[rb][1]);
    const bool mine = __any(wild != 0);
    flags[wave] = mine;
    __syncthreads();
    const int4 any = *reinterpret_cast<const int4*>(flags);
    if (uniform(any.x | any.y | any.z | any.w)) return false;
  }

  const int elane = fresh_lane_id();
  const int half = elane >> 5;
  if (it.partial < 0) {
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      const int row = 64 * wave + 32 * rb + (elane & 31);
      const float2 ml = mark_low(a, trow, it.key0, it.key1, lim[rb],
                                 st[rb].lag > 0.f ? st[rb].shift : kNegInf,
                                 halves_sum(st[rb].l0 + st[rb].l1));
      if (row >= it.nrows) continue;
      const RowOf ro = row_of(a, it, row, kvh);
      store_bf16_rows(reinterpret_cast<bf16*>(a.out + ((long long)ro.token * a.Hq + ro.head) * (kD * 2)),
                      acc[rb], row_factor(ml.x, ml.y), !no_weight(ml.y), half);
    }
    return true;
  }
  // Partial results go through LDS (16 KB of the ring a wave, 16-byte pieces of a row
  // permuted by the row), so that a store covers four whole rows.
  __syncthreads();  // every wave is done with the ring
  char* rows = lds + wave * kSlotBytes;
  const size_t first = (size_t)(kvh * a.cap_rows) + it.partial + 64 * wave;
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int r = 32 * rb + (elane & 31);
    const float2 ml = mark_low(a, trow, it.key0, it.key1, lim[rb],
                               st[rb].lag > 0.f ? st[rb].shift : kNegInf,
                               halves_sum(st[rb].l0 + st[rb].l1));
    if (half == 0 && 64 * wave + r < it.nrows) a.ml[first + r] = ml;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = acc[rb][db][4 * g + i];
        *reinterpret_cast<f32x4*>(rows + r * 256 + (((8 * db + 2 * g + half) ^ (r & 15)) << 4)) = x;
      }
  }
  wave_lds_fence();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = 4 * i + (elane >> 4), piece = elane & 15;
    if (64 * wave + r < it.nrows)
      *reinterpret_cast<f32x4*>(a.acc + (first + r) * kD + 4 * piece) =
          *reinterpret_cast<const f32x4*>(rows + r * 256 + ((piece ^ (r & 15)) << 4));
  }
  return true;
}

// Workgroups: the few-rows shares' (head pairs fastest) and the many-rows shares'
// (KV heads fastest, so that with 8 of them each XCD's L2 holds one head's keys), in
// turn 256 of each while there are both: one for every CU, so that a CU's two
// workgroups are one that waits for memory and one that computes, the longer of the
// many rows first (40 single tokens and three chunks 129 us; the other way round 152).
// ALIKE: the pools of keys and values have the same strides.
template <int HW, bool ALIKE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void paged_attn_bf16_kernel(PagedArgs a) {
  __shared__ __attribute__((aligned(16))) char lds[kSlots * kSlotBytes];
  __shared__ __attribute__((aligned(16))) float lm[4][64], ll[4][64];
  static_assert(4 * FewLds<HW>::kWave <= sizeof(lds), "the waves' blocks fit the ring");
  const int turn = blockIdx.x >> 8, both = 2 * min(a.few_turns, a.many_turns);
  const bool few = turn < both ? turn & 1 : a.few_turns > a.many_turns;
  const int block = (turn < both ? turn >> 1 : turn - both / 2) * 256 + (blockIdx.x & 255);
  if (few) {
    const int share = uniform(fast_div(block, a.div_pairs));
    if (share >= ld_const(a.head, kHeadShares + kFew)) return;
    const int pair = uniform(block - share * a.head_pairs);
    const int wave = uniform(threadIdx.x >> 6);
    const int end = ld_const(a.shares[kFew], share + 1);
    for (int item = ld_const(a.shares[kFew], share); item < end; ++item) {
      const ItemView it = load_item(a.items[kFew], item);
      if (it.nrows < 1) continue;
      few_rows<HW, ALIKE, false>(a, it, pair, wave, lds + wave * FewLds<HW>::kWave, lm[wave], ll[wave]);
      __syncthreads();
      few_merge<HW, kKeyWaves>(a, it, pair, 0, threadIdx.x, lds, lm, ll);
      __syncthreads();
    }
    return;
  }
  const int share = uniform(fast_div(block, a.div_hkv));
  if (share >= ld_const(a.head, kHeadShares + kMany)) return;
  const int kvh = uniform(block - share * a.Hkv);
  const int end = ld_const(a.shares[kMany], share + 1);
  for (int item = ld_const(a.shares[kMany], share); item < end; ++item) {
    const ItemView it = load_item(a.items[kMany], item);
    if (it.nrows < 1) continue;
    if (!many_rows<ALIKE>(a, it, kvh, lds, reinterpret_cast<int(*)[4]>(lm),
                          reinterpret_cast<int*>(ll)))
      many_again<ALIKE>(a, it, kvh, lds, lm, ll);
    __syncthreads();
  }
}

// --------------------------------------------------------------------------
// fp32: always up to 32 rows; the waves split the keys (32x32x2 MFMAs, rows staged
// through registers, as the packed fp32 forward).
// --------------------------------------------------------------------------
__device__ __forceinline__ void f32_item(const PagedArgs& a, const ItemView& it, int kvh,
                                         F32Tile (&kt)[4], F32Tile (&vt)[4], F32Tile& qt,
                                         float (&lm)[4][32], float (&ll)[4][32]) {
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

  f32x16 acc[2];
  float m, l;
  const float c = a.scale_log2;
  auto run = [&](auto how) {
    constexpr bool careful = decltype(how)::value;
    acc[0] = acc[1] = zero16();
    m = kNegInf;
    l = 0.f;
    int b = wave;
    if (b < blocks) fetch(b);
    if (!careful) __syncthreads();  // the query's rows
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
      const bool masked = kb + 32 > least || gone;
      wave_lds_fence();
      if (b + 4 < blocks) fetch(b + 4);
      f32x16 s = zero16();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const f32x4 kr = kt[wave].row4(lane, j), qr = qt.row4(lane, j);
#pragma unroll
        for (int e = 0; e < 4; ++e) s = mfma32x32x2(kr[e], qr[e], s);
      }
      if (masked) mask_scores(s, kb, lim, gone, lane);
      const float mx = halves_max(column_max(s));
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
      if (careful && masked) {
        // (as in the bf16 kernel)
#pragma unroll 1
        for (int key = 0; key < 32; ++key)
#pragma unroll
          for (int db = 0; db < 2; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float x = vt[wave].x[key * kF32Pitch + 32 * db + acc_row(r, lane)];
              const uint32_t mine = kb + key < lim ? wild_mask(x) : 0u;
              acc[db][r] = add_any(acc[db][r], __uint_as_float(__float_as_uint(x) & mine));
            }
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float v0 = vt[wave].col(lane, 0, r), v1 = vt[wave].col(lane, 1, r);
        if (careful && masked) {
          v0 = __uint_as_float(__float_as_uint(v0) & ~wild_mask(v0));
          v1 = __uint_as_float(__float_as_uint(v1) & ~wild_mask(v1));
        }
        acc[0] = mfma32x32x2(v0, s[r], acc[0]);
        acc[1] = mfma32x32x2(v1, s[r], acc[1]);
      }
    }
  };
  run(Plain{});
  if (it.key1 > least && __any((wild_bits(acc[0]) | wild_bits(acc[1])) != 0)) run(Careful{});
  const float2 ml = mark_low(a, trow, it.key0 + 32 * wave, it.key1, lim,
                             m == kNegInf ? kNegInf : m * c, halves_sum(l));
  if (lane < 32) {
    lm[wave][lane] = ml.x;
    ll[wave][lane] = ml.y;
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
    wt[w] = state_weight(lm[w][r], ll[w][r], top);
    sum = fmaf(wt[w], ll[w][r], sum);
  }
  const size_t at = (size_t)(kvh * a.cap_rows) + max(it.partial, 0) + r;
  const RowOf ro = row_of(a, it, r, kvh);
  const bool none = no_weight(sum);
  const float inv = it.partial >= 0 ? 1.f : row_factor(top, sum);
  float* dst = it.partial >= 0 ? a.acc + at * kD + d0
                               : reinterpret_cast<float*>(a.out) +
                                     ((long long)ro.token * a.Hq + ro.head) * kD + d0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) o += f32_at(kt[w], r, d0 + 4 * h) * wt[w];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = none ? 0.f : o[e] * inv;
    *reinterpret_cast<f32x4*>(dst + 4 * h) = o;
  }
  if (it.partial >= 0 && d0 == 0) a.ml[at] = make_float2(top, sum);
}

__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2)))
void paged_attn_f32_kernel(PagedArgs a) {
  __shared__ F32Tile kt[4], vt[4], qt;
  __shared__ float lm[4][32], ll[4][32];
  const int share = uniform(fast_div(blockIdx.x, a.div_hkv));
  if (share >= ld_const(a.head, kHeadShares + kFew)) return;
  const int kvh = uniform(blockIdx.x - share * a.Hkv);
  const int end = ld_const(a.shares[kFew], share + 1);
  for (int item = ld_const(a.shares[kFew], share); item < end; ++item) {
    const ItemView it = load_item(a.items[kFew], item);
    if (it.nrows < 1) continue;
    f32_item(a, it, kvh, kt, vt, qt, lm, ll);
    __syncthreads();
  }
}

// --------------------------------------------------------------------------
// Joins the items of split tiles, in item order: o = sum_i 2^(m_i - M) acc_i / sum_i
// 2^(m_i - M) l_i.  A workgroup takes up to 8 or 32 rows of a tile (join_rows) for one
// KV head: eight threads of a row take eight dims each, and the threads that are left
// share the items, four at a time in flight.  Workgroups past the rows zero the
// output rows that belong to no sequence, where that is asked for.  Bound: latency
// for few rows (4 us with the launch), and the partial results' way through the
// caches for many (a chunk of 2048 tokens: 34 MB in 11 us).
// --------------------------------------------------------------------------
template <bool F32>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  __shared__ float part[32][68];
  __shared__ float2 pml[32];
  if ((int)blockIdx.x >= a.join_blocks) {
    const long long row = (long long)a.Hq * kD * (F32 ? 4 : 2);
    const long long begin = ld_const(a.head, kHeadBegin) * row;
    const long long end = ld_const(a.head, kHeadEnd) * row;
    const long long at = (long long)(blockIdx.x - a.join_blocks) * 16384;
    for (long long x = at + 16 * threadIdx.x; x < min(at + 16384, a.out_bytes); x += 16 * 256)
      if (x < begin || x >= end) st_u32x4(a.out + x, u32x4{0, 0, 0, 0});
    return;
  }
  const int t = uniform(fast_div(blockIdx.x, a.div_hkv));
  if (t >= ld_const(a.head, kHeadJoins)) return;
  const int kvh = uniform(blockIdx.x - t * a.Hkv);
  const i32x8u j = ld_const8(a.joins, 8 * t);
  ItemView it = {};
  it.start = j[0];
  it.row0 = j[1];
  it.nrows = j[2];
  const int partial = j[3], splits = j[4], step = j[5];
  const int log_rp = it.nrows > 1 ? 32 - __builtin_clz(it.nrows - 1) : 0;
  const int sp = 32 >> log_rp;  // threads' groups that share a row's items
  const int slot = threadIdx.x >> 3, d0 = 8 * (threadIdx.x & 7);
  const int r = slot & ((1 << log_rp) - 1), share = slot >> log_rp;
  const int row = min(r, it.nrows - 1);
  const size_t base = (size_t)(kvh * a.cap_rows) + partial + row;
  float m = kNegInf, l = 0.f, o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = 0.f;
  for (int s0 = share; s0 < splits; s0 += 4 * sp) {
    float2 ml[4];
    f32x4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (past the last item its results again, which then count as none)
      const size_t at = base + (size_t)min(s0 + i * sp, splits - 1) * step;
      ml[i] = a.ml[at];
      x[i] = *reinterpret_cast<const f32x4*>(a.acc + at * kD + d0);
      y[i] = *reinterpret_cast<const f32x4*>(a.acc + at * kD + d0 + 4);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (s0 + i * sp >= splits) {
        ml[i] = make_float2(kNegInf, 0.f);
        x[i] = y[i] = f32x4{0.f, 0.f, 0.f, 0.f};  // (0 times an infinity is NaN)
      }
      top = fmaxf(top, ml[i].x);
    }
    const float wa = state_weight(m, l, top);
    l *= wa;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] *= wa;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = state_weight(ml[i].x, ml[i].y, top);
      l = fmaf(w, ml[i].y, l);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[e] = fmaf(w, x[i][e], o[e]);
        o[4 + e] = fmaf(w, y[i][e], o[4 + e]);
      }
    }
    m = top;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[slot][d0 + i] = o[i];
  if (d0 == 0) pml[slot] = make_float2(m, l);
  __syncthreads();
  // thread = (row, two dims): the shares in order
  const int e0 = 2 * (threadIdx.x & 31);
  for (int er = threadIdx.x >> 5; er < it.nrows; er += 8) {
    float top = kNegInf;
    for (int x = 0; x < sp; ++x) top = fmaxf(top, pml[(x << log_rp) + er].x);
    float sum = 0.f, z0 = 0.f, z1 = 0.f;
    for (int x = 0; x < sp; ++x) {
      const float2 ml = pml[(x << log_rp) + er];
      const float w = state_weight(ml.x, ml.y, top);
      sum = fmaf(w, ml.y, sum);
      z0 = fmaf(w, part[(x << log_rp) + er][e0], z0);
      z1 = fmaf(w, part[(x << log_rp) + er][e0 + 1], z1);
    }
    const RowOf ro = row_of(a, it, er, kvh);
    const bool none = no_weight(sum);
    const float inv = row_factor(top, sum);
    z0 = none ? 0.f : z0 * inv;
    z1 = none ? 0.f : z1 * inv;
    const long long at = ((long long)ro.token * a.Hq + ro.head) * kD + e0;
    if constexpr (F32) {
      *reinterpret_cast<float2*>(reinterpret_cast<float*>(a.out) + at) = make_float2(z0, z1);
    } else {
      const bf16x2 y = {(bf16)z0, (bf16)z1};
      *reinterpret_cast<bf16x2*>(reinterpret_cast<bf16*>(a.out) + at) = y;
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
  a.joins = reinterpret_cast<const int*>(p + lay.joins);
  for (int k = 0; k < 2; ++k) {
    a.shares[k] = reinterpret_cast<const int*>(p + lay.shares[k]);
    a.items[k] = reinterpret_cast<const int*>(p + lay.items[k]);
  }
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
  a.cap_rows = (long long)lay.cap_rows;
  a.head_pairs = Hkv / lay.head_pair;
  const int few_blocks = lay.target[kFew] * a.head_pairs;
  a.few_turns = (few_blocks + 255) / 256;
  a.many_turns = (lay.target[kMany] * Hkv + 255) / 256;
  a.join_blocks = lay.cap_joins * Hkv;
  a.div_pairs = make_fastdiv(a.head_pairs);
  a.scale_log2 = scale * kLog2e;
  a.div_g = make_fastdiv(a.G);
  a.div_page = make_fastdiv(page_size);
  a.div_hkv = make_fastdiv(Hkv);
  const long long rest = zero_rest ? (a.out_bytes + 16383) / 16384 : 0;
  const dim3 join((unsigned)(a.join_blocks + rest));
  if (f32) {
    hipLaunchKernelGGL(paged_attn_f32_kernel, dim3((unsigned)few_blocks), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(paged_join_kernel<true>, join, dim3(256), 0, stream, a);
    return hipGetLastError();
  }
  const dim3 grid(256u * (unsigned)(a.few_turns + a.many_turns));
  const bool alike = a.ks.page == a.vs.page && a.ks.slot == a.vs.slot && a.ks.head == a.vs.head;
  if (lay.head_pair == 2 && alike)
    hipLaunchKernelGGL((paged_attn_bf16_kernel<2, true>), grid, dim3(256), 0, stream, a);
  else if (lay.head_pair == 2)
    hipLaunchKernelGGL((paged_attn_bf16_kernel<2, false>), grid, dim3(256), 0, stream, a);
  else if (alike)
    hipLaunchKernelGGL((paged_attn_bf16_kernel<1, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attn_bf16_kernel<1, false>), grid, dim3(256), 0, stream, a);
  hipLaunchKernelGGL(paged_join_kernel<false>, join, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace mf
