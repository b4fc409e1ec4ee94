// Attention of several new tokens per sequence over a paged key-value cache that holds theirs
// already: a tree of drafted tokens, each of which sees the past and its own ancestors, or a chain.
//
// Sequence b of n cached tokens has the rows [cu[b], cu[b + 1]) of the queries, its last ones: with
// past = n - rows, new token i is at slot past + i. It sees the slots before `past` and the new
// tokens j whose bit j its row of `tree` has (a chain: j <= i); of these the last `window`.
// s_j = scale q . k_j, optionally capped to c tanh(s_j / c); out = sum_j softmax(s)_j v_j over what
// it sees, lse = log sum_j exp(s_j). Nothing seen: out = 0, lse = -inf.
//
// The (token, query head) pairs of a key head are the columns of every product: rows * heads per
// key head of them share each key and value. Few columns take the cache's bytes over the HBM rate;
// many take the products and, as long, the VALU's softmax. So each key and value is read once for
// all columns of a workgroup: its waves copy KT keys at a time into the LDS, straight from memory and
// a stage ahead, and WC of them take CT tiles of 16 columns each. Where that leaves waves without
// columns, WK waves share the columns and split a stage's keys; they join in the LDS at the end.
//
// Layout (16x16 MFMA, lane l, r = l % 16, c = l / 16):
// - S^T = K Q^T: lane l reads a chunk of key r; its accumulator holds keys 4 c + i of column r.
// - O^T = V^T P^T: the product over 32 keys gives lane l's slot j the key 4 c + j (j < 4) of the
//   first and of the second 16 keys, so that P is where S left it. 16-bit values come transposed
//   out of the LDS (tr_read4: 4 keys of one element); of others lane l reads VE consecutive elements
//   of those keys from element VE r on, and the m-th product takes element VE r + m of them.
// - A weight is two terms of the values' 16-bit type, a product each: 2^-17 of it is left out in
//   bf16 and 2^-22 in fp16 and e4m3 (whose values are exact in fp16). One term would be half a
//   step of the output's own type off in every weight, as much again as its rounding.
// - In the LDS a row's 16-byte chunks are swapped by its key's number, so that no two lanes of a
//   pass (256 bytes) meet in a bank: chunk x of key k is at x ^ k_swap(k) or x ^ v_swap(k). The
//   copy does it for nothing: each lane picks the chunk that belongs at its place.
//
// Work: the (chunk, block of WC CT 16 columns) pairs of all sequences are items, a workgroup each, of
// one key head. The chunks' length comes from all sequences' lengths and rows, on the device.
// Sequences of one chunk are finished here; the others leave (O, m, l) per chunk and column to the
// second kernel.
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_FP8 (the cache is e4m3), EK_DP (64, 128 or 256: the
// head dimension it is compiled for), EK_KT (keys of a stage: 16, 32 or 64), EK_CT (column tiles of
// a wave), EK_WC, EK_WK (waves over columns and over a stage's keys), EK_OCC (waves per SIMD that
// registers are left for).
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int DP = EK_DP, KT = EK_KT, CT = EK_CT, WC = EK_WC, WK = EK_WK, W = WC * WK;
constexpr int COLS = WC * CT * 16;                  // columns of a workgroup
constexpr int CS = EK_FP8 ? 1 : sizeof(T);          // bytes of a cache element
constexpr float LN2 = 0.69314718055994531f;
constexpr int NK = KT / 16 / WK;                    // score tiles of a wave and stage
constexpr int KE = 16 / CS;                         // elements of a chunk of 16 bytes
constexpr int KL = DP / (4 * KE);                   // key chunks per score tile and lane
constexpr bool TR = CS == 2;                        // values come transposed out of the LDS
// Elements of a value read: 16 lanes cover at most the whole head.
constexpr int VE0 = EK_FP8 ? 8 : 4;
constexpr int VE = TR ? 1 : VE0 * 16 > DP ? DP / 16 : VE0;
constexpr int NP = DP / 16;                         // output tiles, VE of them from one value read
constexpr int VW = VE * CS / 4 < 1 ? 1 : VE * CS / 4;  // words of a value read
constexpr int CPR = DP * CS / 16;                   // chunks of a row in the LDS
constexpr int ROW = CPR * 16, PART = KT * ROW, STAGE = 2 * PART;   // bytes: keys, then values
constexpr int LOADS = KT * CPR / (64 * W);          // of a lane and stage, of keys and of values
constexpr int UNIT = 64;                            // keys: what chunks are multiples of
constexpr int PARTS = (WK - 1) * WC * CT * (NP * 1024 + 512);    // what waves leave each other
constexpr int LDS = 2 * STAGE > PARTS ? 2 * STAGE : PARTS;
static_assert(KT * CPR % (64 * W) == 0 && KT % (16 * WK) == 0, "a stage is shared evenly");
// Weights are exp2(s - m), with the difference taken of the scores as the product gave them (or
// capped) and scaled after that: the largest is 1 exactly, however large the scores are. fp16 terms
// are lifted by 2^14: they keep a weight down to 2^-39 of the largest one.
constexpr bool HALF = EK_Q == 1 || EK_FP8;          // the weights' terms are fp16
constexpr int TERMS = 2;
constexpr float LIFT = HALF ? 0x1p14f : 1.0f;

typedef uint32_t u32;
template <int N> struct words { u32 w[N]; };
template <int N> EK_INLINE words<N> load_words(const char* p) {
  words<N> r;
  ek::vload_u<uint8_t, N * 4>((uint8_t*)r.w, (const uint8_t*)p);
  return r;
}
template <int N> EK_INLINE words<N> lds_words(const char* p) {
  words<N> r;
  ek::vload<uint8_t, N * 4>((uint8_t*)r.w, (const uint8_t*)p);
  return r;
}

struct Params {
  const T* q;
  const char* k;
  const char* v;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  const uint32_t* tree;              // [tokens, words], or null: chains
  T* out;
  float* lse;
  float* part;   // [slot][key head][column][dim]: O (lifted); then as many (m (not scaled), l);
                 // then a Row for each token; or null: no sequence has two chunks
  int64_t q_row, q_head, out_row, out_head;   // elements
  int64_t c_page, c_token, c_head;   // bytes
  int64_t table_row, lens_step, cu_step, tree_row;      // elements
  int32_t tokens, batch, heads, kv_heads, group, dim, page, pages, capacity, window, words;
  uint32_t page_mul;
  int32_t page_shift, items, slots, min_units;
  uint32_t q_sign;                   // the sign bits of the queries' words, if scale is negative
  float scale, cap, v_scale;         // scale > 0, with log2(e); cap in the same unit, or 0
};

// Where a token's parts are: its index among its sequence's new ones, the first slot of the
// sequence, its chunks and its blocks of columns.
struct Row { int32_t index, slot, chunks, blocks; };

EK_INLINE float* part_ml(const Params& a) {
  return a.part + (int64_t)a.slots * a.kv_heads * COLS * a.dim;
}
EK_INLINE Row* part_rows(const Params& a) {
  return (Row*)(part_ml(a) + (int64_t)a.slots * a.kv_heads * COLS * 2);
}

EK_INLINE int page_of(const Params& a, int key) {
  return a.page == 1 ? key : (int)(__umulhi((u32)key, a.page_mul) >> a.page_shift);
}

template <typename OP, typename X> EK_INLINE X wave_all(X x) {
  x = ek::reduce_xor<OP, 1>(x);
  x = ek::reduce_xor<OP, 2>(x);
  x = ek::reduce_xor<OP, 4>(x);
  x = ek::reduce_xor<OP, 8>(x);
  x = ek::reduce_xor<OP, 16>(x);
  return ek::reduce_xor<OP, 32>(x);
}

// A sequence: its first row, how many, the slot of its first new token (negative where it has more
// rows than tokens), and its keys, [first, end).
struct Seq { int begin, rows, past, first, end; };

EK_INLINE Seq seq_of(const Params& a, int b) {
  Seq s = {0, 0, 0, 0, 0};
  const int i = b < a.batch ? b : a.batch - 1;
  int begin = a.cu[i * a.cu_step], end = a.cu[(i + 1) * a.cu_step], len = a.lens[i * a.lens_step];
  begin = begin < 0 ? 0 : begin > a.tokens ? a.tokens : begin;
  end = end < begin ? begin : end > a.tokens ? a.tokens : end;
  len = len < 0 ? 0 : len;
  s.begin = begin;
  s.rows = b < a.batch ? end - begin : 0;
  s.past = len - s.rows;
  s.end = len < a.capacity ? len : a.capacity;
  // the first key that any row may see: a tree's row may have no bit at all
  const int from = s.past + (a.tree ? 0 : 1) - a.window;
  s.first = a.window > 0 && from > 0 ? (from < s.end ? from : s.end) : 0;
  return s;
}

EK_INLINE int blocks_of(const Params& a, const Seq& s) {
  return (int)(((int64_t)s.rows * a.group + COLS - 1) / COLS);
}
EK_INLINE int units_of(const Seq& s) { return (s.end - s.first + UNIT - 1) / UNIT; }
// A sequence without keys has a chunk as well: its rows become zeros.
EK_INLINE int chunks_of(int units, int per) {
  return units == 0 ? 1 : (int)((u32)(units + per - 1) / (u32)per);
}

struct Item {
  int b;                             // the sequence; -1: nothing to do
  int block, blocks, chunk, chunks, slot;   // slot: the sequence's first, of those with parts
};

// The items of all sequences in their order are 0, 1, ...: a chunk has as many units of UNIT keys
// as give `items` of them in all, and at most one more for each block of columns. Slots are
// counted over the sequences with several chunks alone, of which there are at most 2 `items`.
// Every wave finds its own from lengths and rows, 64 sequences at a time, a lane each.
EK_INLINE Item find_item(const Params& a, int item, Seq& found) {
  const int lane = ek::lane_id();
  const Seq s0 = seq_of(a, lane);
  int total = blocks_of(a, s0) * units_of(s0);
  for (int base = 64; base < a.batch; base += 64) {
    const Seq s = seq_of(a, base + lane);
    total += blocks_of(a, s) * units_of(s);
  }
  total = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(total));
  int per = (int)((u32)(total + a.items - 1) / (u32)a.items);
  // without room for parts each has one chunk, as when rows enough for all items are there
  per = !a.part ? 1 << 30 : per < a.min_units ? a.min_units : per;
  Item it = {-1, 0, 0, 0, 0, 0};
  int before = 0, slots = 0;
  for (int base = 0; base < a.batch; base += 64) {
    const Seq s = base == 0 ? s0 : seq_of(a, base + lane);
    const int blocks = blocks_of(a, s), chunks = chunks_of(units_of(s), per);
    const int mine = blocks * chunks, held = chunks > 1 ? mine : 0;
    const int end = before + ek::wave_prefix_sum(mine), slot = slots + ek::wave_prefix_sum(held);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item < end);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      const auto get = [&](int x) { return __builtin_amdgcn_readlane(x, at); };
      it.blocks = get(blocks);
      it.chunks = get(chunks);
      const int local = item - (get(end) - get(mine));
      // rows that descend may break the sums above
      if (local < 0 || it.blocks <= 0 || local >= get(mine)) return it;
      it.b = base + at;
      it.slot = get(slot) - get(held);
      it.chunk = (int)((u32)local / (u32)it.blocks);
      it.block = local - it.chunk * it.blocks;
      found = {get(s.begin), get(s.rows), get(s.past), get(s.first), get(s.end)};
      return it;
    }
    before = __builtin_amdgcn_readlane(end, 63);
    slots = __builtin_amdgcn_readlane(slot, 63);
  }
  return it;
}

EK_INLINE float tanh_f(float x) {
  const float y = __builtin_fabsf(x);
  // below 0.35 the odd series (Taylor, to x^11: off by less than 2e-8 of it), above it
  // (1 - e) / (1 + e), e = exp(-2 y), whose difference keeps its digits there
  const float z = y * y;
  float s = __builtin_fmaf(z, -1382.0f / 155925.0f, 62.0f / 2835.0f);
  s = __builtin_fmaf(z, s, -17.0f / 315.0f);
  s = __builtin_fmaf(z, s, 2.0f / 15.0f);
  s = __builtin_fmaf(z, s, -1.0f / 3.0f);
  s = __builtin_fmaf(z * s, y, y);
  const float e = ek::exp2_fast(y * -2.8853900817779268f);
  const float r = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  return __builtin_copysignf(y < 0.35f ? s : r, x);
}

#if EK_FP8
// Four e4m3 values as four fp16 ones, or bf16 ones (exact).
template <bool FP16> EK_INLINE void widen4(u32 w, u32* lo, u32* hi) {
  if constexpr (FP16) {
    *lo = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    *hi = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
  } else {
    *lo = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    *hi = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
  }
}
#endif

#if EK_Q != 0
// acc += a b over 32 k values: four words of 16-bit pairs per lane and operand.
template <bool FP16> EK_INLINE void mma(ek::f32x4& acc, const u32* a, const u32* b) {
  if constexpr (FP16)
    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ek::pack<ek::f16x8>(a), ek::pack<ek::f16x8>(b),
                                                 acc, 0, 0, 0);
  else
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ek::pack<ek::bf16x8>(a),
                                                  ek::pack<ek::bf16x8>(b), acc, 0, 0, 0);
}
// acc += a b over 16 k values.
template <bool FP16> EK_INLINE void mma16(ek::f32x4& acc, const u32* a, const u32* b) {
  if constexpr (FP16)
    acc = __builtin_amdgcn_mfma_f32_16x16x16f16(ek::pack<ek::f16x4>(a), ek::pack<ek::f16x4>(b),
                                                acc, 0, 0, 0);
  else
    acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(ek::pack<ek::s16x4>(a),
                                                    ek::pack<ek::s16x4>(b), acc, 0, 0, 0);
}
EK_INLINE u32 pack2(_Float16 a, _Float16 b) {
  return (u32)__builtin_bit_cast(uint16_t, a) | (u32)__builtin_bit_cast(uint16_t, b) << 16;
}
// The two terms of two weights. bf16: the first is cut off, the second rounded.
EK_INLINE void split(float x0, float x1, u32& first, u32& second) {
  if constexpr (HALF) {
    const _Float16 h0 = (_Float16)x0, h1 = (_Float16)x1;
    first = pack2(h0, h1);
    second = pack2((_Float16)(x0 - (float)h0), (_Float16)(x1 - (float)h1));
  } else {
    const u32 u0 = ek::f32_bits(x0), u1 = ek::f32_bits(x1);
    first = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 y = {(__bf16)(x0 - ek::bits_f32(u0 & 0xFFFF0000u)),
                  (__bf16)(x1 - ek::bits_f32(u1 & 0xFFFF0000u))};
    second = __builtin_bit_cast(u32, y);
  }
}
#endif

// Whether a word of values holds one that is not finite.
EK_INLINE bool odd_word(u32 w) {
#if EK_FP8
  return ((w & 0x7F7F7F7Fu) + 0x01010101u & 0x80808080u) != 0;       // e4m3 has NaN alone
#elif EK_Q == 0
  return (w & 0x7F800000u) == 0x7F800000u;
#else
  constexpr u32 X = EK_Q == 1 ? 0x7C007C00u : 0x7F807F80u;
  constexpr u32 ONE = EK_Q == 1 ? 0x04000400u : 0x00800080u;
  return ((w & X) + ONE & 0x80008000u) != 0;
#endif
}
// A word with 0 for each value that is not finite.
EK_INLINE u32 finite_of(u32 w) {
  constexpr int BITS = CS * 8;
  u32 y = 0;
#pragma unroll
  for (int i = 0; i < 32; i += BITS) {
    const u32 one = w & (BITS == 32 ? ~0u : (1u << (BITS & 31)) - 1 << i);
    y |= odd_word(one) ? 0 : one;
  }
  return y;
}
// The value at p.
EK_INLINE float element(const char* p) {
#if EK_FP8
  return __builtin_amdgcn_cvt_f32_fp8((int)*(const uint8_t*)p, 0);
#else
  return ek::f32(*(const T*)p);
#endif
}

// The query columns as the products' operand: element chunk (i, c) of column r, in the order in
// which a lane reads its keys.
struct Query {
#if EK_Q == 0
  float w[KL][4];
#else
  u32 w[KL * KE / 8][4];
#endif
};

__device__ const u32 s_zeros[4] = {0, 0, 0, 0};

EK_INLINE int k_swap(int key) {
  return CPR >= 16 ? key & 15 : CPR == 8 ? key >> 1 & 7 : key >> 2 & 3;
}
EK_INLINE int v_swap(int key) {
  return !TR ? 0 : CPR >= 16 ? (key & 7) << 1 : (key >> 1 & 3) << 1;
}

// 16 bytes from `from` of each lane to LDS byte `lds` + 16 * lane. The compiler does not see the
// copy: whoever reads waits for vmcnt and a barrier.
EK_INLINE void copy16(u32 lds, const char* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               ::"s"(lds), "v"(from) : "memory", "m0");
}

// Word x of a row of the tree: what lies before the new tokens is seen, behind the mask nothing.
EK_INLINE u32 tree_word(const Params& a, const u32* row, int x) {
  return x < 0 ? ~0u : x < a.words ? row[x] : 0u;
}
// Bits [j, j + 4) of a row.
EK_INLINE u32 tree_bits(const Params& a, const u32* row, int j) {
  const int x = j >> 5;
  const uint64_t w = (uint64_t)tree_word(a, row, x + 1) << 32 | tree_word(a, row, x);
  return (u32)(w >> (j & 31)) & 15u;
}
// How many of bits [lo, hi) are set, lo >= 0.
EK_INLINE int tree_count(const Params& a, const u32* row, int lo, int hi) {
  int n = 0;
  for (int x = lo >> 5; x * 32 < hi && x < a.words; ++x) {
    u32 w = row[x];
    if (x * 32 < lo) w &= ~0u << (lo & 31);
    if (hi - x * 32 < 32) w &= (1u << (hi - x * 32)) - 1;
    n += __builtin_popcount(w);
  }
  return n;
}

EK_INLINE T result(float o, float f, bool any) { return ek::cvt<T>(any ? o * f : 0.0f); }

// What differences of the running maxima are multiplied by for exp2: capped scores are in log2 units.
EK_INLINE float scale_of(const Params& a) { return a.cap > 0.0f ? 1.0f : a.scale; }

extern "C" __global__ __launch_bounds__(64 * W, EK_OCC) void ek_tree_attention(Params a) {
  __shared__ __attribute__((aligned(1024))) char s_stage[LDS];
  const int lane = ek::lane_id(), r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wc = wave % WC, wk = wave / WC;
  const int g = blockIdx.y;
  Seq sq;
  const Item it = find_item(a, blockIdx.x, sq);
  if (it.b < 0) return;
  const int all = sq.rows * a.group;                          // columns of the sequence
  const int block0 = it.block * COLS, col0 = block0 + wc * CT * 16;   // this wave's first

  // this lane's column of each tile: its token, and its head of those of the key head
  const auto valid = [&](int t) { return col0 + t * 16 + r < all; };
  const auto column = [&](int t) { return valid(t) ? col0 + t * 16 + r : all - 1; };
  int index[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) index[t] = (int)((u32)column(t) / (u32)a.group);
  const auto head = [&](int t) { return column(t) - index[t] * a.group; };
  if (a.part && it.chunk == 0 && g == 0 && wk == 0 && c == 0) {
    // for the second kernel, by the column of each token's first head
#pragma unroll
    for (int t = 0; t < CT; ++t)
      if (valid(t) && head(t) == 0)
        part_rows(a)[sq.begin + index[t]] = {index[t], it.slot, it.chunks, it.blocks};
  }

  // units are spread evenly over the chunks: the first few have one more
  const int units = units_of(sq), each = units / it.chunks, more = units - each * it.chunks;
  const int lo_u = it.chunk * each + (it.chunk < more ? it.chunk : more);
  const int hi_u = lo_u + each + (it.chunk < more);
  int lo = sq.first + lo_u * UNIT;
  int hi = hi_u >= units ? sq.end : sq.first + hi_u * UNIT;
  // where each column's keys begin, and (a tree) whether its window ends among the new tokens
  int from[CT];
  bool deep = false;
  const u32* row[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    row[t] = a.tree ? a.tree + (sq.begin + index[t]) * a.tree_row : nullptr;
    from[t] = 0;
    if (a.window > 0) {
      int seen = index[t] + 1;
      if (a.tree) seen = tree_count(a, row[t], sq.past < 0 ? -sq.past : 0, sq.end - sq.past);
      from[t] = sq.past + seen - a.window;
      deep |= a.tree && seen > a.window;
    }
  }
  deep = __builtin_amdgcn_ballot_w64(deep) != 0;
  // Whether a column may not see a key before `next` from `base` on that is there: new ones, and
  // where windows begin (one for all waves: no column's begins behind this).
  const int from_most = a.window > 0 ? sq.past + sq.rows - a.window : 0;
  const auto edge = [&](int base) { return base + KT > sq.past || base < from_most; };
  if (!a.tree) {
    // a block of a chain: no key behind its last token, none before the window of its first
    const int last = block0 + COLS < all ? block0 + COLS : all;
    const int stop = sq.past + (last - 1) / a.group + 1;
    hi = hi < stop ? hi : stop;
    if (a.window > 0) {
      const int begin = sq.past + block0 / a.group + 1 - a.window;
      if (begin > lo) lo += (begin - lo) / UNIT * UNIT;
    }
  }

  const char* kbase = a.k + g * a.c_head;
  const char* vbase = a.v + g * a.c_head;
  const int32_t* table = a.table + it.b * a.table_row;
  const char* zeros = (const char*)s_zeros;
  const u32 lds = ek::lds_addr(s_stage);
  const int row_bytes = a.dim * CS;

  // The page of key base + lane of a stage, read one stage before its keys; -1: none.
  const auto page_id = [&](int base) -> int {
    const int key = base + (lane & (KT - 1));
    return key < hi ? table[page_of(a, key)] : -1;
  };
  // This lane's key's offset in the cache (-1 where there is none), and which keys there are.
  const auto offset = [&](int base, int id, uint64_t& live) -> int64_t {
    const int key = base + (lane & (KT - 1));
    const bool ok = (u32)id < (u32)a.pages;
    live = __builtin_amdgcn_ballot_w64(ok);
    return ok ? id * a.c_page + (key - page_of(a, key) * a.page) * a.c_token : -1;
  };
  // A stage's keys and values on their way: zeros where there is no key, or no element of it.
  const auto fetch = [&](int stage, int64_t off) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int first = (k * W + wave) * 64, key = (first + lane) / CPR;
      const int chunk = (first + lane) % CPR;
      const int64_t o = ek::shfl(off, key);
      const int kc = (chunk ^ k_swap(key)) * 16, vc = (chunk ^ v_swap(key)) * 16;
      const u32 to = lds + stage * STAGE + first * 16;
      copy16(to, o >= 0 && kc < row_bytes ? kbase + o + kc : zeros);
      copy16(to + PART, o >= 0 && vc < row_bytes ? vbase + o + vc : zeros);
    }
  };

  uint64_t live = 0;
  int id = -1;
  if (lo < hi) {
    const int64_t off = offset(lo, page_id(lo), live);
    fetch(0, off);
    id = page_id(lo + KT);
  }

  Query q[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const T* src = a.q + (sq.begin + index[t]) * a.q_row + (g * a.group + head(t)) * a.q_head;
    constexpr int QN = sizeof(q[0].w) / 16, QE = 16 / sizeof(T);
    const auto place = [&](int i) {
      return EK_Q == 0 ? (i * 4 + c) * 4 : (i / (KE / QE) * 4 + c) * KE + i % (KE / QE) * 8;
    };
    words<4> x[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i)
      x[i] = load_words<4>((const char*)(src + (place(i) < a.dim ? place(i) : 0)));
#pragma unroll
    for (int i = 0; i < QN; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const u32 w = valid(t) && place(i) < a.dim ? x[i].w[k] ^ a.q_sign : 0;
        __builtin_memcpy(&q[t].w[i][k], &w, 4);
      }
  }

  // what the scores are multiplied by for exp2: positive, since the queries took the sign
  const float to_cap = a.cap > 0.0f ? a.scale / a.cap : 0.0f;
  const float scale = scale_of(a);
  float m[CT], l[CT];
  ek::f32x4 o[CT][NP];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    m[t] = -__builtin_inff(), l[t] = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; ++p) o[t][p] = ek::f32x4{0, 0, 0, 0};
  }
  // the element of the head that o[t][p][i] is
  const auto element_of = [&](int p, int i) {
    return p / VE * 16 * VE + (c * 4 + i) * VE + p % VE;
  };

  // (all waves: the loads of this stage have arrived, and are seen by the others)
  const auto arrive = [&] {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  arrive();
  int stage = 0;
  bool some_odd = false;
  for (int base = lo; base < hi; base += KT, stage ^= 1) {
    const int next = base + KT;
    uint64_t live_next = 0;
    if (next < hi) {
      fetch(stage ^ 1, offset(next, id, live_next));
      id = page_id(next + KT);
    }
    const char* keys = s_stage + stage * STAGE;
    const char* values = keys + PART;
    constexpr int K0 = 16;                            // keys of a tile
    const int tile0 = wk * NK;                        // this wave's first

    // scores: acc[t][s][i] is key 16 (tile0 + s) + 4 c + i of tile t's column r
    ek::f32x4 acc[CT][NK];
    words<4> kf[2][KL];                               // a tile's chunks, read a tile ahead
    const auto read_keys = [&](int s) {
#pragma unroll
      for (int i = 0; i < KL; ++i)
        kf[s & 1][i] = lds_words<4>(keys + ((tile0 + s) * K0 + r) * ROW +
                                    ((i * 4 + c) ^ k_swap(r)) * 16);
    };
    read_keys(0);
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      if (s + 1 < NK) read_keys(s + 1);
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t][s] = ek::f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const words<4>& k = kf[s & 1][i];
#if EK_Q == 0
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < CT; ++t)
            acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(ek::bits_f32(k.w[e]), q[t].w[i][e],
                                                             acc[t][s], 0, 0, 0);
#elif EK_FP8
        u32 x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) widen4<EK_Q == 1>(k.w[e], &x[2 * e], &x[2 * e + 1]);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          mma<EK_Q == 1>(acc[t][s], x, q[t].w[2 * i]);
          mma<EK_Q == 1>(acc[t][s], x + 4, q[t].w[2 * i + 1]);
        }
#else
#pragma unroll
        for (int t = 0; t < CT; ++t) mma<EK_Q == 1>(acc[t][s], k.w, q[t].w[i]);
#endif
      }
      __builtin_amdgcn_sched_barrier(0);              // no tile further ahead: registers
    }

    // softmax: scores and m stay as the product gave them (or capped, in log2 units) until exp2
    const bool full = live == ~0ull;
    const bool masks = edge(base);
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      if (a.cap > 0.0f) {
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][s][i] = a.cap * tanh_f(acc[t][s][i] * to_cap);
      }
      if (!full || masks) {
#pragma unroll
        for (int s = 0; s < NK; ++s) {
          const int at = (tile0 + s) * K0 + c * 4, key = base + at, j = key - sq.past;
          u32 ok = (u32)(live >> at) & 15u;
          if (masks) {
            if (a.tree) {
              if (next > sq.past) {
                ok &= tree_bits(a, row[t], j);
                if (deep) {
#pragma unroll 1
                  for (int i = 0; i < 4; ++i)
                    if (j + i >= 0 &&
                        tree_count(a, row[t], j + i, sq.end - sq.past) > a.window)
                      ok &= ~(1u << i);
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key + i < from[t] && key + i < sq.past) ok &= ~(1u << i);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key + i < from[t] || j + i > index[t]) ok &= ~(1u << i);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[t][s][i] = ok >> i & 1 ? acc[t][s][i] : -__builtin_inff();
        }
      }
      float mt = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = __builtin_fmaxf(mt, acc[t][s][i]);
      mt = ek::reduce_xor<ek::Max, 16>(mt);
      mt = ek::reduce_xor<ek::Max, 32>(mt);
      const float m_new = __builtin_fmaxf(m[t], mt);
      const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
      const float alpha = ek::exp2_fast((m[t] - m_use) * scale);
      m[t] = m_new;
      // most stages raise no column's maximum
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
        l[t] *= alpha;
#pragma unroll
        for (int p = 0; p < NP; ++p) o[t][p] *= alpha;
      }
#pragma unroll
      for (int s = 0; s < NK; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[t][s][i] = ek::exp2_fast((acc[t][s][i] - m_use) * scale);
          l[t] += acc[t][s][i];
        }
    }

    // A value that is not finite must not reach the columns that don't see its key, whose weight
    // is 0: it becomes 0, and what sees it NaN behind the loop.
    if (masks) {
      bool bad = false;
      char* at = s_stage + stage * STAGE + PART + (lane & (KT - 1)) * ROW;
#pragma unroll 4
      for (int i = 0; i < CPR; ++i) {
        const words<4> v = lds_words<4>(at + (i ^ k_swap(lane)) * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) bad |= odd_word(v.w[w]);
      }
      if (__builtin_amdgcn_ballot_w64(bad) != 0) {    // all waves see the same
        some_odd = true;
        __syncthreads();
        if (bad && wave == 0)
#pragma unroll 1
          for (int i = 0; i < ROW / 4; ++i) {
            u32* w = (u32*)(at + i * 4);
            *w = finite_of(*w);
          }
        __syncthreads();
      }
    }

#if EK_Q == 0
#pragma unroll
    for (int s = 0; s < NK; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = (tile0 + s) * K0 + c * 4 + j;
#pragma unroll
        for (int p = 0; p < NP; p += VE) {
          const words<VW> v = lds_words<VW>(values + key * ROW + (p * 16 + r * VE) * CS);
#pragma unroll
          for (int e = 0; e < VE; ++e)
#pragma unroll
            for (int t = 0; t < CT; ++t)
              o[t][p + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  ek::bits_f32(v.w[e]), acc[t][s][j], o[t][p + e], 0, 0, 0);
        }
      }
#else
    constexpr int SS = NK == 1 ? 1 : 2;               // score tiles of a product
#pragma unroll
    for (int s = 0; s < NK; s += SS) {
      u32 w_p[CT][TERMS][2 * SS];
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int i = 0; i < 2 * SS; ++i) {
          const ek::f32x4& x = acc[t][s + i / 2];
          split(x[i % 2 * 2] * LIFT, x[i % 2 * 2 + 1] * LIFT, w_p[t][0][i], w_p[t][1][i]);
        }
      const auto take = [&](int p, const u32* w) {
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int k = 0; k < TERMS; ++k) {
            if constexpr (SS == 1) mma16<HALF>(o[t][p], w, w_p[t][k]);
            else mma<HALF>(o[t][p], w, w_p[t][k]);
          }
      };
#if EK_FP8
#pragma unroll
      for (int p = 0; p < NP; p += VE) {
        // 4 SS keys' VE elements, 16 bits each
        u32 x[4 * SS][VE / 2];
#pragma unroll
        for (int j = 0; j < 4 * SS; ++j) {
          const int key = (tile0 + s + j / 4) * K0 + c * 4 + (j & 3);
          const words<VW> v = lds_words<VW>(values + key * ROW + p * 16 + r * VE);
#pragma unroll
          for (int w = 0; w < VW; ++w) widen4<HALF>(v.w[w], &x[j][2 * w], &x[j][2 * w + 1]);
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          u32 w[2 * SS];
#pragma unroll
          for (int i = 0; i < 2 * SS; ++i)
            w[i] = __builtin_amdgcn_perm(x[2 * i + 1][e / 2], x[2 * i][e / 2],
                                         e & 1 ? 0x07060302u : 0x05040100u);
          take(p + e, w);
        }
      }
#else
      const int key = (tile0 + s) * K0 + c * 4 + (lane >> 2 & 3);
      const char* at = values + key * ROW + (lane & 1) * 8;
      const int chunk = lane >> 1 & 1, swap = v_swap(key);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        u32 w[2 * SS];
#pragma unroll
        for (int i = 0; i < SS; ++i) {               // v_swap goes by the key within 8
          uint16_t x[4];
          ek::tr_read4(x, (const uint16_t*)(at + i * K0 * ROW + ((2 * p + chunk) ^ swap) * 16));
          __builtin_memcpy(&w[2 * i], x, 8);
        }
        take(p, w);
      }
#endif
    }
#endif
    live = live_next;
    arrive();
  }

  // The same stages' keys once more, one at a time: the elements of their values that are not finite.
  if (some_odd) {
#pragma unroll 1
    for (int key = lo; key < hi; ++key) {
      const int base = lo + (key - lo) / KT * KT, tile = (key - base) / 16;
      if (!edge(base) || tile / NK != wk) continue;
      const int page = table[page_of(a, key)], j = key - sq.past;
      if ((u32)page >= (u32)a.pages) continue;
      const char* v = vbase + page * a.c_page + (key - page_of(a, key) * a.page) * a.c_token;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        bool sees = key >= from[t] && j <= index[t];
        if (a.tree)
          sees = j < 0 ? key >= from[t]
                       : (tree_bits(a, row[t], j) & 1) &&
                             (!deep || tree_count(a, row[t], j, sq.end - sq.past) <= a.window);
        if (!sees) continue;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = element_of(p, i);
            if (d < a.dim && !(__builtin_fabsf(element(v + d * CS)) < __builtin_inff()))
              o[t][p][i] = __builtin_nanf("");
          }
      }
    }
  }

#pragma unroll
  for (int t = 0; t < CT; ++t) {
    l[t] = ek::reduce_xor<ek::Sum, 16>(l[t]);
    l[t] = ek::reduce_xor<ek::Sum, 32>(l[t]);
  }
  if constexpr (WK > 1) {
    // the waves of the same columns: to the first of them, in the order in which it holds its own
    float* part = (float*)s_stage;
    constexpr int SIZE = CT * (NP * 256 + 128);
    float* mine = part + ((wk - 1) * WC + wc) * SIZE;
    if (wk > 0) {
#pragma unroll
      for (int t = 0; t < CT; ++t) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
          *(ek::f32x4*)(mine + (t * NP + p) * 256 + lane * 4) = o[t][p];
        mine[CT * NP * 256 + t * 128 + lane] = m[t];
        mine[CT * NP * 256 + t * 128 + 64 + lane] = l[t];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int k = 0; k < WK - 1; ++k) {
      const float* other = part + (k * WC + wc) * SIZE;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const float mo = other[CT * NP * 256 + t * 128 + lane];
        const float lo = other[CT * NP * 256 + t * 128 + 64 + lane];
        const float top = __builtin_fmaxf(m[t], mo), use = top == -__builtin_inff() ? 0.0f : top;
        const float f = ek::exp2_fast((m[t] - use) * scale), fo = ek::exp2_fast((mo - use) * scale);
        m[t] = top;
        l[t] = l[t] * f + lo * fo;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const ek::f32x4 y = *(const ek::f32x4*)(other + (t * NP + p) * 256 + lane * 4);
          o[t][p] = o[t][p] * f + y * fo;
        }
      }
    }
  }

  // rows of VE or (transposed) 4 adjacent elements
  constexpr int OUT = TR ? 4 : VE;
  const auto each_run = [&](int t, const auto& put) {
    if constexpr (TR) {
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const float y[4] = {o[t][p][0], o[t][p][1], o[t][p][2], o[t][p][3]};
        put(p * 16 + c * 4, y);
      }
    } else {
#pragma unroll
      for (int p = 0; p < NP; p += VE)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) y[e] = o[t][p + e][i];
          put(p * 16 + (c * 4 + i) * VE, y);
        }
    }
  };
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    if (!valid(t)) continue;
    const int64_t token = sq.begin + index[t];
    const int h = g * a.group + head(t);
    if (it.chunks == 1) {
      const bool any = l[t] > 0.0f || l[t] != l[t];
      const float f = any ? a.v_scale / LIFT / l[t] : 0.0f;
      T* dst = a.out + token * a.out_row + h * a.out_head;
      each_run(t, [&](int d, const float* x) {
        T y[OUT];
#pragma unroll
        for (int e = 0; e < OUT; ++e) y[e] = result(x[e], f, any);
        if (d < a.dim) ek::vstore_u<T, OUT>(dst + d, y);
      });
      if (a.lse && c == 0)
        a.lse[token * a.heads + h] =
            any ? (m[t] * scale + __builtin_log2f(l[t])) * LN2 : -__builtin_inff();
    } else {
      const int slot = it.slot + it.chunk * it.blocks + it.block;
      if (!a.part || slot < 0 || slot >= a.slots) continue;
      const int64_t at = ((int64_t)slot * a.kv_heads + g) * COLS + wc * CT * 16 + t * 16 + r;
      float* dst = a.part + at * a.dim;
      each_run(t, [&](int d, const float* y) {
        if (d < a.dim) {
#pragma unroll
          for (int e = 0; e < OUT; e += 4) ek::vstore_u<float, 4>(dst + d + e, y + e);
        }
      });
      if (c == 0) {
        float* ml = part_ml(a) + at * 2;
        ml[0] = m[t];
        ml[1] = l[t];
      }
    }
  }
}

// Joins the chunks of a token's head, a wave each.
extern "C" __global__ __launch_bounds__(256) void ek_tree_attention_join(Params a) {
  constexpr int DW = (DP + 127) / 128;
  const int lane = ek::lane_id(), token = blockIdx.x;
  const int head = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (head >= a.heads || token < a.cu[0] || token >= a.cu[a.batch * a.cu_step]) return;
  const Row row = part_rows(a)[token];
  if (row.chunks <= 1 || row.slot < 0 || row.blocks <= 0 || row.index < 0 ||
      row.slot + (int64_t)row.chunks * row.blocks > a.slots)
    return;
  const int g = head / a.group, col = row.index * a.group + head - g * a.group;
  const int block = col / COLS;
  if (block >= row.blocks) return;
  const float scale = scale_of(a);
  const int64_t first = ((int64_t)(row.slot + block) * a.kv_heads + g) * COLS + col - block * COLS;
  const int64_t step = (int64_t)row.blocks * a.kv_heads * COLS;    // from chunk to chunk
  float m = -__builtin_inff(), l = 0.0f, x[DW][2];
#pragma unroll
  for (int k = 0; k < DW; ++k) x[k][0] = x[k][1] = 0.0f;
#pragma unroll 1
  for (int i0 = 0; i0 < row.chunks; i0 += 64) {
    // a lane each: the weights of 64 chunks
    const int i = i0 + lane;
    const float* ml = part_ml(a) + (first + (i < row.chunks ? i : i0) * step) * 2;
    const float mi = i < row.chunks ? ml[0] : -__builtin_inff();
    const float li = i < row.chunks ? ml[1] : 0.0f;
    const float m_new = __builtin_fmaxf(m, wave_all<ek::Max>(mi));
    const float mu = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float f = ek::exp2_fast((m - mu) * scale), w = ek::exp2_fast((mi - mu) * scale);
    l = l * f + wave_all<ek::Sum>(li * w);
    m = m_new;
#pragma unroll
    for (int k = 0; k < DW; ++k) x[k][0] *= f, x[k][1] *= f;
    const int count = row.chunks - i0 < 64 ? row.chunks - i0 : 64;
    for (int j = 0; j < count; ++j) {
      const float y = ek::bits_f32((u32)__builtin_amdgcn_readlane((int)ek::f32_bits(w), j));
      const float* src = a.part + (first + (i0 + j) * step) * a.dim;
#pragma unroll
      for (int k = 0; k < DW; ++k) {
        const int d = k * 128 + lane * 2;
        float v[2];
        ek::vload_u<float, 2>(v, src + (d < a.dim ? d : 0));
        x[k][0] = __builtin_fmaf(v[0], y, x[k][0]);
        x[k][1] = __builtin_fmaf(v[1], y, x[k][1]);
      }
    }
  }
  const bool any = l > 0.0f || l != l;
  const float f = any ? a.v_scale / LIFT / l : 0.0f;
  T* dst = a.out + token * a.out_row + head * a.out_head;
#pragma unroll
  for (int k = 0; k < DW; ++k) {
    const int d = k * 128 + lane * 2;
    if (d < a.dim) {
      T y[2] = {result(x[k][0], f, any), result(x[k][1], f, any)};
      ek::vstore_u<T, 2>(dst + d, y);
    }
  }
  if (a.lse && lane == 0)
    a.lse[(int64_t)token * a.heads + head] =
        any ? (m * scale + __builtin_log2f(l)) * LN2 : -__builtin_inff();
}
