// Attention of several new tokens per sequence over a paged key-value cache that holds theirs
// already: a tree of drafted tokens, each of which sees the past and its own ancestors, or a chain.
//
// Sequence b of n cached tokens has the rows [cu[b], cu[b + 1]) of the queries, its last ones: with
// past = n - rows, new token i is at slot past + i. It sees the slots before `past` and the new
// tokens j whose bit j its row of `tree` has (a chain: j <= i); of these, as far as the table goes,
// the last `window`.
// s_j = scale q . k_j, optionally capped to c tanh(s_j / c); out = sum_j softmax(s)_j v_j over what
// it sees, lse = log sum_j exp(s_j). Nothing seen: out = 0, lse = -inf.
//
// The (token, query head) pairs of a key head are the columns of every product: rows * heads per
// key head of them share each key and value. Few columns take the cache's bytes over the HBM rate;
// many take the products and, as long, the VALU's softmax. So each key and value is read once for
// all columns of a workgroup: its waves copy KT keys at a time into the LDS, straight from memory
// and a stage ahead, and WC of them take CT tiles of TILE columns each. Where that leaves waves
// without columns, WK waves share the columns and split a stage's keys; they join in the LDS at the
// end. Tiles are 32 columns wide where there are as many: an instruction holds up the VALU as long
// as one of 16 does and multiplies twice as much.
//
// Layout (lane l, r = l % TILE, c = l / TILE; runs of four keys, one for 16 columns, four for 32):
// - S^T = K Q^T: lane l reads a chunk of key r; its accumulator holds the runs' keys 4 c + i (32
//   columns: 8 s + 4 c + i) of column r.
// - O^T = V^T P^T: the product over two runs gives lane l's slots the keys of its own first and its
//   own second run, so that P is where S left it. 16-bit values come transposed out of the LDS
//   (tr_read4: 4 keys of one element); of others lane l reads VE consecutive elements of those keys
//   from element VE r on, and the m-th product takes element VE r + m of them.
// - A weight is some terms of the values' 16-bit type, a product each: three in bf16, which hold
//   it exactly, and two in fp16 and for e4m3 (whose values are exact in fp16), which leave out
//   2^-22 of it. Two in bf16 would leave out 2^-17: trees of up to 27 tokens in 64 sequences of up
//   to 8192 take 167 us with two and 187 with three, and 4.1 and 0.3 of 1000 results are not the
//   nearest to the exact ones.
// - In the LDS a row's 16-byte chunks are swapped by its key's number, so that no two lanes of a
//   pass (256 bytes) meet in a bank: chunk x of key k is at x ^ k_swap(k) or x ^ v_swap(k). The
//   copy does it for nothing: each lane picks the chunk that belongs at its place.
//
// Work: the (chunk, block of COLS columns) pairs of all sequences are items, a workgroup each, of
// one key head. The chunks' length comes from all sequences' lengths and rows, on the device.
// Sequences of one chunk are finished here; the others leave (O, m, l) per chunk and column to the
// second kernel.
//
// 128 columns over 131075 fp16 keys of 8 heads (537 MB, 103 GFLOP of products): 145 to 153 us and
// 10 to join, 3.3 to 3.5 TB/s. The copies alone take 100 us, the rest without them 101 (softmax and
// products in turn, each about half): one covers the other only in part. The matrix units are busy
// 38% of the time, 40% for the bf16 trees above: a stage's softmax has no product beside it, and
// the barriers keep a workgroup's waves in the same part of a stage. Some 33 columns of each of 24
// sequences of up to 16384 8-bit keys (156 MB): 78 us. A tree of 16 tokens after 1983 (8.4 MB, one
// stage for each workgroup): 14 us, of which 6 are the way to the first key (lengths, pages, keys:
// three reads, each waiting for the one before).
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_FP8 (the cache is e4m3), EK_DP (64, 128 or 256: the
// head dimension it is compiled for), EK_PAD (the head dimension is smaller), EK_KT (keys of a
// stage: 16, 32 or 64), EK_TILE (16 or 32: columns of a tile), EK_CT (tiles of
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
constexpr int DP = EK_DP, KT = EK_KT, TILE = EK_TILE, CT = EK_CT, WC = EK_WC, WK = EK_WK;
constexpr int W = WC * WK;
constexpr int COLS = WC * CT * TILE;                // columns of a workgroup
constexpr int NC = 64 / TILE;                       // lanes of a column
constexpr int CS = EK_FP8 ? 1 : sizeof(T);          // bytes of a cache element
constexpr float LN2 = 0.69314718055994531f;
constexpr int NK = KT / TILE / WK;                  // score tiles of a wave and stage
constexpr int RA = TILE * TILE / 256;               // runs of four keys of a lane in a tile
constexpr int RUNS = NK * RA;
constexpr int KE = 16 / CS;                         // elements of a chunk of 16 bytes
constexpr int KL = DP / (NC * KE);                  // key chunks per score tile and lane
constexpr bool TR = CS == 2;                        // values come transposed out of the LDS
// Elements of a value read: the lanes of a tile's rows cover at most the whole head.
constexpr int VE0 = EK_FP8 ? 8 : 4;
constexpr int VE = TR ? 1 : VE0 * TILE > DP ? DP / TILE : VE0;
constexpr int NP = DP / TILE;                       // output tiles, VE of them from one value read
constexpr int VW = VE * CS / 4 < 1 ? 1 : VE * CS / 4;  // words of a value read
constexpr int CPR = DP * CS / 16;                   // chunks of a row in the LDS
constexpr int ROW = CPR * 16, PART = KT * ROW, STAGE = 2 * PART;   // bytes: keys, then values
constexpr int LOADS = KT * CPR / (64 * W);          // of a lane and stage, of keys and of values
constexpr int UNIT = 64;                            // keys: what chunks are multiples of
constexpr int PARTS = (WK - 1) * WC * CT * (NP * RA * 1024 + 512);   // what waves leave each other
constexpr int LDS = 2 * STAGE > PARTS ? 2 * STAGE : PARTS;
static_assert(KT * CPR % (64 * W) == 0 && KT % (TILE * WK) == 0, "a stage is shared evenly");
static_assert(TR || VE * CS >= 4, "values are read in words");
// Weights are exp2(s - m), with the difference taken of the scores as the product gave them (or
// capped) and scaled after that: the largest is 1 exactly, however large the scores are. fp16 terms
// are lifted by 2^14: they keep a weight down to 2^-39 of the largest one.
constexpr bool HALF = EK_Q == 1 || EK_FP8;          // the weights' terms are fp16
constexpr int TERMS = HALF ? 2 : 3;
constexpr float LIFT = HALF ? 14.0f : 0.0f;        // log2, in the exponents: l is lifted too

#define EK_HERE __attribute__((always_inline))      // of a lambda: its captures stay in registers

typedef uint32_t u32;
typedef float Acc __attribute__((ext_vector_type(RA * 4)));    // of a tile
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
  int32_t page_shift, items, rounds, slots, join;
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

EK_INLINE float lane_value(float x, int lane) {
  return ek::bits_f32((u32)__builtin_amdgcn_readlane((int)ek::f32_bits(x), lane));
}
EK_INLINE int64_t lane_value(int64_t x, int lane) {
  const u32 lo = (u32)__builtin_amdgcn_readlane((int)(u32)(uint64_t)x, lane);
  return (int64_t)((uint64_t)(u32)__builtin_amdgcn_readlane((int)((uint64_t)x >> 32), lane) << 32 |
                   lo);
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
  // The first key that any row may see: a tree's row may have no bit at all. Where the table ends
  // before the new tokens, all see the same.
  const int from = (s.past < s.end ? s.past + (a.tree ? 0 : 1) : s.end) - a.window;
  s.first = a.window > 0 && from > 0 ? (from < s.end ? from : s.end) : 0;
  return s;
}

EK_INLINE int blocks_of(const Params& a, const Seq& s) {
  return (int)(((int64_t)s.rows * a.group + COLS - 1) / COLS);
}
EK_INLINE int units_of(const Seq& s) { return (s.end - s.first + UNIT - 1) / UNIT; }
// A sequence without keys has a chunk as well: its rows become zeros.
// There are few enough of them for a division that is off by one at most before it is put right.
EK_INLINE int chunks_of(int units, int per) {
  int n = (int)((float)(units + per - 1) * __builtin_amdgcn_rcpf((float)per));
  n += n * per < units;
  n -= (n - 1) * per >= units;
  return units == 0 ? 1 : n;
}

// A chunk of MOST_UNITS has all of any sequence (at most 2^30 tokens), and keeps the sums above in
// 32 bits.
constexpr int MOST_UNITS = (1 << 30) / UNIT;
EK_INLINE int even_share(int total, int items) {
  const u32 per = total <= items ? 1 : ((u32)total + (u32)items - 1) / (u32)items;
  return per < MOST_UNITS ? (int)per : MOST_UNITS;
}

struct Item {
  int b;                             // the sequence; -1: nothing to do
  int block, blocks, chunk, chunks, slot;   // slot: the sequence's first, of those with parts
};

// The items of all sequences in their order are 0, 1, ...: a chunk has as many units of UNIT keys
// as give `items` of them in all, and at most one more for each block of columns; or some more, so
// that there are at most `items`, or twice as many. Slots are counted over the sequences with
// several chunks alone, of which there are at most 2 `items`. Every wave finds its
// own from lengths and rows, 64 sequences at a time, a lane each.
EK_INLINE Item find_item(const Params& a, int item, Seq& found) {
  const int lane = ek::lane_id();
  const Seq s0 = seq_of(a, lane);
  int total = blocks_of(a, s0) * units_of(s0);
  for (int base = 64; base < a.batch; base += 64) {
    const Seq s = seq_of(a, base + lane);
    total += blocks_of(a, s) * units_of(s);
  }
  total = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(total));
  int per = even_share(total, a.items);
  // Each sequence may have a chunk more than its share for each of its blocks, and a few workgroups
  // beyond `items` make a round of their own. So the chunks are made as long as it takes for all of
  // them to fit into one round, or two where the grid has them, whichever ends first if a chunk
  // costs 3 units besides its own (24 sequences of up to 16384 8-bit keys: 5% less time than with
  // even shares; 64 of up to 8192 in two rounds: 8% less). Chunks of less than 8 units are not
  // worth two rounds (55 sequences of at most 189 keys: 10% more).
  if (a.batch <= 64) {
    int best = (per + 3) + ((per + 3) >> 1);          // of even shares, with a short round more
    const int all_blocks = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(blocks_of(a, s0)));
#pragma unroll 1
    for (int rounds = 1; rounds <= a.rounds; ++rounds) {
      // the even share, and what leaves room for a chunk more of every block but one
      const int room = rounds * a.items;
      int lo = even_share(total, room);
      if (room < all_blocks || (rounds > 1 && lo < 8)) continue;
      int hi = even_share(total, room - all_blocks + 1);
#pragma unroll 1
      for (int k = 0; k < 5 && lo < hi; ++k) {
        const int middle = (lo + hi) >> 1;
        const int all = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(
            blocks_of(a, s0) * chunks_of(units_of(s0), middle)));
        if (all <= room) hi = middle;
        else lo = middle + 1;
      }
      const int cost = rounds * (hi + 3);
      if (cost < best) best = cost, per = hi;
    }
  }
  // without room for parts each has one chunk, as when rows enough for all items are there
  if (!a.part) per = 1 << 30;
  Item it = {-1, 0, 0, 0, 0, 0};
  int before = 0, slots = 0;
  for (int base = 0; base < a.batch; base += 64) {
    Seq s = s0;
    if (base > 0) s = seq_of(a, base + lane);
    const int blocks = blocks_of(a, s), chunks = chunks_of(units_of(s), per);
    const int mine = blocks * chunks, held = chunks > 1 ? mine : 0;
    const int end = before + ek::wave_prefix_sum(mine), slot = slots + ek::wave_prefix_sum(held);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item < end);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      const auto get = [&](int x) EK_HERE { return __builtin_amdgcn_readlane(x, at); };
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

// tanh below 0.35: the odd series (Taylor, to x^11: off by less than 2e-8 of it).
EK_INLINE float tanh_small(float y) {
  const float z = y * y;
  float s = __builtin_fmaf(z, -1382.0f / 155925.0f, 62.0f / 2835.0f);
  s = __builtin_fmaf(z, s, -17.0f / 315.0f);
  s = __builtin_fmaf(z, s, 2.0f / 15.0f);
  s = __builtin_fmaf(z, s, -1.0f / 3.0f);
  return __builtin_fmaf(z * s, y, y);
}
constexpr float SMALL = 0.35f;
// Above it (1 - e) / (1 + e), e = exp(-2 y), whose difference keeps its digits there.
EK_INLINE float tanh_f(float x) {
  const float y = __builtin_fabsf(x), e = ek::exp2_fast(y * -2.8853900817779268f);
  const float r = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
  return __builtin_copysignf(y < SMALL ? tanh_small(y) : r, x);
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
// acc += a b: four words of 16-bit pairs per lane and operand, 32 (16x16) or 16 (32x32) k values.
#if EK_TILE == 32
#define EK_MFMA(type) __builtin_amdgcn_mfma_f32_32x32x16_##type
#else
#define EK_MFMA(type) __builtin_amdgcn_mfma_f32_16x16x32_##type
#endif
template <bool FP16> EK_INLINE void mma(Acc& acc, const u32* a, const u32* b) {
  if constexpr (FP16)
    acc = EK_MFMA(f16)(ek::pack<ek::f16x8>(a), ek::pack<ek::f16x8>(b), acc, 0, 0, 0);
  else acc = EK_MFMA(bf16)(ek::pack<ek::bf16x8>(a), ek::pack<ek::bf16x8>(b), acc, 0, 0, 0);
}
// The same over 16 k values of 16x16 tiles: two words.
template <bool FP16, typename A> EK_INLINE void mma_short(A& acc, const u32* a, const u32* b) {
  static_assert(sizeof(A) == 16);
  if constexpr (FP16)
    acc = __builtin_amdgcn_mfma_f32_16x16x16f16(ek::pack<ek::f16x4>(a), ek::pack<ek::f16x4>(b),
                                                acc, 0, 0, 0);
  else
    acc = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(ek::pack<ek::s16x4>(a),
                                                    ek::pack<ek::s16x4>(b), acc, 0, 0, 0);
}
typedef float f2 __attribute__((ext_vector_type(2)));
// The terms of two weights. bf16 cuts off: three of them are the 24 bits of a weight exactly.
EK_INLINE void split(float x0, float x1, u32 (&y)[TERMS]) {
  if constexpr (HALF) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 h = __builtin_convertvector((f2{x0, x1}), h2);
    y[0] = __builtin_bit_cast(u32, h);
    y[1] = __builtin_bit_cast(
        u32, __builtin_convertvector((f2{__builtin_fmaf((float)h[0], -1.0f, x0),
                                         __builtin_fmaf((float)h[1], -1.0f, x1)}), h2));
  } else {
#pragma unroll
    for (int k = 0; k < TERMS; ++k) {
      const u32 u0 = ek::f32_bits(x0), u1 = ek::f32_bits(x1);
      y[k] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
      x0 -= ek::bits_f32(u0 & 0xFFFF0000u);
      x1 -= ek::bits_f32(u1 & 0xFFFF0000u);
    }
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
// What has been seen of some words' values, in x, and another word: the larger magnitudes, or
// (e4m3) the carry out of the one magnitude that is not finite.
EK_INLINE u32 with_word(u32 x, u32 y) {
#if EK_FP8
  return x | (y & 0x7F7F7F7Fu) + 0x01010101u;
#elif EK_Q == 0
  y &= 0x7FFFFFFFu;
  return x > y ? x : y;
#else
  typedef uint16_t h2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(u32, __builtin_elementwise_max(
      __builtin_bit_cast(h2, x), __builtin_bit_cast(h2, y & 0x7FFF7FFFu)));
#endif
}
EK_INLINE bool any_odd(u32 seen) { return EK_FP8 ? (seen & 0x80808080u) != 0 : odd_word(seen); }
// A word with 0 for each value that is not finite.
EK_INLINE u32 finite_of(u32 w) {
  constexpr int BITS = CS * 8;
  u32 y = 0;
#pragma unroll
  for (int i = 0; i < 32; i += BITS) {
    const u32 one = w & (BITS == 32 ? ~0u : ((1u << (BITS & 31)) - 1) << i);
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
  if (!TR) return 0;
  if (TILE == 32) return CPR >= 16 ? (key & 3) << 2 : (key >> 1 & 1) << 2;
  return CPR >= 16 ? (key & 7) << 1 : (key >> 1 & 3) << 1;
}

// 16 (or 4) bytes from `from` of each lane to LDS byte `lds` + 16 (or 4) * lane. The compiler does
// not see the copy: whoever reads waits for it.
EK_INLINE void copy16(u32 lds, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               ::"s"(lds), "v"(from) : "memory", "m0");
}
EK_INLINE void copy4(u32 lds, const void* from) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off"
               ::"s"(lds), "v"(from) : "memory", "m0");
}
// Until at most the last N copies are on their way (copies arrive in order).
template <int N> EK_INLINE void wait_for() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Word x of a row of the tree: what lies before the new tokens is seen, behind the mask nothing.
EK_INLINE u32 tree_word(const Params& a, const u32* row, int x) {
  return x < 0 ? ~0u : x < a.words ? row[x] : 0u;
}
// Bits [j, j + 4) of a row, of which `first` holds the first 64.
EK_INLINE u32 tree_bits(const Params& a, const u32* row, uint64_t first, int j) {
  if (j < 0) return j <= -4 ? 15u : (u32)(first << -j | ((1u << -j) - 1)) & 15u;
  if (a.words <= 2) return j < 64 ? (u32)(first >> j) & 15u : 0u;
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

// What differences of the running maxima are multiplied by for exp2: capped scores are in log2
// units.
EK_INLINE float scale_of(const Params& a) { return a.cap > 0.0f ? 1.0f : a.scale; }

extern "C" __global__ __launch_bounds__(64 * W, EK_OCC) void ek_tree_attention(Params a) {
  __shared__ __attribute__((aligned(1024))) char s_stage[LDS];
  __shared__ int32_t s_ids[W][2][64];
  const int lane = ek::lane_id(), r = lane % TILE, c = lane / TILE;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wc = wave % WC, wk = wave / WC;
  const int g = blockIdx.y;
  Seq sq;
  const Item it = find_item(a, blockIdx.x, sq);
  if (it.b < 0) return;
  const int all = sq.rows * a.group;                          // columns of the sequence
  const int block0 = it.block * COLS, col0 = block0 + wc * CT * TILE;   // this wave's first

  // this lane's column of each tile, its token and its head (those of no column take the last)
  int index[CT], head[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int col = col0 + t * TILE + r, x = col < all ? col : all - 1;
    index[t] = (int)((u32)x / (u32)a.group);
    head[t] = g * a.group + x - index[t] * a.group;
  }
#define valid(t) (col0 + (t) * TILE + r < all)
#define tree_of(t) (a.tree + (sq.begin + index[t]) * a.tree_row)
  if (a.part && it.chunk == 0 && g == 0 && wk == 0 && c == 0) {
    // for the second kernel, by the column of each token's first head
#pragma unroll
    for (int t = 0; t < CT; ++t)
      if (valid(t) && head[t] == 0)
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
  uint64_t bits[CT];                                  // a tree's row's first 64
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    bits[t] = 0;
    if (a.tree) {
      bits[t] = tree_of(t)[0];
      if (a.words > 1) bits[t] |= (uint64_t)tree_of(t)[1] << 32;
    }
    from[t] = 0;
    if (a.window > 0) {
      if (a.tree) {
        const int seen = tree_count(a, tree_of(t), sq.past < 0 ? -sq.past : 0, sq.end - sq.past);
        from[t] = (sq.past < sq.end ? sq.past : sq.end) + seen - a.window;
        deep |= seen > a.window;
      } else {
        const int stop = sq.past + index[t] + 1;
        from[t] = (stop < sq.end ? stop : sq.end) - a.window;
      }
    }
  }
  deep = __builtin_amdgcn_ballot_w64(deep) != 0;
  // Whether a column may not see a key before `next` from `base` on that is there: new ones, and
  // where windows begin (one for all waves: no column's begins behind this).
  const int from_most = a.window > 0 ? sq.end - a.window : 0;
  const int past = sq.past;
  const auto edge = [past, from_most](int base) EK_HERE {
    return base + KT > past || base < from_most;
  };
  if (!a.tree) {
    // a block of a chain: no key behind its last token, none before the window of its first
    const int last = block0 + COLS < all ? block0 + COLS : all;
    const int stop = sq.past + (last - 1) / a.group + 1;
    hi = hi < stop ? hi : stop;
    if (a.window > 0) {
      const int first = sq.past + block0 / a.group + 1;
      const int begin = (first < sq.end ? first : sq.end) - a.window;
      if (begin > lo) lo += (begin - lo) / UNIT * UNIT;
    }
  }

  const char* kbase = a.k + g * a.c_head;
  const char* vbase = a.v + g * a.c_head;
  const int32_t* table = a.table + it.b * a.table_row;
  const char* zeros = (const char*)s_zeros;
  const u32 lds = ek::lds_addr(s_stage);
  const int row_bytes = a.dim * CS;

  // The page of key base + lane of a stage (`ids` of two stages in turn): copied into the LDS a
  // stage before its keys are, by every wave for itself. There is one at every address read here.
  const auto fetch_ids = [&](int ids, int base) EK_HERE {
    const int key = base + (lane & (KT - 1)), last = hi - 1;
    copy4(ek::lds_addr(s_ids[wave][ids]), table + page_of(a, key < last ? key : last));
  };
  // This lane's key's offset in the cache (-1 where there is none), and which keys there are.
  const auto offset = [&](int ids, int base, uint64_t& live) EK_HERE -> int64_t {
    const int key = base + (lane & (KT - 1)), id = s_ids[wave][ids][lane];
    const bool ok = key < hi && (u32)id < (u32)a.pages;
    live = __builtin_amdgcn_ballot_w64(ok);
    return ok ? id * a.c_page + (key - page_of(a, key) * a.page) * a.c_token : -1;
  };
  // A stage's keys or values on their way: zeros where there is no key, or no element of it.
  const auto fetch = [&](int to, const char* from, const auto& swap, int64_t off,
                         bool full) EK_HERE {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int first = (k * W + wave) * 64, key = (first + lane) / CPR;
      const int byte = (((first + lane) % CPR) ^ swap(key)) * 16;
      const int64_t o = ek::shfl(off, key);
      if (!EK_PAD && full) copy16(lds + to + first * 16, from + o + byte);
      else copy16(lds + to + first * 16, o >= 0 && byte < row_bytes ? from + o + byte : zeros);
    }
  };
  const auto swap_k = [](int key) EK_HERE { return k_swap(key); };
  const auto swap_v = [](int key) EK_HERE { return v_swap(key); };

  uint64_t live = 0;
  if (lo < hi) {
    fetch_ids(0, lo);
    fetch_ids(1, lo + KT);
    wait_for<0>();
    const int64_t off = offset(0, lo, live);
    fetch(0, kbase, swap_k, off, live == ~0ull);
    fetch(PART, vbase, swap_v, off, live == ~0ull);
  }

  Query q[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const T* src = a.q + (sq.begin + index[t]) * a.q_row + head[t] * a.q_head;
    constexpr int QN = sizeof(q[0].w) / 16, QE = 16 / sizeof(T);
    const auto place = [&](int i) EK_HERE {
      return EK_Q == 0 ? (i * NC + c) * 4 : (i / (KE / QE) * NC + c) * KE + i % (KE / QE) * 8;
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
  Acc o[CT][NP];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    m[t] = -__builtin_inff(), l[t] = 0.0f;
#pragma unroll
    for (int p = 0; p < NP; ++p) o[t][p] = Acc{} * 0.0f;
  }
  // the element of the head that o[t][p][i] is
  const auto element_of = [&](int p, int i) EK_HERE {
    return p / VE * TILE * VE + (i / 4 * 8 + c * 4 + i % 4) * VE + p % VE;
  };

  // A stage's copies are waited for where they are needed: its keys at the end of the stage before
  // (its values, the last that were issued, may still be on their way), its values before their
  // products. A barrier behind the wait: the other waves' copies too.
  wait_for<0>();
  __syncthreads();
  int stage = 0;
  bool some_odd = false;
  for (int base = lo; base < hi; base += KT, stage ^= 1) {
    const int next = base + KT, to = (stage ^ 1) * STAGE;
    uint64_t live_next = 0;
    const char* keys = s_stage + stage * STAGE;
    const char* values = keys + PART;
    const int key0 = wk * NK * TILE;                  // this wave's first
    // the first of the four keys of a lane's run s
    const auto run_key = [&](int s) EK_HERE {
      return key0 + s / RA * TILE + s % RA * 8 + c * 4;
    };

    // a tile's chunks, read AHEAD tiles before they are used
    constexpr int AHEAD = NK > 2 ? 2 : 1;
    words<4> kf[AHEAD + 1][KL];
    const auto read_keys = [&](int s) EK_HERE {
#pragma unroll
      for (int i = 0; i < KL; ++i)
        kf[s % (AHEAD + 1)][i] = lds_words<4>(keys + (key0 + s * TILE + r) * ROW +
                                              ((i * NC + c) ^ k_swap(r)) * 16);
    };
#pragma unroll
    for (int s = 0; s < AHEAD && s < NK; ++s) read_keys(s);
    if (next < hi) {
      const int64_t off = offset(stage ^ 1, next, live_next);
      fetch(to, kbase, swap_k, off, live_next == ~0ull);
      fetch_ids(stage, next + KT);
      fetch(to + PART, vbase, swap_v, off, live_next == ~0ull);
    }
    // scores: run s's keys and tile t's column r are at score(t, s, 0) to (t, s, 3)
    Acc acc[CT][NK];
#define score(t, s, i) acc[t][(s) / RA][(s) % RA * 4 + (i)]
#pragma unroll
    for (int s = 0; s < NK; ++s) {
      if (s + AHEAD < NK) read_keys(s + AHEAD);
      __builtin_amdgcn_sched_barrier(0);              // the reads before what they hide behind
#pragma unroll
      for (int t = 0; t < CT; ++t) acc[t][s] = Acc{} * 0.0f;
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const words<4>& k = kf[s % (AHEAD + 1)][i];
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
    float less[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      if (a.cap > 0.0f) {
        // most scores are small next to their cap: where all are, without the other form
        float most = 0.0f;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            score(t, s, i) *= to_cap;
            most = __builtin_fmaxf(most, __builtin_fabsf(score(t, s, i)));
          }
        const bool small = __builtin_amdgcn_ballot_w64(most >= SMALL) == 0;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            score(t, s, i) = a.cap * (small ? tanh_small(score(t, s, i)) : tanh_f(score(t, s, i)));
      }
      if (!full || masks) {
        // four bits for each run
        u32 ok = 0;
#pragma unroll 1
        for (int s = 0; s < RUNS; ++s) {
          const int at = run_key(s), key = base + at, j = key - sq.past;
          u32 run = (u32)(live >> at) & 15u;
          if (masks) {
            if (a.tree) {
              run &= tree_bits(a, tree_of(t), bits[t], j);
              if (deep) {
#pragma unroll 1
                for (int i = 0; i < 4; ++i)
                  if (j + i >= 0 &&
                      tree_count(a, tree_of(t), j + i, sq.end - sq.past) > a.window)
                    run &= ~(1u << i);
              }
            } else {
              const int n = index[t] - j + 1;            // of the run that the token sees
              run &= n <= 0 ? 0u : n < 4 ? (1u << n) - 1 : 15u;
            }
            // before the window: all keys of a chain, those before the new ones of a tree
            const int stop = a.tree && from[t] > sq.past ? sq.past : from[t];
            const int n = stop - key;
            run &= n <= 0 ? 15u : n < 4 ? 15u << n : 0u;
          }
          ok |= run << s * 4;
        }
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            score(t, s, i) = ok >> (s * 4 + i) & 1 ? score(t, s, i) : -__builtin_inff();
      }
      float mt = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < RUNS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = __builtin_fmaxf(mt, score(t, s, i));
      if constexpr (TILE == 16) mt = ek::reduce_xor<ek::Max, 16>(mt);
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
      // The weights are exp2(scale (s - m)): in one step where scale m is off by no more than
      // 2^-17 (as a 32-bit score of that size is by itself), else the difference first.
      const float top = m_use * scale;
      less[t] = LIFT - top;
      if (__builtin_amdgcn_ballot_w64(!(__builtin_fabsf(top) < 256.0f)) != 0) {
        less[t] = LIFT;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) score(t, s, i) -= m_use;
      }
    }
    const auto weigh = [&](int s) EK_HERE {
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          score(t, s, i) = ek::exp2_fast(__builtin_fmaf(score(t, s, i), scale, less[t]));
          l[t] += score(t, s, i);
        }
    };

    if (next < hi) wait_for<2 * LOADS + 1>();
    else wait_for<0>();
    __syncthreads();
    // A value that is not finite must not reach the columns that don't see its key, whose weight
    // is 0: it becomes 0, and what sees it NaN behind the loop.
    if (masks) {
      u32 seen = 0;
      char* at = s_stage + stage * STAGE + PART + (lane & (KT - 1)) * ROW;
#pragma unroll 4
      for (int i = 0; i < CPR; ++i) {
        const words<4> v = lds_words<4>(at + (i ^ k_swap(lane)) * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) seen = with_word(seen, v.w[w]);
      }
      const bool bad = any_odd(seen);
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

    // O^T += V^T P^T in steps of some reads of values, each step's made a step ahead
#if EK_Q == 0
    constexpr int STEPS = RUNS * 4;                   // a key of each lane
    words<VW> vf[2][NP / VE];
    const auto read_values = [&](int k) EK_HERE {
      const char* at = values + (run_key(k / 4) + k % 4) * ROW + r * VE * CS;
#pragma unroll
      for (int p = 0; p < NP; p += VE) vf[k & 1][p / VE] = lds_words<VW>(at + p * TILE * CS);
    };
    read_values(0);
#pragma unroll
    for (int s = 0; s < RUNS; ++s) weigh(s);
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (k + 1 < STEPS) read_values(k + 1);
      __builtin_amdgcn_sched_barrier(0);              // the reads before what they hide behind
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int t = 0; t < CT; ++t)
          o[t][p] = __builtin_amdgcn_mfma_f32_16x16x4f32(
              ek::bits_f32(vf[k & 1][p / VE].w[p % VE]), score(t, k / 4, k % 4), o[t][p], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
#else
    constexpr int SS = RUNS == 1 ? 1 : 2;             // runs of a product
    constexpr int GROUP = !TR ? VE : NP < 4 ? NP : 4; // output tiles of a step
    constexpr int PER = NP / GROUP, STEPS = RUNS / SS * PER;
    // The weights of a step's runs are made between the products of the step before: the VALU has
    // work while an instruction multiplies.
    u32 w_p[2][CT][TERMS][2 * SS];
    const auto weights = [&](int k) EK_HERE {
#pragma unroll
      for (int s = 0; s < SS; ++s) weigh(k * SS + s);
#pragma unroll
      for (int t = 0; t < CT; ++t)
#pragma unroll
        for (int i = 0; i < 2 * SS; ++i) {
          const int s = k * SS + i / 2, x = i % 2 * 2;
          u32 y[TERMS];
          split(score(t, s, x), score(t, s, x + 1), y);
#pragma unroll
          for (int n = 0; n < TERMS; ++n) w_p[k & 1][t][n][i] = y[n];
        }
    };
    const auto products = [&](int k, int p, const auto* w) EK_HERE {
#pragma unroll
      for (int x = 0; x < TERMS; ++x)
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          const auto* y = w_p[k / PER & 1][t][x];
          if constexpr (SS * sizeof(*w) == 4) mma_short<HALF>(o[t][p], w, y);
          else mma<HALF>(o[t][p], w, y);
        }
    };
#if EK_FP8
    words<VW> vf[2][4 * SS];
    const auto read_values = [&](int k) EK_HERE {
#pragma unroll
      for (int j = 0; j < 4 * SS; ++j) {
        const char* at = values + (run_key(k / PER * SS + j / 4) + (j & 3)) * ROW;
        vf[k & 1][j] = lds_words<VW>(at + k % PER * GROUP * TILE + r * VE);
      }
    };
#else
    // four lanes of 16 read a key each (its 4 elements from 4 * lane on): tr_read4
    u32 vf[2][GROUP][2 * SS];
    const int quad = lane >> 2 & 3, swap = v_swap(c * 4 + quad);
    const int half = (TILE == 32 ? lane >> 4 & 1 : 0) * 2 + (lane >> 1 & 1);     // chunk
    const char* at = values + quad * ROW + (lane & 1) * 8;
    const auto read_values = [&](int k) EK_HERE {
#pragma unroll
      for (int x = 0; x < GROUP; ++x)
#pragma unroll
        for (int i = 0; i < SS; ++i) {                 // v_swap goes by the key within 8
          const int p = k % PER * GROUP + x;
          uint16_t y[4];
          ek::tr_read4(y, (const uint16_t*)(at + run_key(k / PER * SS + i) * ROW +
                                            ((p * TILE / 8 + half) ^ swap) * 16));
          __builtin_memcpy(&vf[k & 1][x][2 * i], y, 8);
        }
    };
#endif
    read_values(0);
    weights(0);
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
      if (k + 1 < STEPS) read_values(k + 1);
      __builtin_amdgcn_sched_barrier(0);              // the reads before what they hide behind
      const int p0 = k % PER * GROUP;
#if EK_FP8
      // 4 SS keys' VE elements, 16 bits each
      u32 x[4 * SS][VE / 2];
#pragma unroll
      for (int j = 0; j < 4 * SS; ++j)
#pragma unroll
        for (int w = 0; w < VW; ++w)
          widen4<HALF>(vf[k & 1][j].w[w], &x[j][2 * w], &x[j][2 * w + 1]);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        u32 w[2 * SS];
#pragma unroll
        for (int i = 0; i < 2 * SS; ++i)
          w[i] = __builtin_amdgcn_perm(x[2 * i + 1][e / 2], x[2 * i][e / 2],
                                       e & 1 ? 0x07060302u : 0x05040100u);
        products(k, p0 + e, w);
      }
#else
#pragma unroll
      for (int x = 0; x < GROUP; ++x) products(k, p0 + x, vf[k & 1][x]);
#endif
      if ((k + 1) % PER == 0 && k + 1 < STEPS) {
        weights((k + 1) / PER);
        // of the step's products and what makes the next weights, in turn
#pragma unroll
        for (int x = 0; x < GROUP * TERMS * CT; ++x) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x402, (6), 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#endif
#undef score
    live = live_next;
    wait_for<LOADS>();
    __syncthreads();
  }

  // The same stages' keys once more, one at a time: the elements of their values that are not
  // finite.
  if (some_odd) {
#pragma unroll 1
    for (int key = lo; key < hi; ++key) {
      const int base = lo + (key - lo) / KT * KT, tile = (key - base) / TILE;
      const int page = table[page_of(a, key)], j = key - sq.past;
      if (!edge(base) || tile / NK != wk || (u32)page >= (u32)a.pages) continue;
      const char* v = vbase + page * a.c_page + (key - page_of(a, key) * a.page) * a.c_token;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        bool sees = key >= from[t] && j <= index[t];
        if (a.tree) {
          sees = j < 0 ? key >= from[t] : tree_bits(a, tree_of(t), bits[t], j) & 1;
          if (deep && j >= 0)
            sees = sees && tree_count(a, tree_of(t), j, sq.end - sq.past) <= a.window;
        }
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int i = 0; i < RA * 4; ++i) {
            const int d = element_of(p, i);
            const float x = element(v + (d < a.dim ? d : 0) * CS);
            // 0x207: a NaN or an infinity
            if (sees && __builtin_amdgcn_classf(x, 0x207)) o[t][p][i] = __builtin_nanf("");
          }
      }
    }
  }

#pragma unroll
  for (int t = 0; t < CT; ++t) {
    if constexpr (TILE == 16) l[t] = ek::reduce_xor<ek::Sum, 16>(l[t]);
    l[t] = ek::reduce_xor<ek::Sum, 32>(l[t]);
  }
  if constexpr (WK > 1) {
    // the waves of the same columns: to the first of them, in the order in which it holds its own
    float* part = (float*)s_stage;
    constexpr int SIZE = CT * (NP * RA * 256 + 128), ML = CT * NP * RA * 256;
    float* mine = part + ((wk - 1) * WC + wc) * SIZE + lane * 4;
    if (wk > 0) {
#pragma unroll
      for (int t = 0; t < CT; ++t) {
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int k = 0; k < RA; ++k)
            *(ek::f32x4*)(mine + ((t * NP + p) * RA + k) * 256) = ek::f32x4{
                o[t][p][k * 4], o[t][p][k * 4 + 1], o[t][p][k * 4 + 2], o[t][p][k * 4 + 3]};
        mine[ML + t * 128 - lane * 3] = m[t];
        mine[ML + t * 128 + 64 - lane * 3] = l[t];
      }
    }
    __syncthreads();
    if (wk > 0) return;
#pragma unroll
    for (int x = 0; x < WK - 1; ++x) {
      const float* other = part + (x * WC + wc) * SIZE;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        const float mo = other[ML + t * 128 + lane], lo = other[ML + t * 128 + 64 + lane];
        const float top = __builtin_fmaxf(m[t], mo), use = top == -__builtin_inff() ? 0.0f : top;
        const float f = ek::exp2_fast((m[t] - use) * scale), fo = ek::exp2_fast((mo - use) * scale);
        m[t] = top;
        l[t] = l[t] * f + lo * fo;
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int k = 0; k < RA; ++k) {
            const ek::f32x4 y = *(const ek::f32x4*)(other + ((t * NP + p) * RA + k) * 256 +
                                                    lane * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[t][p][k * 4 + i] = o[t][p][k * 4 + i] * f + y[i] * fo;
          }
      }
    }
  }

  // runs of VE or (transposed) 4 adjacent elements
  constexpr int OUT = TR ? 4 : VE;
  const auto each_run = [&](int t, const auto& put) EK_HERE {
    if constexpr (TR) {
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int k = 0; k < RA; ++k) {
          const float y[4] = {o[t][p][k * 4], o[t][p][k * 4 + 1], o[t][p][k * 4 + 2],
                              o[t][p][k * 4 + 3]};
          put(element_of(p, k * 4), y);
        }
    } else {
#pragma unroll
      for (int p = 0; p < NP; p += VE)
#pragma unroll
        for (int i = 0; i < RA * 4; ++i) {
          float y[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) y[e] = o[t][p + e][i];
          put(element_of(p, i), y);
        }
    }
  };
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    if (!valid(t)) continue;
    const int64_t token = sq.begin + index[t];
    const int h = head[t];
    if (it.chunks == 1) {
      const bool any = l[t] > 0.0f || l[t] != l[t];
      const float f = any ? a.v_scale / l[t] : 0.0f;
      T* dst = a.out + token * a.out_row + h * a.out_head;
      each_run(t, [&](int d, const float* x) EK_HERE {
        T y[OUT];
#pragma unroll
        for (int e = 0; e < OUT; ++e) y[e] = result(x[e], f, any);
        if (d < a.dim) ek::vstore_u<T, OUT>(dst + d, y);
      });
      if (a.lse && c == 0)
        a.lse[token * a.heads + h] =
            any ? (m[t] * scale + (__builtin_log2f(l[t]) - LIFT)) * LN2 : -__builtin_inff();
    } else {
      const int slot = it.slot + it.chunk * it.blocks + it.block;
      if (!a.part || slot < 0 || slot >= a.slots) continue;
      const int64_t at = ((int64_t)slot * a.kv_heads + g) * COLS + (wc * CT + t) * TILE + r;
      float* dst = a.part + at * a.dim;
      each_run(t, [&](int d, const float* y) EK_HERE {
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
#undef valid
#undef tree_of

// Joins the chunks of H heads of a token in a wave, CHUNKS of each at once: lane h CHUNKS + i has
// head h and chunk i, and all of their loads are on their way together. With `join` 1 or 4, H is
// as much: 4 where chunks are few, since a wave takes as long for one head as for four (64
// sequences of 27 tokens and less, 32 heads, 2 or 3 chunks: 20 us with 1, 12 with 4). Where
// chunks are many (`join` 0), a workgroup's four waves take one head's in turn and meet in the LDS.
template <int H> EK_INLINE void join_heads(const Params& a, int token, int head0, int first,
                                           int waves) {
  constexpr int DW = (DP + 127) / 128, CHUNKS = 16 / H;
  __shared__ float s_o[4][H == 1 ? DP : 1], s_m[4], s_l[4];
  const int lane = ek::lane_id(), i = lane % CHUNKS, mine = head0 + lane / CHUNKS % H;
  if (head0 >= a.heads || token < a.cu[0] || token >= a.cu[a.batch * a.cu_step]) return;
  const Row row = part_rows(a)[token];
  // rows that descend may have left this unwritten
  if (row.chunks <= 1 || row.slot < 0 || row.blocks <= 0 || row.index < 0 ||
      row.slot + (int64_t)row.chunks * row.blocks > a.slots)
    return;
  const int head = mine < a.heads ? mine : a.heads - 1, g = head / a.group;
  const u32 col = (u32)row.index * a.group + (head - g * a.group);
  const int block = col / COLS;
  if (__builtin_amdgcn_ballot_w64(block >= row.blocks) != 0) return;
  const float scale = scale_of(a);
  const int64_t at = ((int64_t)(row.slot + block) * a.kv_heads + g) * COLS + col - block * COLS;
  const int64_t step = (int64_t)row.blocks * a.kv_heads * COLS;    // from chunk to chunk
  float m = -__builtin_inff(), l = 0.0f, x[H][DW][2];
  int64_t from[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    from[h] = lane_value(at, h * CHUNKS);
#pragma unroll
    for (int k = 0; k < DW; ++k) x[h][k][0] = x[h][k][1] = 0.0f;
  }
#pragma unroll 1
  for (int i0 = first * CHUNKS; i0 < row.chunks; i0 += waves * CHUNKS) {
    const int count = row.chunks - i0 < CHUNKS ? row.chunks - i0 : CHUNKS;
    const float* ml = part_ml(a) + (at + (i0 + (i < count ? i : 0)) * step) * 2;
    float mi = ml[0], li = ml[1], v[H][CHUNKS][DW][2];
#pragma unroll
    for (int j0 = 0; j0 < CHUNKS; j0 += 4)
      if (j0 < count) {
#pragma unroll
        for (int j = j0; j < j0 + 4; ++j)
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const float* src = a.part + (from[h] + (i0 + (j < count ? j : 0)) * step) * a.dim;
#pragma unroll
            for (int k = 0; k < DW; ++k) {
              const int d = k * 128 + lane * 2;
              ek::vload_u<float, 2>(v[h][j][k], src + (d < a.dim ? d : 0));
            }
          }
      }
    __builtin_amdgcn_sched_barrier(0);               // all of them before the first wait
    mi = i < count ? mi : -__builtin_inff();
    li = i < count ? li : 0.0f;
    // over the lanes of a head's chunks
    float top = ek::reduce_xor<ek::Max, 1>(mi);
    top = ek::reduce_xor<ek::Max, 2>(top);
    if constexpr (CHUNKS == 16) {
      top = ek::reduce_xor<ek::Max, 4>(top);
      top = ek::reduce_xor<ek::Max, 8>(top);
    }
    top = __builtin_fmaxf(m, top);
    const float use = top == -__builtin_inff() ? 0.0f : top;
    const float f = ek::exp2_fast((m - use) * scale), w = ek::exp2_fast((mi - use) * scale);
    float sum = ek::reduce_xor<ek::Sum, 1>(li * w);
    sum = ek::reduce_xor<ek::Sum, 2>(sum);
    if constexpr (CHUNKS == 16) {
      sum = ek::reduce_xor<ek::Sum, 4>(sum);
      sum = ek::reduce_xor<ek::Sum, 8>(sum);
    }
    l = __builtin_fmaf(l, f, sum);
    m = top;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const float less = lane_value(f, h * CHUNKS);
#pragma unroll
      for (int k = 0; k < DW; ++k) x[h][k][0] *= less, x[h][k][1] *= less;
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
        if (j < count) {
          const float y = lane_value(w, h * CHUNKS + j);
#pragma unroll
          for (int k = 0; k < DW; ++k) {
            x[h][k][0] = __builtin_fmaf(v[h][j][k][0], y, x[h][k][0]);
            x[h][k][1] = __builtin_fmaf(v[h][j][k][1], y, x[h][k][1]);
          }
        }
    }
  }
  if constexpr (H == 1) {
    if (waves > 1) {
      // a part whose m is -inf has no weight, whatever wave it is
#pragma unroll
      for (int k = 0; k < DW; ++k) {
        const int d = k * 128 + lane * 2;
        if (d < DP) s_o[first][d] = x[0][k][0], s_o[first][d + 1] = x[0][k][1];
      }
      if (lane == 0) s_m[first] = m, s_l[first] = l;
      __syncthreads();
      if (first != 0) return;
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        const float mo = s_m[w], top = __builtin_fmaxf(m, mo);
        const float use = top == -__builtin_inff() ? 0.0f : top;
        const float f = ek::exp2_fast((m - use) * scale), fo = ek::exp2_fast((mo - use) * scale);
        l = l * f + s_l[w] * fo;
        m = top;
#pragma unroll
        for (int k = 0; k < DW; ++k) {
          const int d = k * 128 + lane * 2;
          if (d < DP) {
            x[0][k][0] = x[0][k][0] * f + s_o[w][d] * fo;
            x[0][k][1] = x[0][k][1] * f + s_o[w][d + 1] * fo;
          }
        }
      }
    }
  }
  const bool any = l > 0.0f || l != l;
  const float f = any ? a.v_scale / l : 0.0f;
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (head0 + h >= a.heads) break;
    T* dst = a.out + token * a.out_row + (head0 + h) * a.out_head;
    const float fh = lane_value(f, h * CHUNKS);
    const bool some = lane_value(any ? 1.0f : 0.0f, h * CHUNKS) != 0.0f;
#pragma unroll
    for (int k = 0; k < DW; ++k) {
      const int d = k * 128 + lane * 2;
      if (d < a.dim) {
        T y[2] = {result(x[h][k][0], fh, some), result(x[h][k][1], fh, some)};
        ek::vstore_u<T, 2>(dst + d, y);
      }
    }
  }
  if (a.lse && lane < H * CHUNKS && i == 0 && mine < a.heads)
    a.lse[(int64_t)token * a.heads + mine] =
        any ? (m * scale + (__builtin_log2f(l) - LIFT)) * LN2 : -__builtin_inff();
}

extern "C" __global__ __launch_bounds__(256) void ek_tree_attention_join(Params a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), token = blockIdx.x;
  const int at = blockIdx.y * 4 + wave;
  if (a.join == 4) join_heads<4>(a, token, at * 4, 0, 1);
  else if (a.join == 1) join_heads<1>(a, token, at, 0, 1);
  else join_heads<1>(a, token, blockIdx.y, wave, 4);
}
