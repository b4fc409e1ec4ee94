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
// key head of them share each key and value. A wave takes CT tiles of 16 columns through a chunk of
// the keys, reads them straight into the registers that feed the matrix instructions and uses them
// for all of its tiles, so that few columns take the cache's bytes over the HBM rate and many the
// matrix products' time. The W waves of a workgroup take neighbouring columns of the same chunk: what
// one reads the others find in the CU's cache.
//
// Layout (16x16 MFMA, lane l, r = l % 16, c = l / 16), as for one token per sequence:
// - S^T = K Q^T: lane l reads a chunk of key r; its accumulator holds keys 4 c + i of column r.
// - O^T = V^T P^T: the product over 32 keys gives lane l's slot j the key 4 c + j (j < 4) of the
//   first and of the second 16 keys, so that P is where S left it. Lane l reads VE consecutive
//   elements of those keys' values from element VE r on; the m-th product takes element VE r + m
//   of them (a register permute pairs the keys).
// - A weight is two terms of the values' 16-bit type, a product each: 2^-17 of it is left out in
//   bf16 and 2^-22 in fp16 and e4m3 (whose values are exact in fp16). One term would be half a
//   step of the output's own type off in every weight, as much again as its rounding.
//
// Work: the (chunk, block of W CT 16 columns) pairs of all sequences are items, a workgroup each, of
// one key head. The chunks' length comes from all sequences' lengths and rows, on the device.
// Sequences of one chunk are finished here; the others leave (O, m, l) per chunk and column to the
// second kernel.
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_FP8 (the cache is e4m3), EK_DP (64, 128 or 256: the
// head dimension it is compiled for), EK_PAD (the head dimension is smaller), EK_KT (keys per wave
// and step: 16 or 32), EK_CT (column tiles of a wave), EK_W (waves of a workgroup), EK_OCC (waves
// per SIMD that registers are left for).
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int DP = EK_DP, KT = EK_KT, CT = EK_CT, W = EK_W;
constexpr int COLS = W * CT * 16;                   // columns of a workgroup
constexpr int CS = EK_FP8 ? 1 : sizeof(T);          // bytes of a cache element
constexpr float LN2 = 0.69314718055994531f;
constexpr int ST = KT / 16;                         // score tiles
constexpr int KE = 16 / CS;                         // elements of a 16-byte key load
constexpr int KL = DP / (4 * KE);                   // key loads per score tile and lane
// Elements of a value load: 16 lanes cover at most the whole head.
constexpr int VE0 = EK_Q == 0 ? 4 : 8;
constexpr int VE = VE0 * 16 > DP ? DP / 16 : VE0;
constexpr int PANELS = DP / (16 * VE);
constexpr int VR = KT / 4;                          // value rows per lane
constexpr int VW = VE * CS / 4 < 1 ? 1 : VE * CS / 4;  // words of a value load
constexpr int UNIT = 16;                            // keys: what chunks are multiples of
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
// Element e of a load of values.
EK_INLINE float element(const u32* w, int e) {
#if EK_FP8
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 y = (e & 2) ? __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e / 4], true)
                       : __builtin_amdgcn_cvt_pk_f32_fp8((int)w[e / 4], false);
  return e & 1 ? y[1] : y[0];
#elif EK_Q == 0
  return ek::bits_f32(w[e]);
#else
  const uint16_t h = (uint16_t)(w[e / 2] >> (e & 1) * 16);
  if constexpr (EK_Q == 1) return (float)__builtin_bit_cast(_Float16, h);
  else return ek::bits_f32((u32)h << 16);
#endif
}

// The query columns as the products' operand: element chunk (s, c) of column r, in the order in
// which a lane reads its keys.
struct Query {
#if EK_Q == 0
  float w[KL][4];
#else
  u32 w[KL * KE / 8][4];
#endif
};

__device__ const u32 s_zeros[4] = {0, 0, 0, 0};

struct Tile {
  words<4> k[ST][KL];
  words<VW> v[VR][PANELS];
};

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
  const int lane = ek::lane_id(), r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = blockIdx.y;
  Seq sq;
  const Item it = find_item(a, blockIdx.x, sq);
  if (it.b < 0) return;
  const int all = sq.rows * a.group;                          // columns of the sequence
  const int col0 = it.block * COLS + wave * CT * 16;          // this wave's first
  if (col0 >= all) return;

  // this lane's column of each tile: its token and head
  int index[CT], head[CT];
  bool valid[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const int col = col0 + t * 16 + r;
    valid[t] = col < all;
    const int x = valid[t] ? col : all - 1;
    index[t] = (int)((u32)x / (u32)a.group);
    head[t] = g * a.group + x - index[t] * a.group;
  }
  if (a.part && it.chunk == 0 && g == 0 && c == 0) {
    // for the second kernel, by the column of each token's first head
#pragma unroll
    for (int t = 0; t < CT; ++t)
      if (valid[t] && head[t] == 0)
        part_rows(a)[sq.begin + index[t]] = {index[t], it.slot, it.chunks, it.blocks};
  }

  // units are spread evenly over the chunks: the first few have one more
  const int units = units_of(sq), each = units / it.chunks, more = units - each * it.chunks;
  const int lo_u = it.chunk * each + (it.chunk < more ? it.chunk : more);
  const int hi_u = lo_u + each + (it.chunk < more);
  int lo = sq.first + lo_u * UNIT;
  int hi = hi_u >= units ? sq.end : sq.first + hi_u * UNIT;
  // where each column's keys begin, and (a tree) whether its window ends among the new tokens
  int from[CT], from_most = 0;
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
      from_most = from[t] > from_most ? from[t] : from_most;
    }
  }
  if (a.window > 0) {
    from_most = __builtin_amdgcn_readfirstlane(wave_all<ek::Max>(from_most));
    deep = __builtin_amdgcn_ballot_w64(deep) != 0;
  }
  if (!a.tree) {
    // a chain's wave: no key behind its last token, none before the window of its first
    const int last = col0 + CT * 16 < all ? col0 + CT * 16 : all;
    const int stop = sq.past + (last - 1) / a.group + 1;
    hi = hi < stop ? hi : stop;
    if (a.window > 0) {
      const int begin = sq.past + col0 / a.group + 1 - a.window;
      if (begin > lo) lo += (begin - lo) / UNIT * UNIT;
    }
  }

  const char* kbase = a.k + g * a.c_head;
  const char* vbase = a.v + g * a.c_head;
  const int32_t* table = a.table + it.b * a.table_row;

  // Loads first, without branches between them, then zeros for columns and elements that are not
  // there: a wait per load would cost a latency each.
  Query q[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const T* src = a.q + (sq.begin + index[t]) * a.q_row + head[t] * a.q_head;
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
        const u32 w = valid[t] && place(i) < a.dim ? x[i].w[k] ^ a.q_sign : 0;
        __builtin_memcpy(&q[t].w[i][k], &w, 4);
      }
  }

  // what the scores are multiplied by for exp2: positive, since the queries took the sign
  const float to_cap = a.cap > 0.0f ? a.scale / a.cap : 0.0f;
  const float scale = scale_of(a);
  float m[CT], l[CT];
  ek::f32x4 o[CT][PANELS][VE];
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    m[t] = -__builtin_inff(), l[t] = 0.0f;
#pragma unroll
    for (int p = 0; p < PANELS; ++p)
#pragma unroll
      for (int e = 0; e < VE; ++e) o[t][p][e] = ek::f32x4{0, 0, 0, 0};
  }

  // The page of key base + lane of a step, read one step before its keys; -1: none.
  const auto page_id = [&](int base) -> int {
    const int key = base + (lane & (KT - 1));
    return key < hi ? table[page_of(a, key)] : -1;
  };
  // This lane's key's offset in the cache (0 where there is none), and which keys there are.
  const auto offset = [&](int base, int id, uint64_t& live) -> int64_t {
    const int key = base + (lane & (KT - 1));
    const bool ok = (u32)id < (u32)a.pages;
    live = __builtin_amdgcn_ballot_w64(ok);
    return ok ? id * a.c_page + (key - page_of(a, key) * a.page) * a.c_token : 0;
  };
  // lanes past the end of a head read zeros: loads without a branch
  const char* zeros = (const char*)s_zeros;
  const auto load_k = [&](Tile& t, int64_t off) {
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      const char* p = kbase + ek::shfl(off, s * 16 + r);
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int d = (i * 4 + c) * KE;
        t.k[s][i] = load_words<4>(!EK_PAD || d < a.dim ? p + d * CS : zeros);
      }
    }
  };
  const auto load_v = [&](Tile& t, int64_t off) {
#pragma unroll
    for (int j = 0; j < VR; ++j) {
      const char* p = vbase + ek::shfl(off, (j / 4) * 16 + c * 4 + (j & 3));
#pragma unroll
      for (int i = 0; i < PANELS; ++i) {
        const int d = i * 16 * VE + r * VE;
        t.v[j][i] = load_words<VW>(!EK_PAD || d < a.dim ? p + d * CS : zeros);
      }
    }
  };

  Tile tile;
  uint64_t live = 0;
  int64_t off = 0;
  int id = -1;
  if (lo < hi) {
    off = offset(lo, page_id(lo), live);
    load_k(tile, off);
    load_v(tile, off);
    id = page_id(lo + KT);
  }
  for (int base = lo; base < hi; base += KT) {
    const int next = base + KT;
    const int64_t here = off;
    uint64_t live_next = 0;
    // scores of KT keys: acc[t][s][i] is key 16 s + 4 c + i of tile t's column r
    ek::f32x4 acc[CT][ST];
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int s = 0; s < ST; ++s) acc[t][s] = ek::f32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < ST; ++s)
#pragma unroll
      for (int i = 0; i < KL; ++i) {
#if EK_Q == 0
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < CT; ++t)
            acc[t][s] = __builtin_amdgcn_mfma_f32_16x16x4f32(ek::bits_f32(tile.k[s][i].w[e]),
                                                             q[t].w[i][e], acc[t][s], 0, 0, 0);
#elif EK_FP8
        u32 x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) widen4<EK_Q == 1>(tile.k[s][i].w[e], &x[2 * e], &x[2 * e + 1]);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
          mma<EK_Q == 1>(acc[t][s], x, q[t].w[2 * i]);
          mma<EK_Q == 1>(acc[t][s], x + 4, q[t].w[2 * i + 1]);
        }
#else
#pragma unroll
        for (int t = 0; t < CT; ++t) mma<EK_Q == 1>(acc[t][s], tile.k[s][i].w, q[t].w[i]);
#endif
      }
    if (next < hi) {
      off = offset(next, id, live_next);
      id = page_id(next + KT);
      load_k(tile, off);
    }
    // softmax: scores and m stay as the product gave them (or capped, in log2 units) until exp2
    const bool full = live == ~0ull;
    // whether a column may not see a key of this step that is there
    const bool masks = next > sq.past || base < from_most;
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      if (a.cap > 0.0f) {
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][s][i] = a.cap * tanh_f(acc[t][s][i] * to_cap);
      }
      if (!full || masks) {
#pragma unroll
        for (int s = 0; s < ST; ++s) {
          const int key = base + s * 16 + c * 4, j = key - sq.past;
          u32 ok = (u32)(live >> (s * 16 + c * 4)) & 15u;
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
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = __builtin_fmaxf(mt, acc[t][s][i]);
      mt = ek::reduce_xor<ek::Max, 16>(mt);
      mt = ek::reduce_xor<ek::Max, 32>(mt);
      const float m_new = __builtin_fmaxf(m[t], mt);
      const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
      const float alpha = ek::exp2_fast((m[t] - m_use) * scale);
      m[t] = m_new;
      // most steps raise no column's maximum
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
        l[t] *= alpha;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int e = 0; e < VE; ++e) o[t][p][e] *= alpha;
      }
#pragma unroll
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[t][s][i] = ek::exp2_fast((acc[t][s][i] - m_use) * scale);
          l[t] += acc[t][s][i];
        }
    }
    // values without a key are taken as zeros: their memory may hold anything
    if (!full) {
#pragma unroll
      for (int j = 0; j < VR; ++j) {
        const bool ok = live >> ((j / 4) * 16 + c * 4 + (j & 3)) & 1;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int w = 0; w < VW; ++w) tile.v[j][p].w[w] = ok ? tile.v[j][p].w[w] : 0;
      }
    }
    // A value that is not finite must not reach the columns that don't see its key, whose weight
    // is 0: its key is left out of the products and added by itself below.
    uint64_t odd = 0;
    if (masks) {
#pragma unroll
      for (int j = 0; j < VR; ++j) {
        bool bad = false;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int w = 0; w < VW; ++w) bad |= odd_word(tile.v[j][p].w[w]);
        const uint64_t any = __builtin_amdgcn_ballot_w64(bad);
        if (any == 0) continue;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (any >> (x * 16) & 0xFFFF) odd |= 1ull << ((j / 4) * 16 + x * 4 + (j & 3));
        const bool out = any >> (c * 16) & 0xFFFF;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int w = 0; w < VW; ++w) tile.v[j][p].w[w] = out ? 0 : tile.v[j][p].w[w];
      }
    }
#if EK_Q == 0
#pragma unroll
    for (int j = 0; j < VR; ++j)
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int t = 0; t < CT; ++t)
            o[t][p][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                ek::bits_f32(tile.v[j][p].w[e]), acc[t][j / 4][j & 3], o[t][p][e], 0, 0, 0);
#else
    constexpr int SS = ST == 1 ? 1 : 2;            // score tiles of a product
    u32 w_p[CT][TERMS][ST / SS][2 * SS];
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          split(acc[t][s][2 * i] * LIFT, acc[t][s][2 * i + 1] * LIFT,
                w_p[t][0][s / SS][s % SS * 2 + i], w_p[t][1][s / SS][s % SS * 2 + i]);
#pragma unroll
    for (int s = 0; s < ST; s += SS) {
#pragma unroll
      for (int p = 0; p < PANELS; ++p) {
        // 4 SS keys' VE elements, 16 bits each
        u32 x[4 * SS][VE / 2];
#pragma unroll
        for (int j = 0; j < 4 * SS; ++j) {
          const words<VW>& v = tile.v[s * 4 + j][p];
#if EK_FP8
#pragma unroll
          for (int w = 0; w < VW; ++w) widen4<HALF>(v.w[w], &x[j][2 * w], &x[j][2 * w + 1]);
#else
#pragma unroll
          for (int w = 0; w < VW; ++w) x[j][w] = v.w[w];
#endif
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          u32 w[2 * SS];
#pragma unroll
          for (int i = 0; i < 2 * SS; ++i)
            w[i] = __builtin_amdgcn_perm(x[2 * i + 1][e / 2], x[2 * i][e / 2],
                                         e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int t = 0; t < CT; ++t) {
            if constexpr (SS == 2) {
#pragma unroll
              for (int k = 0; k < TERMS; ++k) mma<HALF>(o[t][p][e], w, w_p[t][k][s / SS]);
            } else {
              // 16 keys: a product over 32 for each term, which next to each other would lose
              // digits in the product's own sum
              const u32 twice[4] = {w[0], w[1], w[0], w[1]};
#pragma unroll
              for (int k = 0; k < TERMS; ++k) {
                const u32 one[4] = {w_p[t][k][s][0], w_p[t][k][s][1], 0, 0};
                mma<HALF>(o[t][p][e], twice, one);
              }
            }
          }
        }
      }
    }
#endif
    // keys with values that are not finite: each lane's elements of the head, for its columns
#pragma unroll 1
    while (odd != 0) {
      const int k = __builtin_ctzll(odd);
      odd &= odd - 1;
      const char* v = vbase + ek::shfl(here, k);
      float weight[CT];
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        float x = 0.0f;
#pragma unroll
        for (int s = 0; s < ST; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x = k >> 4 == s && (k & 3) == i ? acc[t][s][i] : x;
        weight[t] = ek::shfl(x, (k >> 2 & 3) * 16 + r) * LIFT;
      }
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = p * 16 * VE + (c * 4 + i) * VE;
          const words<VW> y = load_words<VW>(!EK_PAD || d < a.dim ? v + d * CS : zeros);
#pragma unroll
          for (int e = 0; e < VE; ++e)
#pragma unroll
            for (int t = 0; t < CT; ++t)
              if (weight[t] != 0.0f) o[t][p][e][i] += weight[t] * element(y.w, e);
        }
    }
    if (next < hi) load_v(tile, off);
    live = live_next;
  }

#pragma unroll
  for (int t = 0; t < CT; ++t) {
    l[t] = ek::reduce_xor<ek::Sum, 16>(l[t]);
    l[t] = ek::reduce_xor<ek::Sum, 32>(l[t]);
    if (!valid[t]) continue;
    const int64_t token = sq.begin + index[t];
    if (it.chunks == 1) {
      const bool any = l[t] > 0.0f || l[t] != l[t];
      const float f = any ? a.v_scale / LIFT / l[t] : 0.0f;
      T* dst = a.out + token * a.out_row + head[t] * a.out_head;
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = p * 16 * VE + (c * 4 + i) * VE;
          T y[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) y[e] = result(o[t][p][e][i], f, any);
          if (!EK_PAD || d < a.dim) ek::vstore_u<T, VE>(dst + d, y);
        }
      if (a.lse && c == 0)
        a.lse[token * a.heads + head[t]] =
            any ? (m[t] * scale + __builtin_log2f(l[t])) * LN2 : -__builtin_inff();
    } else {
      const int slot = it.slot + it.chunk * it.blocks + it.block;
      if (!a.part || slot < 0 || slot >= a.slots) continue;
      const int64_t at = ((int64_t)slot * a.kv_heads + g) * COLS + wave * CT * 16 + t * 16 + r;
      float* dst = a.part + at * a.dim;
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = p * 16 * VE + (c * 4 + i) * VE;
          float y[VE];
#pragma unroll
          for (int e = 0; e < VE; ++e) y[e] = o[t][p][e][i];
          if (!EK_PAD || d < a.dim) {
#pragma unroll
            for (int e = 0; e < VE; e += 4) ek::vstore_u<float, 4>(dst + d + e, y + e);
          }
        }
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
