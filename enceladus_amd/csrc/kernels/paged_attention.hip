// Attention of one new token per sequence over a paged key-value cache.
//
// For sequence b with n cached tokens, query head h and its key head g = h / (heads per key
// head): s_j = scale q_h . k_j over j in [max(0, n - window), n), optionally capped to
// c tanh(s_j / c); out = sum_j softmax(s)_j v_j, lse = log sum_j exp(s_j). No tokens: out = 0,
// lse = -inf.
//
// The cache is read once and each byte takes part in few operations (4 flops per element for
// each of the query heads that share it), so the time is the cache's bytes over the HBM rate, as
// long as enough loads are in flight on every CU. So nothing goes through the LDS on the way in:
// a wave reads KT keys and values straight into the registers that feed the matrix instructions
// and keeps them in flight behind the arithmetic of the tile before.
//
// Layout (16x16 MFMA, lane l, r = l % 16, c = l / 16; query heads are the columns of every
// product, up to 16 of one key head):
// - S^T = K Q^T: lane l reads a chunk of key r; its accumulator holds keys 4 c + i of head r.
// - O^T = V^T P^T: the product over 32 keys gives lane l's slot j the key 4 c + j (j < 4) of the
//   first and of the second 16 keys, so that P is where S left it. Lane l reads VE consecutive
//   elements of those keys' values from element VE r on; the m-th product takes element VE r + m
//   of them, so that the VE products cover 16 VE elements of the head without any transpose
//   through the LDS (a register permute pairs the keys).
// - The weights are split into terms of the values' 16-bit type, a product each (the matrix units
//   idle anyway), so that little is lost of their 32 bits: three bf16 terms hold a weight exactly,
//   two fp16 terms are off by 2^-22 of it at most. e4m3 values are exact in fp16, whose two terms
//   take bf16 queries' weights as well.
//
// Work: a chunk of one sequence is an item; one wave takes an item of one key head, by itself.
// The chunks' length comes from all sequences' lengths, on the device, so that ragged batches
// give items of about one size. Sequences of one chunk are finished here; the others leave
// (O, m, l) per chunk to the second kernel.
//
// Measured, both kernels: 64 ragged sequences, 8 key heads of 128, 32 query heads, bf16, 501 MB: 89
// us, 5.6 TB/s; one sequence of 131075, fp16, 537 MB: 94 us, 5.7 (a kernel that only reads: 6.0
// to 6.2). One sequence of 1999: 6.9 + 3.6 us, a chain of lengths, table, keys, then the join's.
// Joining in the first kernel, by the last wave of a sequence to arrive, took longer (18 instead
// of 12 us there: its counters are as far away as memory), and so did workgroups of 4 waves that
// merge in the LDS (they start and end together).
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_FP8 (the cache is e4m3), EK_DP (64, 128 or 256: the
// head dimension it is compiled for), EK_PAD (the head dimension is smaller than EK_DP), EK_KT
// (keys per wave and step: 16, 32 or 64).
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int DP = EK_DP;
constexpr int CS = EK_FP8 ? 1 : sizeof(T);          // bytes of a cache element
constexpr float LN2 = 0.69314718055994531f;
constexpr int KT = EK_KT;                           // keys per wave and step
constexpr int ST = KT / 16;                         // score tiles
constexpr int KE = 16 / CS;                         // elements of a 16-byte key load
constexpr int KL = DP / (4 * KE);                   // key loads per score tile and lane
// Elements of a value load: 16 lanes cover at most the whole head.
constexpr int VE0 = EK_Q == 0 ? 4 : 8;
constexpr int VE = VE0 * 16 > DP ? DP / 16 : VE0;
constexpr int PANELS = DP / (16 * VE);
constexpr int VR = KT / 4;                          // value rows per lane
constexpr int VW = VE * CS / 4 < 1 ? 1 : VE * CS / 4;  // words of a value load
constexpr bool PACKS = EK_FP8 && ST > 1;            // see the softmax of few heads
constexpr int UNIT = 16;                            // keys: what chunks are multiples of
// Weights are exp2(s - m), with the difference taken of the scores as the product gave them (or
// capped) and scaled after that: the largest is 1 exactly, however large the scores are. Fp16 has
// no more than 24 binary places below 1: terms lifted by 2^14 keep a weight down to 2^-39 of the
// largest one (131072 keys of a weight of 2^-26 each are 0.2% of the sum). bf16 and fp32 have the
// exponents for it.
constexpr bool HALF = EK_Q == 1 || EK_FP8;          // the weights' terms are fp16
constexpr int TERMS = HALF ? 2 : 3;
constexpr float LIFT = HALF ? 0x1p14f : 1.0f;

typedef uint32_t u32;
template <int W> struct words { u32 w[W]; };
template <int W, bool NT = false> EK_INLINE words<W> load_words(const char* p) {
  words<W> r;
  if constexpr (NT) ek::vload_nt_u<uint8_t, W * 4>((uint8_t*)r.w, (const uint8_t*)p);
  else ek::vload_u<uint8_t, W * 4>((uint8_t*)r.w, (const uint8_t*)p);
  return r;
}

template <bool B> struct flag { static constexpr bool value = B; };

struct Params {
  const T* q;
  const char* k;
  const char* v;
  const int32_t* table;
  const int32_t* lens;
  T* out;
  float* lse;
  float* part;   // [item][head][dim]: O (lifted); then [item][head][2]: m (not scaled), l; then
                 // [sequence][2] words: its first item and how many; or null: no sequence has
                 // two chunks
  int64_t q_row, q_head, out_row, out_head;   // elements
  int64_t c_page, c_token, c_head;   // bytes
  int64_t table_row, lens_step;      // elements
  int32_t batch, heads, group, dim, page, pages, capacity, window;
  uint32_t page_mul;
  int32_t page_shift, items, min_units, stream;
  uint32_t q_sign;                   // the sign bits of the queries' words, if scale is negative
  float scale, cap, v_scale;         // scale > 0, with log2(e); cap in the same unit, or 0
};

EK_INLINE int page_of(const Params& a, int key) {
  return a.page == 1 ? key : (int)(__umulhi((u32)key, a.page_mul) >> a.page_shift);
}

// Keys that sequence b attends to: [first, first + count).
EK_INLINE int length_of(const Params& a, int b) {
  return a.lens[(b < a.batch ? b : a.batch - 1) * a.lens_step];
}
EK_INLINE void span_of(const Params& a, int b, int n, int& first, int& count) {
  n = n < 0 || b >= a.batch ? 0 : n > a.capacity ? a.capacity : n;
  first = a.window > 0 && n > a.window ? n - a.window : 0;
  count = n - first;
}
EK_INLINE void span_of(const Params& a, int b, int& first, int& count) {
  span_of(a, b, length_of(a, b), first, count);
}

EK_INLINE int units_of(int count) { return (count + UNIT - 1) / UNIT; }

EK_INLINE int chunks_of(int units, int per) { return (u32)(units + per - 1) / (u32)per; }

template <typename OP, typename V> EK_INLINE V wave_all(V x) {
  x = ek::reduce_xor<OP, 1>(x);
  x = ek::reduce_xor<OP, 2>(x);
  x = ek::reduce_xor<OP, 4>(x);
  x = ek::reduce_xor<OP, 8>(x);
  x = ek::reduce_xor<OP, 16>(x);
  return ek::reduce_xor<OP, 32>(x);
}

// What an item is: chunk `index` of the `chunks` of sequence b, or, with chunks 0, an empty
// sequence b; b is -1 for items without work. `start` is the sequence's first item.
struct Item {
  int b, first, count, index, chunks, start;
};

// The chunks of all sequences in their order are items 0, 1, ...: at most `items` of them and
// one more for each sequence with tokens, so that the grid's further `batch` items are enough
// to give every empty sequence one as well. A chunk has as many units of UNIT keys as give
// `items` chunks in all. Every wave finds its own from the lengths: 64 sequences at a time, a
// lane each, of which the first HELD times 64 stay in registers between the sum and the search.
EK_INLINE Item find_item(const Params& a, int item) {
  constexpr int HELD = 4;
  const int lane = ek::lane_id();
  int f[HELD], n[HELD], total = 0;
#pragma unroll
  for (int i = 0; i < HELD; ++i) n[i] = length_of(a, i * 64 + lane);   // one wait for all
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    span_of(a, i * 64 + lane, n[i], f[i], n[i]);
    total += units_of(n[i]);
  }
  for (int base = HELD * 64; base < a.batch; base += 64) {
    int first, count;
    span_of(a, base + lane, first, count);
    total += units_of(count);
  }
  total = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(total));
  int per = chunks_of(total, a.items);
  per = per < a.min_units ? a.min_units : per;
  // Each sequence may have a chunk more than its share. If chunks of up to half as many units
  // again fit all of them into `items`, that saves a last round of few waves.
  if (a.batch <= HELD * 64) {
    int try_per = per;
#pragma unroll 1
    for (int k = 0; k < 4; ++k) {
      int all = 0;
#pragma unroll
      for (int i = 0; i < HELD; ++i)
        if (i * 64 < a.batch) all += chunks_of(units_of(n[i]), try_per);
      all = __builtin_amdgcn_readfirstlane(wave_all<ek::Sum>(all));
      if (all <= a.items) per = try_per;
      if (all <= a.items || all > a.items + a.items / 2) break;
      try_per += (try_per + 7) >> 3;
    }
  }

  int before = 0;
  const auto search = [&](int base, int first, int count, Item& it) {
    const int mine = chunks_of(units_of(count), per);
    const int end = before + ek::wave_prefix_sum(mine);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item < end);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      it.b = base + at;
      it.first = __builtin_amdgcn_readlane(first, at);
      it.count = __builtin_amdgcn_readlane(count, at);
      it.chunks = __builtin_amdgcn_readlane(mine, at);
      it.start = __builtin_amdgcn_readlane(end, at) - it.chunks;
      it.index = item - it.start;
      return true;
    }
    before = __builtin_amdgcn_readlane(end, 63);
    return false;
  };
  Item it = {-1, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < HELD; ++i)
    if (i * 64 < a.batch && search(i * 64, f[i], n[i], it)) return it;
  for (int base = HELD * 64; base < a.batch; base += 64) {
    int first, count;
    span_of(a, base + lane, first, count);
    if (search(base, first, count, it)) return it;
  }
  // past the last chunk: the empty sequence of that rank
  int rank = item - before;
  for (int base = 0; base < a.batch; base += 64) {
    int first, count;
    span_of(a, base + lane, first, count);
    uint64_t none = __builtin_amdgcn_ballot_w64(base + lane < a.batch && count == 0);
    const int here = __builtin_popcountll(none);
    if (rank < here) {
      for (; rank > 0; --rank) none &= none - 1;
      it.b = base + __builtin_ctzll(none);
      return it;
    }
    rank -= here;
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
// The next term of two weights: x0 and x1 become what it leaves. bf16 cuts off, so that three terms
// are the 24 bits of a weight exactly, and that no conversion is waited for.
EK_INLINE u32 next_term(float& x0, float& x1) {
  if constexpr (HALF) {
    const _Float16 h0 = (_Float16)x0, h1 = (_Float16)x1;
    x0 -= (float)h0;
    x1 -= (float)h1;
    return pack2(h0, h1);
  } else {
    const u32 u0 = ek::f32_bits(x0), u1 = ek::f32_bits(x1);
    x0 -= ek::bits_f32(u0 & 0xFFFF0000u);
    x1 -= ek::bits_f32(u1 & 0xFFFF0000u);
    return __builtin_amdgcn_perm(u1, u0, 0x07060302u);
  }
}
#endif

// Lanes 8 to 15 of each row of 16 against lanes 0 to 7: the value 8 lanes away; x with lanes 8
// to 15 replaced by y of lanes 0 to 7; x of lanes 8 to 15 in lanes 0 to 7 (0 in the others).
EK_INLINE float half_row(float x) {
  return ek::bits_f32((u32)__builtin_amdgcn_update_dpp(0, (int)ek::f32_bits(x), 0x128, 0xF, 0xF,
                                                       true));
}
EK_INLINE float upper_half(float x, float y) {
  return ek::bits_f32((u32)__builtin_amdgcn_update_dpp(
      (int)ek::f32_bits(x), (int)ek::f32_bits(y), 0x118, 0xF, 0xC, false));
}
EK_INLINE u32 to_lower_half(u32 x) {
  return (u32)__builtin_amdgcn_update_dpp(0, (int)x, 0x108, 0xF, 0xF, true);
}

// The query heads as the products' operand: element chunk (s, c) of head r, in the order in
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

// A sequence's chunks are joined in groups of up to 16, or in 16 groups: its group size.
EK_INLINE int group_of(int chunks) {
  return chunks <= 256 ? (chunks < 16 ? chunks : 16) : (chunks + 15) / 16;
}

// A head's value: o f, rounded once to T.
EK_INLINE T result(float o, float f, bool any) { return ek::cvt<T>(any ? o * f : 0.0f); }

// What differences of the running maxima are multiplied by for exp2: capped scores are in log2 units.
EK_INLINE float scale_of(const Params& a) { return a.cap > 0.0f ? 1.0f : a.scale; }

EK_INLINE float* part_ml(const Params& a) {
  return a.part + (int64_t)(a.items + a.batch) * a.heads * a.dim;
}

// The weights of up to 16 parts (m, l) of a head, one in each lane of a group of 16 (m -inf
// where there is none): m and l become the whole's, in all 16 lanes.
EK_INLINE float weigh16(float& m, float& l, float scale) {
  const float mine = m;
  m = ek::reduce_xor<ek::Max, 1>(m);
  m = ek::reduce_xor<ek::Max, 2>(m);
  m = ek::reduce_xor<ek::Max, 4>(m);
  m = ek::reduce_xor<ek::Max, 8>(m);
  const float w = ek::exp2_fast((mine - (m == -__builtin_inff() ? 0.0f : m)) * scale);
  l *= w;
  l = ek::reduce_xor<ek::Sum, 1>(l);
  l = ek::reduce_xor<ek::Sum, 2>(l);
  l = ek::reduce_xor<ek::Sum, 4>(l);
  l = ek::reduce_xor<ek::Sum, 8>(l);
  return w;
}

EK_INLINE float lane_value(float x, int lane) {
  return ek::bits_f32((u32)__builtin_amdgcn_readlane((int)ek::f32_bits(x), lane));
}

extern "C" __global__ __launch_bounds__(64, EK_Q == 0 && DP == 256 ? 1 : 2) void
ek_paged_attention(Params a) {
  const int lane = ek::lane_id(), r = lane & 15, c = lane >> 4;
  const int tiles16 = (a.group + 15) / 16;
  const int g = blockIdx.y / tiles16, h0 = (blockIdx.y - g * tiles16) * 16;
  const int nh = a.group - h0 < 16 ? a.group - h0 : 16;

  const Item it = find_item(a, blockIdx.x);
  const int b = it.b, chunks = it.chunks;
  if (b < 0) return;
  if (a.part && it.index == 0 && blockIdx.y == 0 && lane == 0) {
    // for the second kernel: which items the sequence's chunks are
    int32_t* info = (int32_t*)(a.part + (int64_t)(a.items + a.batch) * a.heads * (a.dim + 2));
    info[2 * b] = it.start;
    info[2 * b + 1] = chunks;
  }
  if (chunks == 0) {
    for (int x = lane; x < nh * a.dim; x += 64) {
      const int h = x / a.dim, d = x - h * a.dim, head = g * a.group + h0 + h;
      a.out[b * a.out_row + head * a.out_head + d] = ek::cvt<T>(0.0f);
      if (a.lse && d == 0) a.lse[(int64_t)b * a.heads + head] = -__builtin_inff();
    }
    return;
  }
  // units are spread evenly over the chunks: the first few have one more
  const int units = units_of(it.count), each = units / chunks, more = units - each * chunks;
  const int lo_u = it.index * each + (it.index < more ? it.index : more);
  const int hi_u = lo_u + each + (it.index < more);
  const int lo = it.first + lo_u * UNIT;
  const int hi = hi_u == units ? it.first + it.count : it.first + hi_u * UNIT;

  const char* kbase = a.k + g * a.c_head;
  const char* vbase = a.v + g * a.c_head;
  const int32_t* row = a.table + b * a.table_row;

  // Loads first, without branches between them, then zeros for heads and elements that are not
  // there: a wait per load would cost a latency each.
  Query q;
  {
    const T* src = a.q + b * a.q_row +
                   (int64_t)(g * a.group + h0 + (r < nh ? r : 0)) * a.q_head;
    constexpr int QN = sizeof(q.w) / 16, QE = 16 / sizeof(T);
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
        const u32 w = r < nh && place(i) < a.dim ? x[i].w[k] ^ a.q_sign : 0;
        __builtin_memcpy(&q.w[i][k], &w, 4);
      }
  }

  // what the scores are multiplied by for exp2: positive, since the queries took the sign
  const float to_cap = a.cap > 0.0f ? a.scale / a.cap : 0.0f;
  const float scale = scale_of(a);
  float m = -__builtin_inff(), l = 0.0f;
  ek::f32x4 o[PANELS][VE];
#pragma unroll
  for (int p = 0; p < PANELS; ++p)
#pragma unroll
    for (int e = 0; e < VE; ++e) o[p][e] = ek::f32x4{0, 0, 0, 0};

  // The page of key base + lane of a step, read one step before its keys; -1: none.
  const auto page_id = [&](int base) -> int {
    const int key = base + (lane & (KT - 1));
    return key < hi ? row[page_of(a, key)] : -1;
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
    const auto go = [&](auto nt) {
#pragma unroll
      for (int s = 0; s < ST; ++s) {
        const char* p = kbase + ek::shfl(off, s * 16 + r);
#pragma unroll
        for (int i = 0; i < KL; ++i) {
          const int d = (i * 4 + c) * KE;
          t.k[s][i] = load_words<4, nt.value>(!EK_PAD || d < a.dim ? p + d * CS : zeros);
        }
      }
    };
    if (a.stream) go(flag<true>());
    else go(flag<false>());
  };
  const auto load_v = [&](Tile& t, int64_t off) {
    const auto go = [&](auto nt) {
#pragma unroll
      for (int j = 0; j < VR; ++j) {
        const char* p = vbase + ek::shfl(off, (j / 4) * 16 + c * 4 + (j & 3));
#pragma unroll
        for (int i = 0; i < PANELS; ++i) {
          const int d = i * 16 * VE + r * VE;
          t.v[j][i] = load_words<VW, nt.value>(!EK_PAD || d < a.dim ? p + d * CS : zeros);
        }
      }
    };
    if (a.stream) go(flag<true>());
    else go(flag<false>());
  };

  Tile t;
  uint64_t live = 0;
  int64_t off = offset(lo, page_id(lo), live);
  load_k(t, off);
  load_v(t, off);
  int id = page_id(lo + KT);
  for (int base = lo; base < hi; base += KT) {
    const int next = base + KT;
    uint64_t live_next = 0;
    // scores of KT keys: acc[s][i] is key 16 s + 4 c + i of head r
    ek::f32x4 acc[ST];
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      acc[s] = ek::f32x4{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
#if EK_Q == 0
#pragma unroll
        for (int e = 0; e < 4; ++e)
          acc[s] = __builtin_amdgcn_mfma_f32_16x16x4f32(ek::bits_f32(t.k[s][i].w[e]),
                                                        q.w[i][e], acc[s], 0, 0, 0);
#elif EK_FP8
        u32 x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) widen4<EK_Q == 1>(t.k[s][i].w[e], &x[2 * e], &x[2 * e + 1]);
        mma<EK_Q == 1>(acc[s], x, q.w[2 * i]);
        mma<EK_Q == 1>(acc[s], x + 4, q.w[2 * i + 1]);
#else
        mma<EK_Q == 1>(acc[s], t.k[s][i].w, q.w[i]);
#endif
      }
    }
    if (next < hi) {
      off = offset(next, id, live_next);
      id = page_id(next + KT);
      load_k(t, off);
    }
    // softmax: scores and m stay as the product gave them (or capped, in log2 units) until exp2
    const bool full = live == ~0ull;
    const auto soften = [&](auto& x, const auto& key_of) {
      constexpr int N = sizeof(x) / sizeof(x[0]);
      if (a.cap > 0.0f) {
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][i] = a.cap * tanh_f(x[s][i] * to_cap);
      }
      if (!full) {
#pragma unroll
        for (int s = 0; s < N; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[s][i] = live >> (key_of(s) + i) & 1 ? x[s][i] : -__builtin_inff();
      }
      float mt = -__builtin_inff();
#pragma unroll
      for (int s = 0; s < N; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) mt = __builtin_fmaxf(mt, x[s][i]);
      if constexpr (N < ST) mt = __builtin_fmaxf(mt, half_row(mt));
      mt = ek::reduce_xor<ek::Max, 16>(mt);
      mt = ek::reduce_xor<ek::Max, 32>(mt);
      const float m_new = __builtin_fmaxf(m, mt);
      const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
      const float alpha = ek::exp2_fast((m - m_use) * scale);
      m = m_new;
      // most steps raise no head's maximum
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
        l *= alpha;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int e = 0; e < VE; ++e) o[p][e] *= alpha;
      }
#pragma unroll
      for (int s = 0; s < N; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[s][i] = ek::exp2_fast((x[s][i] - m_use) * scale);
          l += x[s][i];
        }
    };
    const auto own = [&](int s) { return s * 16 + c * 4; };   // a lane's first key of a tile
    // values without a key are taken as zeros: their memory may hold anything
    const auto clear_absent = [&] {
      if (full) return;
#pragma unroll
      for (int j = 0; j < VR; ++j) {
        const bool ok = live >> ((j / 4) * 16 + c * 4 + (j & 3)) & 1;
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int w = 0; w < VW; ++w) t.v[j][p].w[w] = ok ? t.v[j][p].w[w] : 0;
      }
    };
#if EK_Q == 0
    soften(acc, own);
    clear_absent();
#pragma unroll
    for (int j = 0; j < VR; ++j)
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int e = 0; e < VE; ++e)
          o[p][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(ek::bits_f32(t.v[j][p].w[e]),
                                                         acc[j / 4][j & 3], o[p][e], 0, 0, 0);
#else
    constexpr int SS = ST == 1 ? 1 : 2;            // score tiles of a product
    u32 w_p[TERMS][ST / SS][2 * SS];
    // the weights' terms from word `at` on: each is what the ones before it leave
    const auto split = [&](const ek::f32x4& x, int at) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x0 = x[2 * i] * LIFT, x1 = x[2 * i + 1] * LIFT;
#pragma unroll
        for (int k = 0; k < TERMS; ++k)
          w_p[k][at / (2 * SS)][at % (2 * SS) + i] = next_term(x0, x1);
      }
    };
    if constexpr (PACKS) {
      // A key head of at most 8 query heads leaves lanes 8 to 15 of a row without one: they take
      // the scores of every second tile, and give the weights back (24 sequences, 153 MB of
      // e4m3, 64 heads over 8 key heads: with a softcap 40.4 us instead of 42.1).
      if (nh <= 8) {
        ek::f32x4 x[PACKS ? ST / 2 : 1];
#pragma unroll
        for (int s = 0; s < ST / 2; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][i] = upper_half(acc[2 * s][i], acc[2 * s + 1][i]);
        soften(x, [&](int s) { return s * 32 + (r >> 3) * 16 + c * 4; });
#pragma unroll
        for (int s = 0; s < ST / 2; ++s) {
          split(x[s], s * 4);
#pragma unroll
          for (int k = 0; k < TERMS; ++k)
#pragma unroll
            for (int i = 0; i < 2; ++i) w_p[k][s][2 + i] = to_lower_half(w_p[k][s][i]);
        }
      }
    }
    if (!PACKS || nh > 8) {
      soften(acc, own);
#pragma unroll
      for (int s = 0; s < ST; ++s) split(acc[s], s * 2);
    }
    clear_absent();
#pragma unroll
    for (int s = 0; s < ST; s += SS) {
#pragma unroll
      for (int p = 0; p < PANELS; ++p) {
        // 4 SS keys' VE elements, 16 bits each
        u32 x[4 * SS][VE / 2];
#pragma unroll
        for (int j = 0; j < 4 * SS; ++j) {
          const words<VW>& v = t.v[s * 4 + j][p];
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
          if constexpr (SS == 2) {
#pragma unroll
            for (int k = 0; k < TERMS; ++k) mma<HALF>(o[p][e], w, w_p[k][s / SS]);
          } else {
            // 16 keys: a product over 32 for the first term and one for the others, which next to
            // the first would lose digits in the product's own sum (64 ragged sequences, bf16: off
            // from 32-bit sums by 4.0e-5 of the result's norm with the first two together, 2.6e-5 so)
            const u32 twice[4] = {w[0], w[1], w[0], w[1]};
            const u32 first[4] = {w_p[0][s][0], w_p[0][s][1], 0, 0};
            const u32 rest[4] = {w_p[1][s][0], w_p[1][s][1],
                                 TERMS > 2 ? w_p[TERMS - 1][s][0] : 0,
                                 TERMS > 2 ? w_p[TERMS - 1][s][1] : 0};
            mma<HALF>(o[p][e], twice, first);
            mma<HALF>(o[p][e], twice, rest);
          }
        }
      }
    }
#endif
    if (next < hi) load_v(t, off);
    live = live_next;
  }

  if (PACKS && nh <= 8) l += half_row(l);
  l = ek::reduce_xor<ek::Sum, 16>(l);
  l = ek::reduce_xor<ek::Sum, 32>(l);
  if (r >= nh) return;
  const int head = g * a.group + h0 + r;
  if (chunks == 1) {
    const bool any = l > 0.0f || l != l;
    const float f = any ? a.v_scale / LIFT / l : 0.0f;
    T* dst = a.out + b * a.out_row + head * a.out_head;
#pragma unroll
    for (int p = 0; p < PANELS; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = p * 16 * VE + (c * 4 + i) * VE;
        T y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = result(o[p][e][i], f, any);
        if (!EK_PAD || d < a.dim) ek::vstore_u<T, VE>(dst + d, y);
      }
    if (a.lse && c == 0)
      a.lse[(int64_t)b * a.heads + head] =
          any ? (m * scale + __builtin_log2f(l)) * LN2 : -__builtin_inff();
  } else {
    const int64_t at = (int64_t)blockIdx.x * a.heads + head;
    float* dst = a.part + at * a.dim;
#pragma unroll
    for (int p = 0; p < PANELS; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = p * 16 * VE + (c * 4 + i) * VE;
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) y[e] = o[p][e][i];
        if (!EK_PAD || d < a.dim) {
#pragma unroll
          for (int e = 0; e < VE; e += 4) ek::vstore_u<float, 4>(dst + d + e, y + e);
        }
      }
    if (c == 0) {
      float* ml = part_ml(a) + at * 2;
      ml[0] = m;
      ml[1] = l;
    }
  }
}

// Joins the chunks of a sequence that has several, for one head: a wave per group of up to 16,
// whose loads are all on their way at once, then the groups. Two latencies of a launch that reads
// what other XCDs wrote: 3.4 us for 32 heads of one sequence of 32 chunks, 6 us for 256 chunks, 5.4
// for 24 sequences of 64 heads (8.6 MB of parts).
extern "C" __global__ __launch_bounds__(1024) void ek_paged_attention_join(Params a) {
  constexpr int DW = (DP + 127) / 128;
  __shared__ float s_o[16][DP];
  __shared__ float s_m[16], s_l[16];
  const int lane = ek::lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6, b = blockIdx.x, head = blockIdx.y;
  const float* ml = part_ml(a);
  const int32_t* info = (const int32_t*)(ml + (int64_t)(a.items + a.batch) * a.heads * 2);
  const int start = info[2 * b], chunks = info[2 * b + 1];
  if (chunks <= 1) return;
  const float scale = scale_of(a);
  const int gs = group_of(chunks), groups = (chunks + gs - 1) / gs;
  float x[DW][2];
  for (int group = wave; group < groups; group += waves) {
    const int begin = start + group * gs;
    const int size = chunks - group * gs < gs ? chunks - group * gs : gs;
    float mm = -__builtin_inff(), ll = 0.0f;
#pragma unroll
    for (int k = 0; k < DW; ++k) x[k][0] = x[k][1] = 0.0f;
#pragma unroll 1
    for (int i0 = 0; i0 < size; i0 += 16) {
      const int count = size - i0 < 16 ? size - i0 : 16, i = lane & 15;
      // Loads without branches: lanes and chunks that are not there read the last one, which
      // then has no weight.
      const int64_t at = (int64_t)(begin + i0) * a.heads + head;
      const float* mls = ml + (at + (int64_t)(i < count ? i : count - 1) * a.heads) * 2;
      float m = mls[0], l = mls[1];
      float v[16][DW][2];
      const char* base = (const char*)(a.part + at * a.dim);
      const u32 step = (u32)a.heads * a.dim * 4;   // of 15 at most: below 2^32
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const u32 row = (u32)(j < count ? j : count - 1) * step;
#pragma unroll
        for (int k = 0; k < DW; ++k) {
          const int d = k * 128 + lane * 2;
          ek::vload_u<float, 2>(v[j][k], (const float*)(base + (row + (d < a.dim ? d : 0) * 4u)));
        }
      }
      __builtin_amdgcn_sched_barrier(0);           // all of them before the first wait
      m = i < count ? m : -__builtin_inff();
      l = i < count ? l : 0.0f;
      float w = weigh16(m, l, scale);
      // onto what came before (with more than 16 chunks)
      const float m_new = __builtin_fmaxf(mm, m);
      const float mu = m_new == -__builtin_inff() ? 0.0f : m_new;
      const float f = ek::exp2_fast((mm - mu) * scale), part = ek::exp2_fast((m - mu) * scale);
      w *= part;
      ll = __builtin_fmaf(ll, f, l * part);
      mm = m_new;
#pragma unroll
      for (int k = 0; k < DW; ++k) x[k][0] *= f, x[k][1] *= f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float y = lane_value(w, j);
#pragma unroll
        for (int k = 0; k < DW; ++k) {
          x[k][0] = j < count ? __builtin_fmaf(v[j][k][0], y, x[k][0]) : x[k][0];
          x[k][1] = j < count ? __builtin_fmaf(v[j][k][1], y, x[k][1]) : x[k][1];
        }
      }
    }
    if (lane == 0) {
      s_m[group] = lane_value(mm, 0);
      s_l[group] = lane_value(ll, 0);
    }
#pragma unroll
    for (int k = 0; k < DW; ++k) {
      const int d = k * 128 + lane * 2;
      if (d < DP) {
        s_o[group][d] = x[k][0];
        s_o[group][d + 1] = x[k][1];
      }
    }
  }
  __syncthreads();
  if (wave != 0) return;
  float m = (lane & 15) < groups ? s_m[lane & 15] : -__builtin_inff();
  float l = (lane & 15) < groups ? s_l[lane & 15] : 0.0f;
  if (groups > 1) {
    const float w = weigh16(m, l, scale);
#pragma unroll
    for (int k = 0; k < DW; ++k) x[k][0] = x[k][1] = 0.0f;
    for (int j = 0; j < groups; ++j) {
      const float f = lane_value(w, j);
#pragma unroll
      for (int k = 0; k < DW; ++k) {
        const int d = k * 128 + lane * 2;
        if (d < DP) {
          x[k][0] = __builtin_fmaf(s_o[j][d], f, x[k][0]);
          x[k][1] = __builtin_fmaf(s_o[j][d + 1], f, x[k][1]);
        }
      }
    }
  }
  m = lane_value(m, 0);
  l = lane_value(l, 0);
  const bool any = l > 0.0f || l != l;
  const float f = any ? a.v_scale / LIFT / l : 0.0f;
  T* dst = a.out + b * a.out_row + head * a.out_head;
#pragma unroll
  for (int k = 0; k < DW; ++k) {
    const int d = k * 128 + lane * 2;
    if (d < a.dim) {
      T y[2] = {result(x[k][0], f, any), result(x[k][1], f, any)};
      ek::vstore_u<T, 2>(dst + d, y);
    }
  }
  if (a.lse && lane == 0)
    a.lse[(int64_t)b * a.heads + head] =
        any ? (m * scale + __builtin_log2f(l)) * LN2 : -__builtin_inff();
}
