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
// - The weights are split into two terms of the 16-bit type (p = hi + lo), two products each:
//   the matrix units idle anyway, and the output keeps the accuracy of 32-bit weights.
//
// Work: a chunk of one sequence is an item; a workgroup (4 waves, tiles in turn) takes one item
// of one key head. The chunk's length comes from all sequences' lengths, on the device, so that
// ragged batches give items of about one size. Sequences of one chunk are finished here;
// the others leave (m, l, O) per chunk to the second kernel.
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_FP8 (the cache is e4m3), EK_DP (64, 128 or 256: the
// head dimension it is compiled for), EK_PAD (the head dimension is smaller than EK_DP).
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
constexpr int WAVES = 4;
constexpr float LN2 = 0.69314718055994531f;
// Keys per wave and step: 16 KB of keys and values, where the products' shapes allow it.
constexpr int KT0 = 8192 / (DP * CS);
constexpr int KTMIN = EK_Q == 0 ? 16 : 32;
constexpr int KT = KT0 < KTMIN ? KTMIN : KT0 > 64 ? 64 : KT0;
constexpr int ST = KT / 16;                         // score tiles
constexpr int KE = 16 / CS;                         // elements of a 16-byte key load
constexpr int KL = DP / (4 * KE);                   // key loads per score tile and lane
// Elements of a value load: 16 lanes cover at most the whole head.
constexpr int VE0 = EK_Q == 0 ? 4 : 8;
constexpr int VE = VE0 * 16 > DP ? DP / 16 : VE0;
constexpr int PANELS = DP / (16 * VE);
constexpr int VR = KT / 4;                          // value rows per lane
constexpr int VW = VE * CS / 4 < 1 ? 1 : VE * CS / 4;  // words of a value load
constexpr int UNIT = 64;                            // keys: what chunks are multiples of
// Weights are exp2(s - m + LIFT). Fp16 has no more than 24 binary places below 1: lifted to
// 2^14, a weight keeps them down to 2^-39 of the largest one (131072 keys of a weight of 2^-26
// each are 0.2% of the sum). bf16 and fp32 have the exponents for it.
constexpr float LIFT = EK_Q == 1 ? 14.0f : 0.0f;

typedef uint32_t u32;
template <int W> struct words { u32 w[W]; };
template <int W> EK_INLINE words<W> load_words(const char* p) {
  words<W> r;
  ek::vload_u<uint8_t, W * 4>((uint8_t*)r.w, (const uint8_t*)p);
  return r;
}

struct Params {
  const T* q;
  const char* k;
  const char* v;
  const int32_t* table;
  const int32_t* lens;
  T* out;
  float* lse;
  float* part;                       // [item][head][dim + 2]: O, m, l
  int64_t q_row, q_head, out_row, out_head;   // elements
  int64_t c_page, c_token, c_head;   // bytes
  int64_t table_row, lens_step;      // elements
  int32_t batch, heads, group, dim, page, pages, capacity, window;
  uint32_t page_mul;
  int32_t page_shift, items, min_units;
  float scale, cap, v_scale;         // scale includes log2(e); cap in the same unit, or 0
};

EK_INLINE int page_of(const Params& a, int key) {
  return a.page == 1 ? key : (int)(__umulhi((u32)key, a.page_mul) >> a.page_shift);
}

// Keys that sequence b attends to: [first, first + count).
EK_INLINE void span_of(const Params& a, int b, int& first, int& count) {
  int n = b < a.batch ? a.lens[b * a.lens_step] : 0;
  n = n < 0 ? 0 : n > a.capacity ? a.capacity : n;
  first = a.window > 0 && n > a.window ? n - a.window : 0;
  count = n - first;
}

EK_INLINE int units_of(int count) { return (count + UNIT - 1) / UNIT; }

// The units of 64 keys per chunk, the same for every wave of both kernels.
EK_INLINE int chunk_units(const Params& a) {
  const int lane = ek::lane_id();
  int total = 0;
  for (int b = lane; b - lane < a.batch; b += 64) {
    int first, count;
    span_of(a, b, first, count);
    total += units_of(count);
  }
  total = ek::reduce_xor<ek::Sum, 1>(total);
  total = ek::reduce_xor<ek::Sum, 2>(total);
  total = ek::reduce_xor<ek::Sum, 4>(total);
  total = ek::reduce_xor<ek::Sum, 8>(total);
  total = ek::reduce_xor<ek::Sum, 16>(total);
  total = ek::reduce_xor<ek::Sum, 32>(total);
  const int u = (total + a.items - 1) / a.items;
  return u < a.min_units ? a.min_units : u;
}

EK_INLINE int chunks_of(int units, int per) { return (units + per - 1) / per; }

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
  const float r = (1.0f - e) / (1.0f + e);
  return __builtin_copysignf(y < 0.35f ? s : r, x);
}

#if EK_FP8
// Four e4m3 values as four 16-bit ones (exact).
EK_INLINE void widen4(u32 w, u32* lo, u32* hi) {
#if EK_Q == 1
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
#else
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
  const auto b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
#endif
  *lo = __builtin_bit_cast(u32, a);
  *hi = __builtin_bit_cast(u32, b);
}
#endif

#if EK_Q != 0
// acc += a b over 32 k values: four words of 16-bit pairs per lane and operand.
EK_INLINE void mma(ek::f32x4& acc, const u32* a, const u32* b) {
#if EK_Q == 1
  acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ek::pack<ek::f16x8>(a), ek::pack<ek::f16x8>(b),
                                               acc, 0, 0, 0);
#else
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ek::pack<ek::bf16x8>(a), ek::pack<ek::bf16x8>(b),
                                                acc, 0, 0, 0);
#endif
}
#if EK_Q == 1
typedef _Float16 half_t;
#else
typedef __bf16 half_t;
#endif
EK_INLINE u32 pack2(half_t a, half_t b) {
  return (u32)__builtin_bit_cast(uint16_t, a) | (u32)__builtin_bit_cast(uint16_t, b) << 16;
}
#endif

// The query heads as the products' operand: element chunk (s, c) of head r, in the order in
// which a lane reads its keys.
struct Query {
#if EK_Q == 0
  float w[KL][4];
#else
  u32 w[KL * KE / 8][4];
#endif
};

struct Tile {
  words<4> k[ST][KL];
  words<VW> v[VR][PANELS];
};

extern "C" __global__ __launch_bounds__(256) void ek_paged_attention(Params a) {
  __shared__ float s_o[WAVES][16][DP + 4];
  __shared__ float s_m[WAVES][16], s_l[WAVES][16];
  const int lane = ek::lane_id(), r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles16 = (a.group + 15) / 16;
  const int g = blockIdx.y / tiles16, h0 = (blockIdx.y - g * tiles16) * 16;
  const int nh = a.group - h0 < 16 ? a.group - h0 : 16;

  // which sequence and chunk this item is
  const int per = chunk_units(a);
  int item = blockIdx.x, b = -1, first = 0, count = 0, chunks = 0, all = 0;
  for (int base = 0; base < a.batch; base += 64) {
    int f, n;
    span_of(a, base + lane, f, n);
    const int mine = chunks_of(units_of(n), per);
    const int end = all + ek::wave_prefix_sum(mine);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(item < end);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      b = base + at;
      first = __builtin_amdgcn_readlane(f, at);
      count = __builtin_amdgcn_readlane(n, at);
      chunks = __builtin_amdgcn_readlane(mine, at);
      item -= __builtin_amdgcn_readlane(end, at) - chunks;
      break;
    }
    all = __builtin_amdgcn_readlane(end, 63);
  }
  if (b < 0) {
    // there are at least as many items past the last one as sequences without tokens
    // (chunks <= items + sequences with tokens): each finishes one of those
    int skip = blockIdx.x - all;
    for (int base = 0; base < a.batch; base += 64) {
      int f, n;
      span_of(a, base + lane, f, n);
      uint64_t none = __builtin_amdgcn_ballot_w64(base + lane < a.batch && n == 0);
      const int here = __builtin_popcountll(none);
      if (skip >= here) {
        skip -= here;
        continue;
      }
      for (; skip > 0; --skip) none &= none - 1;
      const int64_t e = base + __builtin_ctzll(none);
      for (int x = threadIdx.x; x < nh * a.dim; x += 256) {
        const int h = x / a.dim, d = x - h * a.dim, head = g * a.group + h0 + h;
        a.out[e * a.out_row + head * a.out_head + d] = ek::cvt<T>(0.0f);
        if (a.lse && d == 0) a.lse[e * a.heads + head] = -__builtin_inff();
      }
      return;
    }
    return;
  }
  const int units = units_of(count);
  const int lo_u = (int)((int64_t)units * item / chunks);
  const int hi_u = (int)((int64_t)units * (item + 1) / chunks);
  const int lo = first + lo_u * UNIT;
  const int hi = hi_u == units ? first + count : first + hi_u * UNIT;

  const char* kbase = a.k + g * a.c_head;
  const char* vbase = a.v + g * a.c_head;
  const int32_t* row = a.table + b * a.table_row;

  Query q;
  {
    const T* src = a.q + b * a.q_row + (int64_t)(g * a.group + h0 + r) * a.q_head;
    const bool head = r < nh;
#if EK_Q == 0
#pragma unroll
    for (int s = 0; s < KL; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = s * 16 + c * 4 + i;
        q.w[s][i] = head && d < a.dim ? src[d] : 0.0f;
      }
#else
#pragma unroll
    for (int s = 0; s < KL; ++s)
#pragma unroll
      for (int e = 0; e < KE / 8; ++e) {
        const int d = (s * 4 + c) * KE + e * 8;
        words<4> x = {{0, 0, 0, 0}};
        if (head && d < a.dim) x = load_words<4>((const char*)(src + d));
#pragma unroll
        for (int i = 0; i < 4; ++i) q.w[s * (KE / 8) + e][i] = x.w[i];
      }
#endif
  }

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
  const auto load_k = [&](Tile& t, int64_t off) {
#pragma unroll
    for (int s = 0; s < ST; ++s) {
      const char* p = kbase + ek::shfl(off, s * 16 + r);
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        const int d = (i * 4 + c) * KE;
        if (EK_PAD) {
          t.k[s][i] = words<4>{{0, 0, 0, 0}};
          if (d < a.dim) t.k[s][i] = load_words<4>(p + d * CS);
        } else {
          t.k[s][i] = load_words<4>(p + d * CS);
        }
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
        if (EK_PAD) {
          t.v[j][i] = words<VW>{};
          if (d < a.dim) t.v[j][i] = load_words<VW>(p + d * CS);
        } else {
          t.v[j][i] = load_words<VW>(p + d * CS);
        }
      }
    }
  };

  const int step = WAVES * KT;
  int base = lo + wave * KT;
  if (base < hi) {
    Tile t;
    uint64_t live, live_next = 0;
    int64_t off = offset(base, page_id(base), live);
    load_k(t, off);
    load_v(t, off);
    int id = page_id(base + step);
    for (;;) {
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
          for (int e = 0; e < 4; ++e) widen4(t.k[s][i].w[e], &x[2 * e], &x[2 * e + 1]);
          mma(acc[s], x, q.w[2 * i]);
          mma(acc[s], x + 4, q.w[2 * i + 1]);
#else
          mma(acc[s], t.k[s][i].w, q.w[i]);
#endif
        }
      }
      const int next = base + step;
      if (next < hi) {
        off = offset(next, id, live_next);
        id = page_id(next + step);
        load_k(t, off);
      }
      // softmax
      float mt = -__builtin_inff();
      const bool full = live == ~0ull;
#pragma unroll
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = acc[s][i] * a.scale;
          if (a.cap > 0.0f) x = a.cap * tanh_f(x / a.cap);
          if (!full && !(live >> (s * 16 + c * 4 + i) & 1)) x = -__builtin_inff();
          acc[s][i] = x;
          mt = __builtin_fmaxf(mt, x);
        }
      mt = ek::reduce_xor<ek::Max, 16>(mt);
      mt = ek::reduce_xor<ek::Max, 32>(mt);
      const float m_new = __builtin_fmaxf(m, mt);
      const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
      const float alpha = ek::exp2_fast(m - m_use);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int p = 0; p < PANELS; ++p)
#pragma unroll
        for (int e = 0; e < VE; ++e) o[p][e] *= alpha;
#pragma unroll
      for (int s = 0; s < ST; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[s][i] = ek::exp2_fast(acc[s][i] - (m_use - LIFT));
          l += acc[s][i];
        }
      // values without a key are taken as zeros: their memory may hold anything
      if (!full) {
#pragma unroll
        for (int j = 0; j < VR; ++j) {
          const bool ok = live >> ((j / 4) * 16 + c * 4 + (j & 3)) & 1;
#pragma unroll
          for (int p = 0; p < PANELS; ++p)
#pragma unroll
            for (int w = 0; w < VW; ++w) t.v[j][p].w[w] = ok ? t.v[j][p].w[w] : 0;
        }
      }
#if EK_Q == 0
#pragma unroll
      for (int j = 0; j < VR; ++j)
#pragma unroll
        for (int p = 0; p < PANELS; ++p)
#pragma unroll
          for (int e = 0; e < VE; ++e)
            o[p][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(ek::bits_f32(t.v[j][p].w[e]),
                                                           acc[j / 4][j & 3], o[p][e], 0, 0, 0);
#else
#pragma unroll
      for (int s = 0; s < ST; s += 2) {
        u32 ph[4], pl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = acc[s + i / 2][(i & 1) * 2], y = acc[s + i / 2][(i & 1) * 2 + 1];
          const half_t xh = (half_t)x, yh = (half_t)y;
          ph[i] = pack2(xh, yh);
          pl[i] = pack2((half_t)(x - (float)xh), (half_t)(y - (float)yh));
        }
#pragma unroll
        for (int p = 0; p < PANELS; ++p) {
          // eight keys' VE elements, 16 bits each
          u32 x[8][VE / 2];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const words<VW>& v = t.v[s * 4 + j][p];
#if EK_FP8
#pragma unroll
            for (int w = 0; w < VW; ++w) widen4(v.w[w], &x[j][2 * w], &x[j][2 * w + 1]);
#else
#pragma unroll
            for (int w = 0; w < VW; ++w) x[j][w] = v.w[w];
#endif
          }
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            u32 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = __builtin_amdgcn_perm(x[2 * i + 1][e / 2], x[2 * i][e / 2],
                                           e & 1 ? 0x07060302u : 0x05040100u);
            mma(o[p][e], w, ph);
            mma(o[p][e], w, pl);
          }
        }
      }
#endif
      if (next >= hi) break;
      load_v(t, off);
      base = next;
      live = live_next;
    }
  }

  // the four waves' parts of the chunk
  l = ek::reduce_xor<ek::Sum, 16>(l);
  l = ek::reduce_xor<ek::Sum, 32>(l);
  if (c == 0) {
    s_m[wave][r] = m - LIFT;
    s_l[wave][r] = l;
  }
#pragma unroll
  for (int p = 0; p < PANELS; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) s_o[wave][r][p * 16 * VE + (c * 4 + i) * VE + e] = o[p][e][i];
  __syncthreads();
  const int total = nh * a.dim;
  for (int x = threadIdx.x; x < total; x += 256) {
    const int h = x / a.dim, d = x - h * a.dim;
    float mm = s_m[0][h];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) mm = __builtin_fmaxf(mm, s_m[w][h]);
    const float mu = mm == -__builtin_inff() ? 0.0f : mm;
    float ll = 0.0f, oo = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = ek::exp2_fast(s_m[w][h] - mu);
      ll += s_l[w][h] * f;
      oo += s_o[w][h][d] * f;
    }
    const int head = g * a.group + h0 + h;
    if (chunks == 1) {
      const float y = ll > 0.0f || ll != ll ? oo / ll * a.v_scale : 0.0f;
      a.out[b * a.out_row + head * a.out_head + d] = ek::cvt<T>(y);
      if (a.lse && d == 0)
        a.lse[(int64_t)b * a.heads + head] =
            ll > 0.0f || ll != ll ? (mm + __builtin_log2f(ll)) * LN2 : -__builtin_inff();
    } else {
      float* dst = a.part + ((int64_t)blockIdx.x * a.heads + head) * (a.dim + 2);
      dst[d] = oo;
      if (d == 0) {
        dst[a.dim] = mm;
        dst[a.dim + 1] = ll;
      }
    }
  }
}

// One workgroup per sequence and query head: joins the chunks of a sequence that has several.
extern "C" __global__ __launch_bounds__(256) void ek_paged_attention_join(Params a) {
  __shared__ float s_o[WAVES][DP];
  __shared__ float s_m[WAVES], s_l[WAVES];
  const int lane = ek::lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b = blockIdx.x, head = blockIdx.y;
  const int per = chunk_units(a);
  int start = 0, chunks = 0;
  for (int base = 0; base <= b; base += 64) {
    int f, n;
    span_of(a, base + lane, f, n);
    const int mine = chunks_of(units_of(n), per);
    const int end = ek::wave_prefix_sum(mine);
    const int at = b - base < 63 ? b - base : 63;
    start += __builtin_amdgcn_readlane(end, at);
    chunks = __builtin_amdgcn_readlane(mine, at);
  }
  start -= chunks;
  if (chunks <= 1) return;
  float m = -__builtin_inff(), l = 0.0f, o[DP / 64];
#pragma unroll
  for (int i = 0; i < DP / 64; ++i) o[i] = 0.0f;
  for (int i = wave; i < chunks; i += WAVES) {
    const float* src = a.part + ((int64_t)(start + i) * a.heads + head) * (a.dim + 2);
    const float mi = src[a.dim], li = src[a.dim + 1];
    const float m_new = __builtin_fmaxf(m, mi);
    const float mu = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float fa = ek::exp2_fast(m - mu), fb = ek::exp2_fast(mi - mu);
    m = m_new;
    l = l * fa + li * fb;
#pragma unroll
    for (int k = 0; k < DP / 64; ++k) {
      const int d = k * 64 + lane;
      if (!EK_PAD || d < a.dim) o[k] = o[k] * fa + src[d] * fb;
    }
  }
  if (lane == 0) {
    s_m[wave] = m;
    s_l[wave] = l;
  }
#pragma unroll
  for (int k = 0; k < DP / 64; ++k) s_o[wave][k * 64 + lane] = o[k];
  __syncthreads();
  float mm = s_m[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) mm = __builtin_fmaxf(mm, s_m[w]);
  const float mu = mm == -__builtin_inff() ? 0.0f : mm;
  for (int d = threadIdx.x; d < a.dim; d += 256) {
    float ll = 0.0f, oo = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const float f = ek::exp2_fast(s_m[w] - mu);
      ll += s_l[w] * f;
      oo += s_o[w][d] * f;
    }
    const bool any = ll > 0.0f || ll != ll;
    a.out[b * a.out_row + head * a.out_head + d] =
        ek::cvt<T>(any ? oo / ll * a.v_scale : 0.0f);
    if (a.lse && d == 0)
      a.lse[(int64_t)b * a.heads + head] =
          any ? (mm + __builtin_log2f(ll)) * LN2 : -__builtin_inff();
  }
}
