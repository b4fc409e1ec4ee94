// New keys and values into a paged cache, their keys (and the queries) rotated by position.
//
// Token t, the i-th of the n new ones of sequence b, is at position p = lens[b] - n + i; its
// slot is token p % page of page table[b][p / page]. Rotation of the first `rotary` elements of
// a head, in pairs (x, y) = (j, j + rotary / 2), or (2 j, 2 j + 1) when EK_PAIRS:
// (x cos - y sin, y cos + x sin) with cos, sin at [p, j]. Cached values are divided by the
// cache's scale in 32 bits and rounded to its type (e4m3: saturated to +-448, NaN stays NaN).
//
// A handful of flops per element: the time is the bytes over the HBM rate, or a launch. A wave
// takes one token, or a part of its rows (query, key and value heads) when there are few tokens;
// a lane keeps one place in the head, so its cos and sin are read once for all rows, and pairs
// meet in one lane, so that queries can be rotated in place.
// Measured: 21152 tokens of 32 query, 8 key and 8 value heads of 128 in bf16, 531 MB: 90 us, 5.9
// TB/s (the framework's own copies: 6.4). One token of such heads: 3.2 us, a launch and a chain of
// loads. The same 531 MB by positions of three axes: 92 us, each pair's row of angles being its
// own; 115 to 120 with the axes woven pair by pair, a load for each pair. 378 drafted tokens by
// positions of their own: 5.5 us.
//
// Macros: EK_Q (new rows: 0 fp32, 1 fp16, 2 bf16), EK_FP8 (e4m3 cache), EK_V (elements of a
// vector access: a power of two up to 16 bytes that divides the parts of a head), EK_PAIRS,
// EK_STREAM (the rows are more than the caches keep: loaded and stored past them), EK_AXES (0:
// tokens turn by their slots' positions; else by positions of their own, up to four of them, of
// which each pair has one: 1 where the pairs of a vector have the same, 2 where they may differ).
#include "enceladus_cdna4.h"
#ifndef EK_AXES
#define EK_AXES 0
#endif

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int V = EK_V;

struct Params {
  const T* q;
  const T* k;
  const T* v;
  T* q_out;
  char* k_cache;
  char* v_cache;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;                 // [batch + 1], or null: one token of each sequence
  const float* cos;
  const float* sin;
#if EK_AXES
  const int32_t* turns;              // [axes][tokens]: the positions that tokens turn by
#endif
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, out_row, out_head;  // elements
  int64_t c_page, c_token, c_head;   // bytes
  int64_t table_row, lens_step, cu_step, cos_row, sin_row;
  int32_t tokens, batch, heads, kv_heads, dim, rotary, page, pages, capacity, positions;
  int32_t parts;                     // waves per token
  float k_scale, v_scale, k_inv, v_inv;   // and 1 / scale
#if EK_AXES
  int32_t axes;
  int64_t turn_axis, turn_step;
  uint64_t pair_axes[4];             // two bits a pair
#endif
};

EK_INLINE float sat8(float x) { return x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x; }

template <int N, typename S> EK_INLINE void put(S* p, const S* w) {
  if constexpr (EK_STREAM) ek::vstore_nt_u<S, N>(p, w);
  else ek::vstore_u<S, N>(p, w);
}

// V floats into the cache at p.
EK_INLINE void store_cache(char* p, const float* x, float scale, float inv) {
#if EK_FP8
  uint8_t w[V < 4 ? 4 : V];
#pragma unroll
  for (int i = 0; i < V; i += 4) {
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = i + j < V ? sat8(ek::quotient(x[i + j], scale, inv)) : 0.0f;
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    u = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], u, true);
    __builtin_memcpy(w + i, &u, 4);
  }
  put<V>((uint8_t*)p, w);
#else
  T w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = ek::cvt<T>(ek::quotient(x[i], scale, inv));
  put<V>((T*)p, w);
#endif
}

EK_INLINE void store_out(T* p, const float* x) {
  T w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = ek::cvt<T>(x[i]);
  put<V>(p, w);
}

template <bool NT = false, typename S> EK_INLINE void load(float* x, const S* p) {
  S w[V];
  constexpr int M = sizeof(S) * V > 16 ? 16 / sizeof(S) : V;
#pragma unroll
  for (int i = 0; i < V; i += M) {
    if constexpr (NT) ek::vload_nt_u<S, M>(w + i, p + i);
    else ek::vload_u<S, M>(w + i, p + i);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = ek::f32(w[i]);
}

__device__ const float s_zeros[8] = {};              // what is no cos or sin

#if EK_AXES
// The row of cos and sin by which pair j turns, of those on the four axes.
EK_INLINE int turn_at(const Params& a, int j, int on0, int on1, int on2, int on3) {
  const uint64_t w = j < 64 ? j < 32 ? a.pair_axes[0] : a.pair_axes[1]
                            : j < 96 ? a.pair_axes[2] : a.pair_axes[3];
  const int x = (int)(w >> 2 * (j & 31)) & 3;
  return x < 2 ? x < 1 ? on0 : on1 : x < 3 ? on2 : on3;
}
#endif

extern "C" __global__ __launch_bounds__(256) void ek_append_kv(Params a) {
  const int lane = ek::lane_id();
  const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = (int)(unit / (uint32_t)a.parts), part = (int)unit - t * a.parts;
  if (t >= a.tokens) return;

  int b = t, back = 1;               // the sequence, and how far before its end the token is
  if (a.cu) {
    // sequences that end before the token: of many, first the stretches whose last one does
    const auto ends = [&](int i) { return a.cu[((i < a.batch ? i : a.batch - 1) + 1) * a.cu_step]; };
    b = 0;
    int count = a.batch;
    while (count > 256) {
      const int step = (count + 63) / 64, at = (lane + 1) * step - 1;
      const int over = __builtin_popcountll(
          __builtin_amdgcn_ballot_w64(ends(b + at) <= t && at < count));
      b += over * step;
      count = count - over * step < step ? count - over * step : step;
    }
    int end[4];                      // on their way at once
#pragma unroll
    for (int k = 0; k < 4; ++k) end[k] = ends(b + k * 64 + lane);
    int over = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      over += __builtin_popcountll(
          __builtin_amdgcn_ballot_w64(k * 64 + lane < count && end[k] <= t));
    b += over;
    if (b >= a.batch) return;
  }
  int len = a.lens[b * a.lens_step];
  if (a.cu) {
    int begin = a.cu[b * a.cu_step], end = a.cu[(b + 1) * a.cu_step];
    asm volatile("" : "+s"(begin), "+s"(end), "+s"(len));    // one wait for the three
    if (begin > t) return;
    back = end - t;
  }
  const int pos = (len > 0 ? len : 0) - back;      // a negative length is none: no wrapping round
#if EK_AXES
  if (pos < 0 || pos >= a.capacity) return;
  // its rows of cos and sin, on their way at once: an axis that is not there is the first
  const int32_t* turns = a.turns + t * a.turn_step;
  const int on0 = turns[0], on1 = turns[a.axes > 1 ? a.turn_axis : 0];
  const int on2 = turns[a.axes > 2 ? 2 * a.turn_axis : 0];
  const int on3 = turns[a.axes > 3 ? 3 * a.turn_axis : 0];
  const uint32_t most = a.positions;
  if ((uint32_t)on0 >= most || (uint32_t)on1 >= most || (uint32_t)on2 >= most ||
      (uint32_t)on3 >= most)
    return;
#else
  if (pos < 0 || pos >= a.capacity || (a.rotary && pos >= a.positions)) return;
#endif
  const int pg = pos / a.page, page_id = a.table[b * a.table_row + pg];

  // places of a head: `pairs` of two vectors that are rotated together, then single vectors
  const int half = a.rotary / 2;
  const int pairs = EK_PAIRS ? 0 : half / V;
  const int places = EK_PAIRS ? a.dim / V : pairs + (a.dim - a.rotary) / V;
  const int lanes = places < 64 ? 64 / places : 1;   // rows at once
  const int sub = lane / places;
  const int rows = a.heads + 2 * a.kv_heads;
  if (places <= 64 && sub >= lanes) return;

  for (int place = places <= 64 ? lane - sub * places : lane; place < places; place += 64) {
    const bool two = place < pairs;
    const int d = two ? place * V : EK_PAIRS ? place * V : a.rotary + (place - pairs) * V;
    float cs[V], sn[V];
    const bool turn = EK_PAIRS ? d < a.rotary : two;
    // where nothing turns, zeros, so that no branch has to wait for what it loaded
    const int j0 = EK_PAIRS ? d / 2 : d;               // the vector's first pair
#if EK_AXES == 2
#pragma unroll
    for (int i = 0; i < (EK_PAIRS ? V / 2 : V); ++i) {
      const int at = turn_at(a, turn ? j0 + i : 0, on0, on1, on2, on3);
      cs[i] = turn ? a.cos[at * a.cos_row + j0 + i] : 0.0f;
      sn[i] = turn ? a.sin[at * a.sin_row + j0 + i] : 0.0f;
    }
#else
#if EK_AXES
    const int at = turn_at(a, turn ? j0 : 0, on0, on1, on2, on3);
#else
    const int at = pos;
#endif
    const float* cp = turn ? a.cos + at * a.cos_row + j0 : s_zeros;
    const float* sp = turn ? a.sin + at * a.sin_row + j0 : s_zeros;
    if constexpr (EK_PAIRS) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) cs[i] = cp[i], sn[i] = sp[i];
    } else {
      load(cs, cp);
      load(sn, sp);
    }
#endif
    for (int row = part * lanes + (places <= 64 ? sub : 0); row < rows;
         row += a.parts * lanes) {
      const bool is_q = row < a.heads, is_k = !is_q && row < a.heads + a.kv_heads;
      const int h = is_q ? row : is_k ? row - a.heads : row - a.heads - a.kv_heads;
      const T* src = (is_q ? a.q + t * a.q_row + h * a.q_head
                      : is_k ? a.k + t * a.k_row + h * a.k_head
                             : a.v + t * a.v_row + h * a.v_head) + d;
      float x[V], y[V];
      load<EK_STREAM>(x, src);
      // without a branch, whose wait for the first load would come before the second
      if constexpr (!EK_PAIRS) load<EK_STREAM>(y, src + (two ? half : 0));
      // the page is looked at with the first row on its way (and not moved in front of that)
      int id;
      asm volatile("v_mov_b32 %0, %1" : "=v"(id) : "v"(page_id));
      if ((uint32_t)id >= (uint32_t)a.pages) return;
      const int64_t slot = id * a.c_page + (pos - pg * a.page) * a.c_token;
      if (turn && (is_q || is_k)) {
        if constexpr (EK_PAIRS) {
#pragma unroll
          for (int i = 0; i < V; i += 2) {
            const float u = x[i], w = x[i + 1];
            x[i] = u * cs[i / 2] - w * sn[i / 2];
            x[i + 1] = w * cs[i / 2] + u * sn[i / 2];
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = x[i], w = y[i];
            x[i] = u * cs[i] - w * sn[i];
            y[i] = w * cs[i] + u * sn[i];
          }
        }
      }
      if (is_q) {
        T* dst = a.q_out + t * a.out_row + h * a.out_head + d;
        store_out(dst, x);
        if (two) store_out(dst + half, y);
      } else {
        char* dst = (is_k ? a.k_cache : a.v_cache) + slot + h * a.c_head +
                    (int64_t)d * (EK_FP8 ? 1 : sizeof(T));
        const float scale = is_k ? a.k_scale : a.v_scale, inv = is_k ? a.k_inv : a.v_inv;
        store_cache(dst, x, scale, inv);
        if (two) store_cache(dst + (int64_t)half * (EK_FP8 ? 1 : sizeof(T)), y, scale, inv);
      }
    }
  }
}
