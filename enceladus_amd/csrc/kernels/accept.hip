// Which drafted tokens the model itself would have chosen: the largest logit of every drafted
// token's row, then each sequence's walk from its first token to the child that is that choice.
//
// The first kernel reads the logits once, which is the time of a large call (the HBM rate); a small
// one is two launches. A lane keeps the largest of each vector that it reads and which vector that
// was, two instructions per logit; only the row's best vector is looked into, by the second kernel
// (every lane's own, in the first, read them twice as far as memory goes: 1381 rows of 128000 bf16,
// 354 MB, 151 us a call instead of 62). Whole numbers alone leave it: the order of a row's
// stretches does not matter. Of the 354 MB the first kernel takes 57.7 us, 6.1 TB/s, and the walks
// 6; of 16 rows of 32000, 2.8 and 4.4 us, a launch and a chain of loads each.
//
// Macros: EK_Q (logits: 0 fp32, 1 fp16, 2 bf16).
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
typedef uint32_t u32;
constexpr int E = 16 / sizeof(T);                   // logits of a vector
constexpr int THREADS = 256, UNROLL = 8;
constexpr int MOST = 1024;                          // nodes of a tree

struct Params {
  const T* logits;
  const int32_t* tokens;
  const int32_t* cu;
  const int32_t* tree;               // [rows, words], or null: chains
  int32_t* path;                     // [batch, most]
  int32_t* count;
  int32_t* chosen;
  uint64_t* best;                    // [rows, pieces]: a stretch's largest value, and its vector
  int64_t logits_row, tokens_step, cu_step, tree_row;
  int32_t rows, vocab, batch, words, most, pieces, span;
};

// A whole number that orders as the value does, NaN above all, 0 and -0 alike; and the place, the
// lower the better.
EK_INLINE uint64_t rank(float x, u32 at) {
  const u32 u = ek::f32_bits(x + 0.0f);
  const u32 key = x != x ? ~0u : u & 0x80000000u ? ~u : u | 0x80000000u;
  return (uint64_t)key << 32 | (u32)~at;
}
EK_INLINE int place(uint64_t r) { return (int)~(u32)r; }

EK_INLINE uint64_t larger(uint64_t a, uint64_t b) { return a > b ? a : b; }
template <int MASK> EK_INLINE uint64_t larger_of(uint64_t x) {
  return larger(x, ek::shfl_xor<MASK>(x));
}
EK_INLINE uint64_t largest(uint64_t x) {
  x = larger_of<1>(x);
  x = larger_of<2>(x);
  x = larger_of<4>(x);
  x = larger_of<8>(x);
  x = larger_of<16>(x);
  return larger_of<32>(x);
}

// A lane's largest so far, the vector that it is in, and the first vector with a NaN.
struct Top { float value; int at, nan_at; };

EK_INLINE void look_at(Top& top, const T* w, int at) {
  float m = ek::f32(w[0]);
  bool nan = false;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float x = ek::f32(w[e]), y = ek::f32(w[e + 1]);
    m = __builtin_fmaxf(m, __builtin_fmaxf(x, y));
    nan |= __builtin_isunordered(x, y);
  }
  top.at = m > top.value ? at : top.at;
  top.value = m > top.value ? m : top.value;
  top.nan_at = nan && at < top.nan_at ? at : top.nan_at;
}

extern "C" __global__ __launch_bounds__(THREADS) void ek_row_best(Params a) {
  __shared__ uint64_t s_best[THREADS / 64];
  const int row = blockIdx.x / (u32)a.pieces, piece = blockIdx.x - row * a.pieces;
  const T* x = a.logits + row * a.logits_row;
  const int begin = piece * a.span;
  const int end = a.vocab - begin < a.span ? a.vocab : begin + a.span;
  const int first = begin + threadIdx.x * E;
  constexpr int STEP = THREADS * E;
  Top top = {-__builtin_inff(), first, 0x7FFFFFFF};
  int base = begin;
  // whole rounds without a branch, so that all of their loads are on their way at once
  for (; base + STEP * UNROLL <= end; base += STEP * UNROLL) {
    T w[UNROLL][E];
#pragma unroll
    for (int k = 0; k < UNROLL; ++k)
      ek::vload_nt_u<T, E>(w[k], x + base + threadIdx.x * E + k * STEP);
#pragma unroll
    for (int k = 0; k < UNROLL; ++k) look_at(top, w[k], base + threadIdx.x * E + k * STEP);
  }
  for (; base < end; base += STEP) {
    const int at = base + threadIdx.x * E;
    T w[E];
    if (at + E <= end) ek::vload_nt_u<T, E>(w, x + at);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = at + e < end ? x[at + e] : ek::cvt<T>(-__builtin_inff());
    if (at < end) look_at(top, w, at);
  }
  uint64_t mine = rank(top.value, top.at);
  if (top.nan_at != 0x7FFFFFFF) mine = rank(__builtin_nanf(""), top.nan_at);
  if (first >= end) mine = 0;
  mine = largest(mine);
  if (ek::lane_id() == 0) s_best[threadIdx.x >> 6] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) mine = larger(mine, s_best[w]);
    a.best[blockIdx.x] = mine;
  }
}

// The place of a row's largest logit: the best of its stretches, then the first of its vector.
EK_INLINE int best_of(const Params& a, int row) {
  uint64_t r = 0;
#pragma unroll 4
  for (int p = 0; p < a.pieces; ++p) r = larger(r, a.best[(int64_t)row * a.pieces + p]);
  const int at = place(r);
  const T* x = a.logits + row * a.logits_row + at;
  float w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = ek::f32(x[at + e < a.vocab ? e : 0]);
  int found = 0;
#pragma unroll
  for (int e = E - 1; e >= 0; --e)
    if (at + e < a.vocab && rank(w[e], 0) >> 32 == r >> 32) found = e;
  return at + found;
}

extern "C" __global__ __launch_bounds__(THREADS) void ek_accept(Params a) {
  __shared__ int s_best[MOST], s_token[MOST], s_depth[MOST], s_stop;
  const int b = blockIdx.x, tid = threadIdx.x, lane = ek::lane_id();
  int begin = a.cu[b * a.cu_step], end = a.cu[(b + 1) * a.cu_step];
  begin = begin < 0 ? 0 : begin > a.rows ? a.rows : begin;
  end = end < begin ? begin : end > a.rows ? a.rows : end;
  int n = end - begin;
  int32_t* path = a.path + (int64_t)b * a.most;
  if (n == 0 || a.most == 0) {
    for (int i = tid; i < a.most; i += THREADS) path[i] = -1;
    if (tid == 0) a.count[b] = 0, a.chosen[b] = -1;
    return;
  }
  if (!a.tree) {                                   // a chain: until a token is not the choice
    const int all = n < a.most ? n : a.most;
    int count = all;
    if (tid == 0) s_stop = all;
    __syncthreads();
    for (int j0 = 1; j0 < all; j0 += THREADS) {
      const int j = j0 + tid;
      if (j < all && best_of(a, begin + j - 1) != a.tokens[(begin + j) * a.tokens_step])
        atomicMin(&s_stop, j);
      __syncthreads();
      count = s_stop;
      __syncthreads();                             // all have seen it before any goes on
      if (count < all) break;
    }
    for (int i = tid; i < a.most; i += THREADS) path[i] = i < count ? i : -1;
    if (tid == 0) a.count[b] = count, a.chosen[b] = best_of(a, begin + count - 1);
    return;
  }
  n = n < a.words * 32 ? n : a.words * 32;         // the others have no bit
  for (int j = tid; j < n; j += THREADS) {
    const int32_t* mask = a.tree + (begin + j) * a.tree_row;
    int depth = 0;
    for (int w = 0; w * 32 < n; ++w) {
      const u32 live = n - w * 32 < 32 ? (1u << (n - w * 32)) - 1 : ~0u;
      depth += __builtin_popcount((u32)mask[w] & live);
    }
    s_depth[j] = depth;
    s_token[j] = a.tokens[(begin + j) * a.tokens_step];
    s_best[j] = best_of(a, begin + j);
  }
  __syncthreads();
  if (tid >= 64) return;
  int now = 0, count = 1;
  if (lane == 0) path[0] = 0;
  while (count < a.most) {
    const int want = s_best[now], deep = s_depth[now] + 1;
    int next = -1;
    for (int j0 = 0; j0 < n && next < 0; j0 += 64) {
      const int j = j0 + lane;
      bool ok = j < n && j != now && s_token[j] == want && s_depth[j] == deep;
      if (ok) ok = (u32)a.tree[(begin + j) * a.tree_row + (now >> 5)] >> (now & 31) & 1;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(ok);
      if (hit) next = j0 + __builtin_ctzll(hit);
    }
    if (next < 0) break;
    now = next;
    if (lane == 0) path[count] = now;
    ++count;
  }
  for (int i = count + lane; i < a.most; i += 64) path[i] = -1;
  if (lane == 0) a.count[b] = count, a.chosen[b] = s_best[now];
}
