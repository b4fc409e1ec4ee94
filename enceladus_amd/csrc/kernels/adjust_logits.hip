// Penalties for repeated tokens, biases, a temperature and a mask of allowed tokens on logits.
//
// Per row: x = logit; tokens of the row's history (its prompt, then what was generated):
// x = x > 0 ? x / repetition : x * repetition; with c the count among the generated ones,
// x -= frequency c + presence [c > 0]; x += bias (the sum of the entries with that id);
// x /= temperature where it is above 0; tokens whose mask bit is 0: -inf.
//
// One pass over the logits: a workgroup takes EK_N consecutive logits of a row, counts the
// row's history over them in the LDS (bit 31: seen; the rest: the count among generated tokens)
// and streams the logits through. Each of a row's workgroups reads the whole history, which
// stays in the L2: a longer stretch (EK_N) reads it fewer times, a shorter one gives few rows
// more workgroups.
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_N (logits per workgroup), EK_THREADS, EK_BIAS.
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int N = EK_N, THREADS = EK_THREADS;
constexpr int V = 16 / sizeof(T);                   // logits of a vector access
constexpr int VN = N / (V * THREADS);               // vectors per thread
static_assert(VN * V * THREADS == N, "whole vectors");

struct Params {
  const T* logits;
  T* out;
  const int32_t* tokens;             // or null
  const int32_t* token_lens;         // or null: all of a row
  const int32_t* prompt_lens;        // or null: 0
  const float* repetition;           // each of these four: per row, or null for the number below
  const float* frequency;
  const float* presence;
  const float* temperature;
  const int32_t* bias_ids;
  const float* bias;
  const uint32_t* allowed;           // or null
  int64_t row, out_row, token_row, id_row, bias_row, allowed_row;   // elements
  int64_t lens_step, prompt_step, rep_step, freq_step, pres_step, temp_step;
  int32_t vocab, history, biases;
  float rep, freq, pres, temp;
};

extern "C" __global__ __launch_bounds__(THREADS) void ek_adjust_logits(Params a) {
  __shared__ __attribute__((aligned(16))) uint32_t s_count[N];
#if EK_BIAS
  __shared__ __attribute__((aligned(16))) float s_bias[N];
#endif
  const int stretches = (a.vocab + N - 1) / N, tid = threadIdx.x;
  const int64_t b = blockIdx.x / stretches;
  const int v0 = (int)(blockIdx.x - b * stretches) * N;
  const int n = a.vocab - v0 < N ? a.vocab - v0 : N;
  const T* src = a.logits + b * a.row + v0;

  // the logits are on their way while the history is counted
  T x[VN][V];
#pragma unroll
  for (int i = 0; i < VN; ++i) {
    const int at = (i * THREADS + tid) * V;
    if (at + V <= n) {
      ek::vload_u<T, V>(x[i], src + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = at + j < n ? src[at + j] : ek::cvt<T>(0.0f);
    }
  }
  const bool counts = a.tokens != nullptr;
  if (counts || EK_BIAS) {
    for (int i = tid * 4; i < N; i += THREADS * 4) {
      *(ek::u32x4*)(s_count + i) = ek::u32x4{0, 0, 0, 0};
#if EK_BIAS
      *(ek::u32x4*)(s_bias + i) = ek::u32x4{0, 0, 0, 0};
#endif
    }
    __syncthreads();
  }
  if (counts) {
    const int32_t* row = a.tokens + b * a.token_row;
    int len = a.token_lens ? a.token_lens[b * a.lens_step] : a.history;
    len = len < 0 ? 0 : len > a.history ? a.history : len;
    const int prompt = a.prompt_lens ? a.prompt_lens[b * a.prompt_step] : 0;
    const auto count = [&](int i, int32_t id) {
      const uint32_t at = (uint32_t)id - (uint32_t)v0;
      if (at < (uint32_t)n) {
        if (i < prompt) atomicOr(&s_count[at], 0x80000000u);
        else atomicAdd(&s_count[at], 1u);
      }
    };
    const int whole = len & ~3;
    for (int i = tid * 4; i < whole; i += THREADS * 4) {
      int32_t id[4];
      ek::vload_u<int32_t, 4>(id, row + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) count(i + j, id[j]);
    }
    if (tid < len - whole) count(whole + tid, row[whole + tid]);
  }
#if EK_BIAS
  {
    // the first of the entries with one id adds all of them up in their order: the sum does not
    // depend on which thread comes first
    const int32_t* ids = a.bias_ids + b * a.id_row;
    const float* val = a.bias + b * a.bias_row;
    for (int i = tid; i < a.biases; i += THREADS) {
      const int32_t id = ids[i];
      const uint32_t at = (uint32_t)id - (uint32_t)v0;
      if (id < 0 || at >= (uint32_t)n) continue;
      bool first = true;
      for (int j = 0; j < i && first; ++j) first = ids[j] != id;
      if (!first) continue;
      float sum = 0.0f;
      for (int j = i; j < a.biases; ++j)
        if (ids[j] == id) sum += val[j];
      s_bias[at] = sum;
    }
  }
#endif
  if (counts || EK_BIAS) __syncthreads();

  const float rep = a.repetition ? a.repetition[b * a.rep_step] : a.rep;
  const float freq = a.frequency ? a.frequency[b * a.freq_step] : a.freq;
  const float pres = a.presence ? a.presence[b * a.pres_step] : a.pres;
  const float temp = a.temperature ? a.temperature[b * a.temp_step] : a.temp;
  const float rrep = 1.0f / rep, rtemp = temp > 0.0f ? 1.0f / temp : 1.0f;
  T* dst = a.out + b * a.out_row + v0;
  const uint32_t* allowed = a.allowed ? a.allowed + b * a.allowed_row : nullptr;
#pragma unroll
  for (int i = 0; i < VN; ++i) {
    const int at = (i * THREADS + tid) * V;
    if (at >= n) break;
    uint32_t bits = ~0u;
    if (allowed) bits = allowed[(v0 + at) >> 5] >> ((v0 + at) & 31);
    T y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float f = ek::f32(x[i][j]);
      if (counts) {
        const uint32_t w = s_count[at + j];
        const uint32_t c = w & 0x7fffffffu;
        if (w) f = f > 0.0f ? f * rrep : f * rep;
        if (c) f = f - freq * (float)c - pres;
      }
#if EK_BIAS
      f += s_bias[at + j];
#endif
      f *= rtemp;
      if (!(bits >> j & 1)) f = -__builtin_inff();
      y[j] = ek::cvt<T>(f);
    }
    if (at + V <= n) {
      ek::vstore_u<T, V>(dst + at, y);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < n) dst[at + j] = y[j];
    }
  }
}
