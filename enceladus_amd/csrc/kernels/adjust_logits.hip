// Penalties for repeated tokens, biases, a temperature and a mask of allowed tokens on logits.
//
// Per row: x = logit; tokens of the row's history (its prompt, then what was generated):
// x = x > 0 ? x / repetition : x * repetition; with c the count among the generated ones,
// x -= frequency c + presence [c > 0]; x += bias (the sum of the entries with that id);
// x /= temperature where it is above 0; tokens whose mask bit is 0: -inf.
//
// One pass over the logits: a workgroup takes EK_N consecutive logits of a row into registers,
// marks the row's history and biases over them in the LDS, a word per logit (bit 31: the token
// occurs; bits 21 to 30: one more than the bias entry that holds its sum, or 0; bits 0 to 20: the
// count among generated tokens) and finishes them. Each of a row's workgroups reads the whole
// history, from the L2: a longer stretch (EK_N) reads it fewer times, a shorter one gives few
// rows more workgroups and overlaps one workgroup's counting with another's streaming.
// Measured: 256 x 128000 bf16 with histories of up to 4096, 20 biases and masks, 136 MB: 30 us, 4.6
// TB/s, 8 of them the histories' (the temperature alone: 21 us, 6.2 TB/s); one row of 32000 fp32, 700
// tokens: 4.9 us, a launch and three waits for loads. 32 x 150001
// fp16 with histories of up to 32768 and 300 biases, 20 MB: 12.4 us, of which the histories, read
// by 19 workgroups each, are 5 (more logits per workgroup, 16384 or 32768: 15.4 and 14.7).
//
// Macros: EK_Q (0 fp32, 1 fp16, 2 bf16), EK_N (logits per workgroup), EK_STREAM
// (the output is more than the caches keep: stored past them).
#include "enceladus_cdna4.h"

#if EK_Q == 0
typedef float T;
#elif EK_Q == 1
typedef _Float16 T;
#else
typedef ek::bf16 T;
#endif
constexpr int N = EK_N, THREADS = 512;
constexpr int V = 16 / sizeof(T);                   // logits of a vector access
constexpr int VN = N / (V * THREADS);               // vectors per thread
constexpr int MOST_BIASES = 1023;                   // 10 bits of a word
constexpr int ENTRY = 21;                           // the lowest of them
constexpr uint32_t SEEN = 1u << 31, COUNT = (1u << ENTRY) - 1;
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

// x / t, from r = 1 / t. Of 32-bit logits the rounded quotient; 16-bit ones take the product, off by
// less than 2^-22 of it before it is rounded to 2^-11 or 2^-8 (256 x 128000 bf16, all options: 30.5
// us, and 33.5 with the quotient).
EK_INLINE float divided(float x, float t, float r) {
  return EK_Q == 0 ? ek::quotient(x, t, r) : x * r;
}

extern "C" __global__ __launch_bounds__(THREADS) void ek_adjust_logits(Params a) {
  __shared__ __attribute__((aligned(16))) uint32_t s_mark[N];
  __shared__ __attribute__((aligned(16))) int32_t s_id[MOST_BIASES + 1];
  __shared__ __attribute__((aligned(16))) float s_bias[MOST_BIASES + 1];
  const int stretches = (a.vocab + N - 1) / N, tid = threadIdx.x;
  const int64_t b = blockIdx.x / stretches;
  const int v0 = (int)(blockIdx.x - b * stretches) * N;
  const int n = a.vocab - v0 < N ? a.vocab - v0 : N;
  const T* src = a.logits + b * a.row + v0;

  // Loads arrive in their order: the row's numbers, the first ids of its history and its first
  // biases, which are marked first, then the logits and the mask, which are on their way meanwhile
  // (256 x 128000 bf16 with histories of up to 4096: 41.6 us with the logits first, 34.2 so).
  int len = a.tokens ? a.token_lens ? a.token_lens[b * a.lens_step] : a.history : 0;
  len = len < 0 ? 0 : len > a.history ? a.history : len;
  const int prompt = a.prompt_lens ? a.prompt_lens[b * a.prompt_step] : 0;
  const float rep = a.repetition ? a.repetition[b * a.rep_step] : a.rep;
  const float freq = a.frequency ? a.frequency[b * a.freq_step] : a.freq;
  const float pres = a.presence ? a.presence[b * a.pres_step] : a.pres;
  const float temp = a.temperature ? a.temperature[b * a.temp_step] : a.temp;
  const int32_t* row = a.tokens + b * a.token_row;
  int32_t ids[4] = {-1, -1, -1, -1};
  if (a.tokens) {
    if (tid * 4 + 4 <= a.history) {
      ek::vload_u<int32_t, 4>(ids, row + tid * 4);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (tid * 4 + j < a.history) ids[j] = row[tid * 4 + j];
    }
  }
  int32_t bias_id = -1;
  float bias = 0.0f;
  if (tid < a.biases) {
    bias_id = a.bias_ids[b * a.id_row + tid];
    bias = a.bias[b * a.bias_row + tid];
  }
  T x[VN][V];
  uint32_t bits[VN];
  const uint32_t* allowed = a.allowed ? a.allowed + b * a.allowed_row : nullptr;
#pragma unroll
  for (int i = 0; i < VN; ++i) {
    const int at = (i * THREADS + tid) * V;
    bits[i] = ~0u;
    if (allowed && at < n) bits[i] = allowed[(v0 + at) >> 5];
    if (at + V <= n) {
      ek::vload_u<T, V>(x[i], src + at);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = at + j < n ? src[at + j] : ek::cvt<T>(0.0f);
    }
  }
  const bool marks = a.tokens != nullptr || a.biases > 0;
  if (marks) {
    for (int i = tid * 4; i < N; i += THREADS * 4)
      *(ek::u32x4*)(s_mark + i) = ek::u32x4{0, 0, 0, 0};
    if (tid < a.biases) {
      s_id[tid] = bias_id;
      s_bias[tid] = bias;
    }
    if (tid < (-a.biases & 3)) s_id[a.biases + tid] = -1;    // up to whole vectors
    for (int i = tid + THREADS; i < a.biases; i += THREADS) {
      s_id[i] = a.bias_ids[b * a.id_row + i];
      s_bias[i] = a.bias[b * a.bias_row + i];
    }
    __syncthreads();
  }
  if (a.tokens) {
    const auto prompted = [&](int32_t id) {
      const uint32_t at = (uint32_t)id - (uint32_t)v0;
      if (at < (uint32_t)n) atomicOr(&s_mark[at], SEEN);
    };
    const auto generated = [&](int32_t id) {
      const uint32_t at = (uint32_t)id - (uint32_t)v0;
      if (at < (uint32_t)n) atomicAdd(&s_mark[at], 1u);
    };
    // Tokens `from` to `to`, four vectors of ids on their way at once.
    const auto each = [&](int from, int to, const auto& count) {
      constexpr int STEP = THREADS * 4;
      int i = from + tid * 4;
      for (; i + 3 * STEP + 4 <= to; i += 4 * STEP) {
        int32_t id[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) ek::vload_u<int32_t, 4>(id[k], row + i + k * STEP);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) count(id[k][j]);
      }
      for (; i < to; i += STEP) {
        if (i + 4 <= to) {
          int32_t id[4];
          ek::vload_u<int32_t, 4>(id, row + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) count(id[j]);
        } else {
          for (int j = i; j < to; ++j) count(row[j]);
        }
      }
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (tid * 4 + j < len) {
        if (tid * 4 + j < prompt) prompted(ids[j]);
        else generated(ids[j]);
      }
    constexpr int FIRST = THREADS * 4;
    const int middle = prompt < FIRST ? FIRST : prompt > len ? len : prompt;
    each(FIRST, middle, prompted);
    each(middle, len, generated);
  }
  if (a.biases > 0) {
    // Entries count themselves in first. One that is alone with its id stands for itself; of
    // several, the first adds all of them up in their order. (Each thread has read what it
    // adds before the first write to an entry.)
    constexpr int EACH = (MOST_BIASES + THREADS) / THREADS;
    uint32_t at[EACH];
    float sum[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = k * THREADS + tid;
      at[k] = i < a.biases && s_id[i] >= 0 ? (uint32_t)s_id[i] - (uint32_t)v0 : ~0u;
      if (at[k] < (uint32_t)n) atomicAdd(&s_mark[at[k]], 1u << ENTRY);
    }
    __syncthreads();
    uint32_t change[EACH];
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const int i = k * THREADS + tid;
      change[k] = 0;
      if (at[k] >= (uint32_t)n) continue;
      const uint32_t entries = s_mark[at[k]] >> ENTRY & MOST_BIASES;
      bool first = true;
      sum[k] = s_bias[i];
      if (entries > 1) {
        const int32_t id = s_id[i];
        sum[k] = 0.0f;
#pragma unroll 4
        for (int j = 0; j < a.biases; j += 4) {
          int32_t ids4[4];
          float bias4[4];
          ek::vload<int32_t, 4>(ids4, s_id + j);
          ek::vload<float, 4>(bias4, s_bias + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool same = ids4[e] == id;
            first &= !(same && j + e < i);
            sum[k] = same ? sum[k] + bias4[e] : sum[k];
          }
        }
      }
      if (first) change[k] = ((uint32_t)(i + 1) - entries) << ENTRY;
      else at[k] = ~0u;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (at[k] < (uint32_t)n) {
        s_bias[k * THREADS + tid] = sum[k];
        atomicAdd(&s_mark[at[k]], change[k]);
      }
  }
  if (marks) __syncthreads();

  // lift: the reciprocal of a temperature below 2^-128 would be infinite, and 0 times that NaN
  const float lift = temp > 0.0f && temp < 0x1p-100f ? 0x1p60f : 1.0f;
  const float rrep = 1.0f / rep, t = temp > 0.0f ? temp * lift : 1.0f, rt = 1.0f / t;
  T* dst = a.out + b * a.out_row + v0;
#pragma unroll
  for (int i = 0; i < VN; ++i) {
    const int at = (i * THREADS + tid) * V;
    if (at >= n) break;
    const uint32_t ok = bits[i] >> ((v0 + at) & 31);
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = ek::f32(x[i][j]);
    if (marks) {
      uint32_t w[V], any = 0;
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const ek::u32x4 u = *(const ek::u32x4*)(s_mark + at + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) any |= w[j + k] = u[k];
      }
      if (any) {                     // most tokens are not in the history
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (w[j] & (SEEN | COUNT))
            f[j] = f[j] > 0.0f ? divided(f[j], rep, rrep) : f[j] * rep;
          const uint32_t c = w[j] & COUNT;
          if (c) f[j] = f[j] - freq * (float)c - pres;
          const uint32_t e = w[j] >> ENTRY & MOST_BIASES;
          if (e) f[j] += s_bias[e - 1];
        }
      }
    }
    T y[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float z = divided(f[j] * lift, t, rt);
      y[j] = ek::cvt<T>(ok >> j & 1 ? z : -__builtin_inff());
    }
    if (at + V <= n) {
      if constexpr (EK_STREAM) ek::vstore_nt_u<T, V>(dst + at, y);
      else ek::vstore_u<T, V>(dst + at, y);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (at + j < n) dst[at + j] = y[j];
    }
  }
}
