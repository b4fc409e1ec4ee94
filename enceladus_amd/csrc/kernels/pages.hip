// The pages of paged caches: copied, compacted in place, shared by several sequences, taken and
// given back. `refs[p]` counts the sequences that hold page p (0: free, below 0: never taken);
// row b of the block table holds the pages of sequence b's lens[b] tokens.
//
// All of these move or count bytes; none computes. Copies run at the HBM rate when they are large
// and cost a launch and a chain of dependent loads (counts, ids, pages) when they are small. Every
// layer's caches have the same pages, so one launch takes them all: their addresses are kernel
// arguments. 1258 MB of whole pages copied: 197 us, 6.4 TB/s; 192 forks, 206 MB: 5 us for the plan
// and 36 for the copies; what is kept of 64 sequences' up to 27 drafted tokens moved together in 32
// caches, 22 MB: 8 us; 256 sequences take pages: 5 us, and give them back: 3. Long histories are
// compacted far below that rate: see ek_compact.
//
// Macros: EK_CACHES (addresses in the argument block), EK_V (bytes of an access: the largest power
// of two up to 16 that divides a head), EK_STREAM (more bytes than the caches keep: past them).
#include "enceladus_cdna4.h"

constexpr int V = EK_V;
typedef uint32_t u32;

struct Params {
  char* caches[EK_CACHES];
  int32_t* refs;
  int32_t* table;
  int32_t* lens;
  const int32_t* first;              // sources; compact: starts; take, free: new lengths
  const int32_t* second;             // targets; compact: the tokens kept
  const int32_t* counts;             // compact: how many are kept
  int32_t* served;
  int32_t* work;                     // see ek_take_pages, ek_fork_plan
  int64_t c_page, c_token, c_head;   // bytes
  int64_t table_row, lens_step, first_step, second_step, counts_step;   // elements
  int32_t n, rows, width, pages, page, heads, row_bytes, caches_used, pieces, most;
};

EK_INLINE void get(uint8_t* w, const char* p) {
  if constexpr (EK_STREAM) ek::vload_nt_u<uint8_t, V>(w, (const uint8_t*)p);
  else ek::vload_u<uint8_t, V>(w, (const uint8_t*)p);
}
EK_INLINE void put(char* p, const uint8_t* w) {
  if constexpr (EK_STREAM) ek::vstore_nt_u<uint8_t, V>((uint8_t*)p, w);
  else ek::vstore_u<uint8_t, V>((uint8_t*)p, w);
}

// Where chunk i of a page's first `tokens` tokens is: in the order in which they lie in memory,
// runs of adjacent chunks, of which `mid` are `near` bytes apart, and those `far`.
struct Walk {
  u32 run, mid;
  int64_t near, far;
  EK_INLINE Walk(const Params& a, int tokens) {
    run = (u32)(a.row_bytes / V), mid = 1, near = 0, far = a.c_token;
    if (a.heads > 1 && a.c_token >= a.c_head) mid = a.heads, near = a.c_head;
    if (a.heads > 1 && a.c_token < a.c_head) mid = tokens, near = a.c_token, far = a.c_head;
    if (near == a.row_bytes) run *= mid, mid = 1;
    if (mid == 1 && far == (int64_t)run * V) run = ~0u;      // all of them
  }
  EK_INLINE int64_t operator()(u32 i) const {
    if (run == ~0u) return (int64_t)i * V;
    const u32 q = i / run, o = mid == 1 ? q : q / mid;
    return o * far + (q - o * mid) * near + (int64_t)(i - q * run) * V;
  }
};

constexpr int THREADS = 256;
// Accesses of a thread: whole pages are copied best by small pieces (1258 MB: 197 us with 1, 228
// with 2, 238 with 4, 243 with 8), parts of them by few (192 forks of 7 tokens in 32 caches, 206
// MB: 34 us with 8, 39 with 4, 60 with 1).
constexpr int COPY = 1, FORK = 8;

// `tokens` tokens of page `from` into page `to`: piece `piece` of them, in one cache.
template <int N> EK_INLINE void copy_piece(const Params& a, char* cache, int from, int to,
                                           int tokens, int piece) {
  const u32 all = (u32)tokens * (u32)a.heads * (u32)(a.row_bytes / V);
  const char* src = cache + from * a.c_page;
  char* dst = cache + to * a.c_page;
  const u32 base = (u32)piece * (THREADS * N) + threadIdx.x;
  const Walk place(a, tokens);
  uint8_t w[N][V];
  int64_t at[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const u32 i = base + k * THREADS;
    at[k] = place(i < all ? i : 0);
    if (i < all) get(w[k], src + at[k]);
  }
#pragma unroll
  for (int k = 0; k < N; ++k)
    if (base + k * THREADS < all) put(dst + at[k], w[k]);
}

// Page second[i] becomes page first[i], in every cache. Ids outside of the cache: no copy.
extern "C" __global__ __launch_bounds__(THREADS) void ek_copy_pages(Params a) {
  const int i = blockIdx.x / (u32)a.pieces, piece = blockIdx.x - i * a.pieces;
  const int from = a.first[i * a.first_step], to = a.second[i * a.second_step];
  if ((u32)from >= (u32)a.pages || (u32)to >= (u32)a.pages || from == to) return;
  copy_piece<COPY>(a, a.caches[blockIdx.y], from, to, a.page, piece);
}

// Token first[b] + second[b][i] becomes token first[b] + i of sequence b, for i < counts[b], in
// every cache. The tokens kept ascend, so each moves to the front or stays, and a slot is read
// before any later token is written to it: a wave takes one part of the heads of a sequence's
// tokens in one cache through all of them, in their order, and reads BATCH of them before it
// writes those (what later ones are read from lies behind all that is written before). So few
// sequences are few waves, each bound by its round trips: of 8192 tokens in 32 caches every second
// one kept, 537 MB, takes 1930 us; of 8 such sequences, 4.3 GB, 2570 us, 1.7 TB/s; of 64 with 1024
// tokens, 4.3 GB, 907 us, 4.7 TB/s.
constexpr int BATCH = 16;
EK_INLINE int64_t lane_value(int64_t x, int lane) {
  return (int64_t)((uint64_t)(u32)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 |
                   (u32)__builtin_amdgcn_readlane((int)x, lane));
}
extern "C" __global__ __launch_bounds__(64) void ek_compact(Params a) {
  const int lane = ek::lane_id(), b = blockIdx.x / (u32)a.pieces;
  const int part = blockIdx.x - b * a.pieces;
  int count = a.counts[b * a.counts_step];
  const int start = a.first[b * a.first_step];
  count = count < 0 ? 0 : count > a.most ? a.most : count;
  const int64_t capacity = (int64_t)a.width * a.page;
  if (start < 0) return;
  if (a.lens && part == 0 && blockIdx.y == 0 && lane == 0) {
    const int64_t len = (int64_t)start + count;
    a.lens[b * a.lens_step] = len < 0x7FFFFFFF ? (int)len : 0x7FFFFFFF;
  }
  if (start >= capacity) return;                   // nothing is there to move
  const u32 per = (u32)(a.row_bytes / V), chunk = (u32)part * 64 + lane;
  const bool mine = chunk < per * (u32)a.heads;
  const u32 h = mine ? chunk / per : 0;
  char* base = a.caches[blockIdx.y] + h * a.c_head + (mine ? (int64_t)(chunk - h * per) * V : 0);
  const int32_t* keep = a.second + b * a.second_step;
  const int32_t* row = a.table + b * a.table_row;
  for (int i0 = 0; i0 < count; i0 += 64) {
    // 64 tokens' slots at once, a lane each: byte offsets in the cache, or -1
    int64_t from = -1, to = -1;
    if (i0 + lane < count) {
      const int k = keep[i0 + lane];
      const int64_t old = (int64_t)start + k, now = (int64_t)start + i0 + lane;
      if (k > i0 + lane && old < capacity) {
        // now < old: both fit 32 bits, like the capacity
        const int po = (int)((u32)old / (u32)a.page), pn = (int)((u32)now / (u32)a.page);
        const int ido = row[po], idn = row[pn];
        if ((u32)ido < (u32)a.pages && (u32)idn < (u32)a.pages) {
          from = ido * a.c_page + (old - (int64_t)po * a.page) * a.c_token;
          to = idn * a.c_page + (now - (int64_t)pn * a.page) * a.c_token;
        }
      }
    }
    uint64_t todo = __builtin_amdgcn_ballot_w64(to >= 0);
    while (todo) {
      uint8_t w[BATCH][V];
      int64_t at[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        at[k] = -1;
        if (todo) {
          const int l = __builtin_ctzll(todo);
          todo &= todo - 1;
          at[k] = lane_value(to, l);
          const int64_t of = lane_value(from, l);
          if (mine) get(w[k], base + of);
        }
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (at[k] >= 0 && mine) put(base + at[k], w[k]);
      asm volatile("" ::: "memory");               // later loads stay behind these stores
    }
  }
}

EK_INLINE int pages_of(int64_t tokens, int page) { return (int)((tokens + page - 1) / page); }

// Sequence b is cut to first[b] tokens (no longer than it is): the pages behind them lose a
// holder. A count never falls below 0: each of the decrements that the count allows meets a value
// above 0, in any order, and a further one is taken back. So a count that is seen at 0 or below has
// no decrement left; one that began there is not touched (-2^31 would wrap round under another
// row's eyes).
extern "C" __global__ __launch_bounds__(THREADS) void ek_free_pages(Params a) {
  const int b = blockIdx.x, len = a.lens[b * a.lens_step];
  int to = a.first ? a.first[b * a.first_step] : 0;
  to = to < 0 ? 0 : to;
  __syncthreads();                                 // all have read the length
  if (to >= len) return;
  const int have = pages_of(len, a.page), end = have < a.width ? have : a.width;
  for (int i = pages_of(to, a.page) + threadIdx.x; i < end; i += THREADS) {
    const int id = a.table[b * a.table_row + i];
    if ((u32)id < (u32)a.pages && a.refs[id] > 0 && atomicSub(&a.refs[id], 1) <= 0)
      atomicAdd(&a.refs[id], 1);
  }
  if (threadIdx.x == 0) a.lens[b * a.lens_step] = to;
}

// -- one workgroup of 1024: what is served in an order ---------------------------------------

constexpr int WG = 1024;

// The sum of x (at most 2^25, so that a wave's is below 2^32) over the threads before this one,
// and over all of them.
EK_INLINE int64_t scan_group(u32 x, int64_t* total, u32* s_wave) {
  const int lane = ek::lane_id(), wave = threadIdx.x >> 6;
  const u32 end = ek::wave_prefix_sum(x);
  __syncthreads();                                 // s_wave may still be read
  if (lane == 63) s_wave[wave] = end;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < WG / 64; ++w) {
    const u32 y = s_wave[w];
    before += w < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + end - x;
}

constexpr int EACH = 8;                            // counts of a thread and round
struct Counts { int32_t r[EACH]; };

// The counts of this thread's pages from p on (1 behind the last).
EK_INLINE Counts counts_at(const Params& a, int p) {
  Counts c;
  if (p + EACH <= a.pages) {
    ek::vload_u<int32_t, 4>(c.r, a.refs + p);
    ek::vload_u<int32_t, 4>(c.r + 4, a.refs + p + 4);
  } else {
#pragma unroll
    for (int k = 0; k < EACH; ++k) c.r[k] = p + k < a.pages ? a.refs[p + k] : 1;
  }
  return c;
}

// The lowest `want` free pages into `found`, in their order; how many there are. `c`: the counts of
// the first round, read before they are needed.
EK_INLINE int find_free(const Params& a, int want, int32_t* found, u32* s_wave, Counts c) {
  int have = 0;
  for (int base = 0; base < a.pages && have < want; base += WG * EACH) {
    const int p = base + threadIdx.x * EACH;
    if (base > 0) c = counts_at(a, p);
    int count = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) count += c.r[k] == 0;
    int64_t total;
    int at = have + (int)scan_group(count, &total, s_wave);
#pragma unroll
    for (int k = 0; k < EACH; ++k)
      if (c.r[k] == 0) {
        if (at < want) found[at] = p + k;
        ++at;
      }
    have += (int)total;
  }
  __syncthreads();                                 // `found` is read by others next
  return have < want ? have : want;
}

// What threads exchange about up to SMALL rows is in the LDS, of more in memory.
constexpr int SMALL = 4096;

// Pages that row b still needs for first[b] tokens, or -1 where it can't have them.
EK_INLINE int need_of(const Params& a, int b, int& have) {
  const int len = a.lens[b * a.lens_step], to = a.first[b * a.first_step];
  have = pages_of(len < 0 ? 0 : len, a.page);
  const int want = pages_of(to < 0 ? 0 : to, a.page);
  if (to <= len) return 0;
  return have > a.width || want > a.width ? -1 : want - have;
}

// Sequence b grows to first[b] tokens: rows in their order take the lowest free pages. A row is
// served if the pages that it and the rows before it need are there. `work`: the ends of the rows'
// shares [rows], then the pages found [most]. 256 rows: a chain of loads and barriers, 5.2 us where
// the first 8192 counts have pages enough, whether a tenth of them are free or all; each further
// 8192 counts are a round of 0.8 us (65536 pages of which the last tenth is free: 10.7 us).
extern "C" __global__ __launch_bounds__(WG) void ek_take_pages(Params a) {
  __shared__ u32 s_wave[WG / 64];
  __shared__ int32_t s_ends[SMALL];
  int32_t* ends = a.n <= SMALL ? s_ends : a.work;
  int32_t* found = a.work + a.n;
  const Counts counts = counts_at(a, threadIdx.x * EACH);
  int64_t sum = 0;
  for (int b0 = 0; b0 < a.n; b0 += WG) {
    const int b = b0 + threadIdx.x;
    int have = 0, need = b < a.n ? need_of(a, b, have) : 0;
    // a share or an end beyond all pages is never served, however large it is
    need = need < 0 ? 0 : need > a.pages ? a.pages + 1 : need;
    int64_t total;
    const int64_t end = sum + scan_group(need, &total, s_wave) + need;
    if (b < a.n) ends[b] = end > a.pages ? a.pages + 1 : (int)end;
    sum += total;
  }
  const int want = sum > a.pages ? a.pages : (int)sum;
  __syncthreads();
  const int got = find_free(a, want, found, s_wave, counts);
  // the pages to their rows: the first row whose share ends behind a page's rank
  for (int r = threadIdx.x; r < got; r += WG) {
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    if (ends[lo] > got) continue;                  // not all of its pages are there
    int have;
    const int need = need_of(a, lo, have), page = found[r];
    a.table[lo * a.table_row + have + r - (ends[lo] - need)] = page;
    a.refs[page] = 1;
  }
  __syncthreads();                                 // lengths are still read above
  for (int b = threadIdx.x; b < a.n; b += WG) {
    int have;
    const int need = need_of(a, b, have);
    const bool ok = need == 0 || (need > 0 && ends[b] <= got);
    const int len = a.lens[b * a.lens_step], to = a.first[b * a.first_step];
    a.served[b] = ok;
    if (ok && to > len) a.lens[b * a.lens_step] = to;
  }
}

// Which forks are served, and the fresh pages of those whose source ends inside a page. `work`:
// [rows] the first fork to each row, [rows] whether the row is a source, [n] ends of the shares,
// [n] a fork's fresh page (-1: none), [n] pages found. 192 forks in 256 rows: 5.2 us.
struct Fork { bool ok; int need; };

EK_INLINE Fork fork_of(const Params& a, int i, const int32_t* owner, const int32_t* source) {
  const int from = a.first[i * a.first_step], to = a.second[i * a.second_step];
  if ((u32)from >= (u32)a.rows || (u32)to >= (u32)a.rows) return {false, 0};
  const int len = a.lens[from * a.lens_step], held = a.lens[to * a.lens_step];
  const auto mark = [](const int32_t* p) {         // past this CU's cache: others' atomics wrote it
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  const bool ok = mark(&owner[to]) == i && mark(&source[to]) == 0 && held <= 0 &&
                  pages_of(len < 0 ? 0 : len, a.page) <= a.width;
  if (!ok || len <= 0 || len % a.page == 0) return {ok, 0};
  return {ok, (u32)a.table[from * a.table_row + len / a.page] < (u32)a.pages};
}

extern "C" __global__ __launch_bounds__(WG) void ek_fork_plan(Params a) {
  __shared__ u32 s_wave[WG / 64];
  __shared__ int32_t s_marks[2 * SMALL];
  int32_t* owner = a.rows <= SMALL ? s_marks : a.work;
  int32_t *source = owner + a.rows, *ends = a.work + 2 * a.rows, *fresh = ends + a.n;
  int32_t* found = fresh + a.n;
  const Counts counts = counts_at(a, threadIdx.x * EACH);
  for (int r = threadIdx.x; r < a.rows; r += WG) owner[r] = 0x7FFFFFFF, source[r] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < a.n; i += WG) {
    const int from = a.first[i * a.first_step], to = a.second[i * a.second_step];
    if ((u32)to < (u32)a.rows) atomicMin(&owner[to], i);
    if ((u32)from < (u32)a.rows) atomicOr(&source[from], 1);
  }
  __syncthreads();
  Fork mine = {false, 0};                          // this thread's first, and where its share ends
  int mine_end = 0, sum = 0;
  for (int i0 = 0; i0 < a.n; i0 += WG) {
    const int i = i0 + threadIdx.x;
    const Fork f = i < a.n ? fork_of(a, i, owner, source) : Fork{false, 0};
    int64_t total;
    const int end = sum + (int)scan_group(f.need, &total, s_wave) + f.need;
    if (i0 == 0) mine = f, mine_end = end;
    else if (i < a.n) ends[i] = end;
    sum += (int)total;
  }
  __syncthreads();
  const int got = find_free(a, sum, found, s_wave, counts);
  for (int i = threadIdx.x; i < a.n; i += WG) {
    const Fork f = i < WG ? mine : fork_of(a, i, owner, source);
    const int end = i < WG ? mine_end : ends[i];
    const bool ok = f.ok && (f.need == 0 || end <= got);
    const int page = ok && f.need ? found[end - 1] : -1;
    fresh[i] = page;
    if (page >= 0) a.refs[page] = 1;
    a.served[i] = ok;
  }
}

// The served forks: the live part of a page that is not whole goes to the fresh one in every
// cache; the last workgroups of a fork take its row of the table, the counts and the length. A
// count below 0 stays: nothing lowers one here, so its sign is the same whoever added before.
extern "C" __global__ __launch_bounds__(THREADS) void ek_fork_copy(Params a) {
  const int i = blockIdx.x / (u32)a.pieces, piece = blockIdx.x - i * a.pieces;
  if (!a.served[i]) return;
  const int from = a.first[i * a.first_step], to = a.second[i * a.second_step];
  const int len = a.lens[from * a.lens_step], fresh = a.work[2 * a.rows + a.n + i];
  const int whole = len < 0 ? 0 : len / a.page;
  const int32_t* old = a.table + from * a.table_row;
  if ((int)blockIdx.y < a.caches_used) {
    if (fresh >= 0) copy_piece<FORK>(a, a.caches[blockIdx.y], old[whole], fresh,
                                     len - whole * a.page, piece);
    return;
  }
  int32_t* row = a.table + to * a.table_row;
  const int held = pages_of(len < 0 ? 0 : len, a.page);
  for (int p = piece * THREADS + threadIdx.x; p < held; p += a.pieces * THREADS) {
    const int id = old[p];
    const bool own = p == whole && fresh >= 0;
    row[p] = own ? fresh : id;
    if (!own && (u32)id < (u32)a.pages && a.refs[id] >= 0) atomicAdd(&a.refs[id], 1);
  }
  if (piece == 0 && threadIdx.x == 0) a.lens[to * a.lens_step] = len < 0 ? 0 : len;
}
