// Paged key-value cache: page allocation, writes of new tokens, fork, free and compaction.
//
// The state is a table of page ids per sequence, a reference count per page and one free bit per page. The free bit
// is redundant (refs == 0) and kept because finding free pages then reads 1/32 of the words: the lowest free pages of
// a call are ranked by one popcount scan in one block. Choosing the lowest free pages (no stack) makes the outcome
// independent of the order in which atomics run, and keeps the live pages near the front of the pool.
//
// Each changing call is a plan (one block: checks, ranks, page choice; all or nothing) and, where pages are copied, a
// second launch that moves the data with all SMs: 16-byte loads and stores over (page, piece) tasks.
#include "common.cuh"
#include "registry.h"

namespace {

constexpr int PLAN_T = 1024;
constexpr int BITMAP = 65536 / 8;         // shared memory for one bit per sequence, at most
constexpr int MAX_PAGES = 1 << 20;   // PLAN_T sequences that each lack them all still sum within an int32

struct Cache {
  uint8_t* pool;
  int64_t page_bytes;
  int32_t pages, page_size, seqs, max_pages;
  int32_t *lengths, *refs;
  uint32_t* words;
  int32_t *table, *err, *scratch;
};

// scratch: [0] copies, [1] rows to share, [2] live pages of a compaction, [3] blocks of a fork's plan that are through; then
// src / dst of the copies, a page list, two arrays of `seqs` (per-sequence counts), one of pages + 2 seqs (counts of 32 table
// entries each), and a bit per sequence that its last extend was refused. From call to call only these bits are kept, and [3] is 0.
struct Scratch {
  int32_t *head, *src, *dst, *list, *num, *num2, *part;
  uint32_t* refused;
};
__host__ __device__ inline int64_t scratch_ints(int64_t pages, int64_t seqs) {
  return 8 + 4 * pages + 4 * seqs + (seqs + 31) / 32;
}
SSB_DEV Scratch scratch_of(const Cache& c) {
  Scratch s;
  s.head = c.scratch;
  s.src = s.head + 8;
  s.dst = s.src + c.pages;
  s.list = s.dst + c.pages;
  s.num = s.list + c.pages;
  s.num2 = s.num + c.seqs;
  s.part = s.num2 + c.seqs;
  s.refused = (uint32_t*)(s.part + c.pages + 2 * c.seqs);
  return s;
}

// Exclusive sum of v over the block's threads; *total gets the block's sum. `part` is 33 ints of shared memory.
SSB_DEV int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();                       // `part` may still be read by an earlier call
  if (lane == 31) part[w] = inc;
  __syncthreads();
  if (w == 0) {
    int p = part[lane];
    int q = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      int u = __shfl_up_sync(0xFFFFFFFFu, q, o);
      if (lane >= o) q += u;
    }
    part[lane] = q - p;
    if (lane == 31) part[32] = q;
  }
  __syncthreads();
  *total = part[32];
  return part[w] + inc - v;
}

// The words of a thread: contiguous, so that ranks follow page order.
struct WordSpan {
  int w0, w1;
};
SSB_DEV WordSpan word_span(int pages) {
  const int n = (pages + 31) >> 5, per = (n + PLAN_T - 1) / PLAN_T;
  WordSpan s;
  s.w0 = min((int)threadIdx.x * per, n);
  s.w1 = min(s.w0 + per, n);
  return s;
}

// Takes the `need` lowest free pages: list[0 .. need) in ascending order, their refs 1 and free bits cleared. Returns
// false (and takes nothing) when there are fewer. Called by the whole block; ends with a barrier.
SSB_DEV bool take_pages(const Cache& c, int need, int32_t* list, int* part) {
  const WordSpan ws = word_span(c.pages);
  int have = 0;
  for (int w = ws.w0; w < ws.w1; ++w) have += __popc(c.words[w]);
  int total;
  int r = block_scan(have, part, &total);
  if (total < need) return false;
  for (int w = ws.w0; w < ws.w1 && r < need; ++w) {
    uint32_t bits = c.words[w], keep = bits;
    while (bits && r < need) {
      const int b = __ffs(bits) - 1;
      bits &= bits - 1;
      keep &= ~(1u << b);
      const int p = w * 32 + b;
      list[r++] = p;
      c.refs[p] = 1;
    }
    c.words[w] = keep;
  }
  __syncthreads();
  return true;
}

SSB_DEV bool seen_before(uint32_t* bitmap, int s) {
  const uint32_t bit = 1u << (s & 31);
  return atomicOr(&bitmap[s >> 5], bit) & bit;
}

// Allocation: the table entries that the new tokens fall into, in runs of 32 (a warp each), are counted where they lack a
// page, the counts are scanned, and the lowest free pages dealt out in that order.
// A refused call leaves lengths as they are, so rows written next would land on the newest tokens that are there, in pages
// that nobody shares. Hence the sequences that it was to give room are marked until an extend has made room for them, and
// k_write drops the rows of marked ones: a step that extends and writes (in a captured graph, say) need not look in between.
__global__ void __launch_bounds__(PLAN_T) k_extend(Cache c, const int32_t* __restrict__ ids,
                                                   const int32_t* __restrict__ counts, int n) {
  extern __shared__ uint32_t bitmap[];
  __shared__ int part[33];
  __shared__ int bad;
  const Scratch sc = scratch_of(c);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < (c.seqs + 31) >> 5; i += PLAN_T) bitmap[i] = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  auto refuse = [&](int why) {
    for (int i = threadIdx.x; i < n; i += PLAN_T) {
      const int s = ids[i];
      if (s >= 0 && s < c.seqs && counts[i] != 0) atomicOr(&sc.refused[s >> 5], 1u << (s & 31));
    }
    if (threadIdx.x == 0) set_err(c.err, why);
  };
  // entries of each sequence, its first run, and where in the table they begin; in shared memory where the call is small
  __shared__ int s_num[PLAN_T], s_run[PLAN_T];
  __shared__ int64_t s_at[PLAN_T];
  int32_t *num = n <= PLAN_T ? s_num : sc.num, *run = n <= PLAN_T ? s_run : sc.num2;
  int runs = 0;
  // Every entry is a page of its own at the end, so more entries than pages cannot be had; then runs > pages / 32 + n.
  const int most = c.pages / 32 + n;
  for (int i0 = 0; i0 < n && runs <= most; i0 += PLAN_T) {
    const int i = i0 + threadIdx.x;
    int wrong = 0, e = 0;
    if (i < n) {
      const int s = ids[i], add = counts[i];
      if (s < 0 || s >= c.seqs || add < 0 || seen_before(bitmap, s)) {
        wrong = SSB_ERR_SEQUENCE;
      } else {
        const int64_t len = c.lengths[s], now = len + add;
        if (len < 0) wrong = SSB_ERR_SEQUENCE;
        else if (now > (int64_t)c.max_pages * c.page_size) wrong = SSB_ERR_NO_PAGES;
        else if (add > 0) e = (int)((now + c.page_size - 1) / c.page_size - len / c.page_size);
        if (n <= PLAN_T) s_at[i] = (int64_t)s * c.max_pages + len / c.page_size;
      }
      if (wrong) atomicOr(&bad, wrong);
      e = min(e, c.pages + 32);
    }
    int total;
    const int ex = block_scan((e + 31) >> 5, part, &total);
    if (i < n) {
      num[i] = e;
      run[i] = runs + ex;
    }
    runs += total;
  }
  if (runs > most && threadIdx.x == 0) atomicOr(&bad, SSB_ERR_NO_PAGES);
  __syncthreads();
  if (bad) return refuse(bad);
  // run r: its sequence's table entry for this lane (nullptr past the last)
  auto entry_of = [&](int r) -> int32_t* {
    int lo = 0, hi = n;                                // the last i with run[i] <= r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (run[mid] <= r) lo = mid;
      else hi = mid;
    }
    const int k = (r - run[lo]) * 32 + lane;
    if (k >= num[lo]) return nullptr;
    if (n <= PLAN_T) return c.table + s_at[lo] + k;
    const int s = ids[lo];
    return c.table + (int64_t)s * c.max_pages + c.lengths[s] / c.page_size + k;
  };
  for (int r = warp; r < runs; r += PLAN_T / 32) {
    const int32_t* e = entry_of(r);
    const int p = e ? *e : 0;
    const int wrong = !e || p < 0 ? 0 : p >= c.pages ? SSB_ERR_PAGE_RANGE : c.refs[p] > 1 ? SSB_ERR_SHARED_PAGE : 0;
    const uint32_t lacks = __ballot_sync(0xFFFFFFFFu, e && p < 0);
    if (wrong) atomicOr(&bad, wrong);
    if (lane == 0) sc.part[r] = __popc(lacks);
  }
  __syncthreads();
  int need = 0;
  for (int r0 = 0; r0 < runs; r0 += PLAN_T) {
    const int r = r0 + threadIdx.x;
    int total;
    const int ex = block_scan(r < runs ? sc.part[r] : 0, part, &total);
    if (r < runs) sc.part[r] = need + ex;
    need += total;
  }
  __syncthreads();
  if (bad) return refuse(bad);
  if (!take_pages(c, need, sc.list, part)) return refuse(SSB_ERR_NO_PAGES);
  for (int r = warp; r < runs; r += PLAN_T / 32) {
    int32_t* e = entry_of(r);
    const bool lacks = e && *e < 0;
    const uint32_t m = __ballot_sync(0xFFFFFFFFu, lacks);
    if (lacks) *e = sc.list[sc.part[r] + __popc(m & lanemask_lt())];
  }
  __syncthreads();                                     // entries are found through the old lengths
  for (int i = threadIdx.x; i < n; i += PLAN_T) {
    const int s = ids[i];
    c.lengths[s] += counts[i];
    if (sc.refused[s >> 5] >> (s & 31) & 1) atomicAnd(&sc.refused[s >> 5], ~(1u << (s & 31)));
  }
}

// Look t at the table row of a fork's child, by eight threads: whether one of the LOOK entries is among those that the child
// gets and holds a page already, whose name would be lost. (A sequence that was rolled back to length 0 can hold pages anywhere
// in its row, since a window may have given back the first ones.) The plan's grid grows with these looks, so that a long table
// does not wait for one SM: a fork of 1 child of 600 tokens takes 7.2 us on the device (6.6 without the looks), of 112 children
// 9.0 (7.9), of 112 children of 131,072 tokens 17.9 (14.6); with all looks in one block the last took 82.
constexpr int LOOK = 64, LOOKS = PLAN_T / 8;
SSB_DEV bool holds_any(const Cache& c, const int32_t* parents, const int32_t* children, int64_t t) {
  const int per = (c.max_pages + LOOK - 1) / LOOK, i = (int)(t / per), j0 = (int)(t - (int64_t)i * per) * LOOK;
  const int p = parents[i], k = children[i];
  if (p < 0 || p >= c.seqs || k < 0 || k >= c.seqs) return false;     // refused by the plan itself
  const int64_t gets = ((int64_t)c.lengths[p] + c.page_size - 1) / c.page_size;
  const int end = (int)(gets < c.max_pages ? gets : c.max_pages);
  const int32_t* row = c.table + (int64_t)k * c.max_pages;
  bool holds = false;
#pragma unroll
  for (int u = 0; u < LOOK / 8; ++u) {
    const int j = j0 + u * 8 + (threadIdx.x & 7);
    holds |= j < end && row[j] >= 0;
  }
  return holds;
}

__global__ void __launch_bounds__(PLAN_T) k_fork_plan(Cache c, const int32_t* __restrict__ parents,
                                                      const int32_t* __restrict__ children, int n) {
  pdl_trigger();
  extern __shared__ uint32_t bitmap[];
  __shared__ int part[33];
  __shared__ int bad;
  const Scratch sc = scratch_of(c);
  for (int i = threadIdx.x; i < (c.seqs + 31) >> 5; i += PLAN_T) bitmap[i] = 0;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  const int64_t looks = (int64_t)n * ((c.max_pages + LOOK - 1) / LOOK);
  for (int64_t t = (int64_t)blockIdx.x * LOOKS + threadIdx.x / 8; t < looks; t += (int64_t)gridDim.x * LOOKS)
    if (holds_any(c, parents, children, t)) bad = SSB_ERR_SEQUENCE;
  __syncthreads();
  if (gridDim.x > 1) {                                   // the block that ends last has what all of them found, and plans
    __shared__ int before;
    if (threadIdx.x == 0) {
      __threadfence();
      before = atomicAdd(&sc.head[3], bad ? 0x10001 : 1);
    }
    __syncthreads();
    if ((before & 0xFFFF) != (int)gridDim.x - 1) return;
    if (threadIdx.x == 0) {
      if (before >> 16) bad = SSB_ERR_SEQUENCE;
      sc.head[3] = 0;
    }
    __syncthreads();
  }
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += PLAN_T) {
    const int i = i0 + threadIdx.x;
    int wrong = 0, need = 0;
    if (i < n) {
      const int p = parents[i], k = children[i];
      if (p < 0 || p >= c.seqs || k < 0 || k >= c.seqs || seen_before(bitmap, k)) {
        wrong = SSB_ERR_SEQUENCE;
      } else {
        const int64_t len = c.lengths[p];
        if (c.lengths[k] != 0 || c.table[(int64_t)k * c.max_pages] >= 0) wrong = SSB_ERR_SEQUENCE;
        if (len < 0 || len > (int64_t)c.max_pages * c.page_size) wrong |= SSB_ERR_SEQUENCE;
        else if (len % c.page_size) {
          const int tail = c.table[(int64_t)p * c.max_pages + len / c.page_size];
          if (tail >= c.pages) wrong |= SSB_ERR_PAGE_RANGE;
          need = tail >= 0;
        }
      }
      if (wrong) atomicOr(&bad, wrong);
    }
    int total;
    const int ex = block_scan(need, part, &total);
    if (i < n) sc.num[i] = need ? base + ex : -1;
    base += total;
  }
  __syncthreads();
  bool ok = bad == 0;
  if (ok) {
    ok = take_pages(c, base, sc.list, part);
    if (!ok && threadIdx.x == 0) set_err(c.err, SSB_ERR_NO_PAGES);
  } else if (threadIdx.x == 0) {
    set_err(c.err, bad);
  }
  if (ok)
    for (int i = threadIdx.x; i < n; i += PLAN_T) {
      const int p = parents[i], r = sc.num[i];
      const int64_t len = c.lengths[p];
      sc.num2[i] = (int)(len / c.page_size);              // full pages
      if (r >= 0) {
        sc.src[r] = c.table[(int64_t)p * c.max_pages + len / c.page_size];
        sc.dst[r] = sc.list[r];
        c.table[(int64_t)children[i] * c.max_pages + len / c.page_size] = sc.list[r];
      }
      sc.num[i] = (int)len;                                // from here on: the child's length
    }
  if (threadIdx.x == 0) {
    sc.head[0] = ok ? base : 0;
    sc.head[1] = ok ? n : 0;
  }
}

// Copies pages src[i] -> dst[i], i < head[0], in pieces of PIECE bytes spread over the grid.
constexpr int COPY_T = 256;
constexpr int64_t PIECE = COPY_T * 16 * 8;
SSB_DEV void copy_pages(const Cache& c, const Scratch& sc) {
  const int64_t per = (c.page_bytes + PIECE - 1) / PIECE, total = per * sc.head[0];
  for (int64_t t = blockIdx.x; t < total; t += gridDim.x) {
    const int64_t i = t / per, off = (t - i * per) * PIECE + threadIdx.x * 16;
    const uint8_t* s = c.pool + (int64_t)sc.src[i] * c.page_bytes + off;
    uint8_t* d = c.pool + (int64_t)sc.dst[i] * c.page_bytes + off;
    const int64_t left = c.page_bytes - off;
    uint4 v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u * COPY_T * 16 < left) v[u] = *(const uint4*)(s + u * COPY_T * 16);
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (u * COPY_T * 16 < left) *(uint4*)(d + u * COPY_T * 16) = v[u];
  }
}

__global__ void __launch_bounds__(COPY_T) k_fork_apply(Cache c, const int32_t* __restrict__ parents,
                                                       const int32_t* __restrict__ children) {
  pdl_wait();
  const Scratch sc = scratch_of(c);
  const int n = sc.head[1];
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    const int p = parents[i], k = children[i], full = sc.num2[i];   // a parent may be another pair's (empty) child,
    for (int j = threadIdx.x; j < full; j += COPY_T) {
      const int page = c.table[(int64_t)p * c.max_pages + j];
      c.table[(int64_t)k * c.max_pages + j] = page;
      if (page >= 0 && page < c.pages) atomicAdd(&c.refs[page], 1);
    }
    if (threadIdx.x == 0) c.lengths[k] = sc.num[i];                 // so its length was read by the plan
  }
  copy_pages(c, sc);
}

// One block per (sequence, 1024 entries). atomicExch hands each entry to one taker, so repeated ids are harmless.
__global__ void __launch_bounds__(256) k_free(Cache c, const int32_t* __restrict__ ids,
                                              const int32_t* __restrict__ first, const int32_t* __restrict__ last) {
  const int s = ids[blockIdx.x];
  if (s < 0 || s >= c.seqs) {
    if (threadIdx.x == 0) set_err(c.err, SSB_ERR_SEQUENCE);
    return;
  }
  const int a = first ? max(first[blockIdx.x], 0) : 0, b = first ? min(last[blockIdx.x], c.max_pages) : c.max_pages;
  const int j0 = blockIdx.y * 1024, j1 = min(j0 + 1024, b);
  for (int j = max(j0, a) + threadIdx.x; j < j1; j += 256) {
    int32_t* e = c.table + (int64_t)s * c.max_pages + j;
    if (*e < 0) continue;
    const int p = atomicExch(e, -1);
    if (p < 0) continue;
    if (p >= c.pages) {
      set_err(c.err, SSB_ERR_PAGE_RANGE);
      continue;
    }
    if (atomicSub(&c.refs[p], 1) == 1) atomicOr(&c.words[p >> 5], 1u << (p & 31));
  }
  if (!first && blockIdx.y == 0 && threadIdx.x == 0) c.lengths[s] = 0;
}

__global__ void __launch_bounds__(PLAN_T) k_compact_plan(Cache c) {
  pdl_trigger();
  __shared__ int part[33];
  const Scratch sc = scratch_of(c);
  const WordSpan ws = word_span(c.pages);
  int have = 0;
  for (int w = ws.w0; w < ws.w1; ++w) have += __popc(c.words[w]);
  int free_all;
  block_scan(have, part, &free_all);
  const int live = c.pages - free_all;
  // bits of word w at pages below `live`, and at pages in [live, pages)
  auto below = [&](int w) {
    const int d = live - w * 32;
    return d >= 32 ? 0xFFFFFFFFu : d <= 0 ? 0u : (1u << d) - 1u;
  };
  auto valid = [&](int w) {
    const int d = c.pages - w * 32;
    return d >= 32 ? 0xFFFFFFFFu : (1u << d) - 1u;
  };
  int holes = 0, movers = 0;
  for (int w = ws.w0; w < ws.w1; ++w) {
    const uint32_t f = c.words[w], lo = below(w);
    holes += __popc(f & lo);
    movers += __popc(~f & ~lo & valid(w));
  }
  int n_holes, n_movers;
  int rh = block_scan(holes, part, &n_holes);
  int rm = block_scan(movers, part, &n_movers);
  for (int w = ws.w0; w < ws.w1; ++w) {
    const uint32_t f = c.words[w], lo = below(w);
    for (uint32_t b = f & lo; b; b &= b - 1) sc.dst[rh++] = w * 32 + __ffs(b) - 1;
    for (uint32_t b = ~f & ~lo & valid(w); b; b &= b - 1) sc.src[rm++] = w * 32 + __ffs(b) - 1;
    c.words[w] = ~lo & valid(w);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n_movers; i += PLAN_T) {
    const int s = sc.src[i], d = sc.dst[i];
    sc.list[s - live] = d;
    c.refs[d] = c.refs[s];
    c.refs[s] = 0;
  }
  if (threadIdx.x == 0) {
    sc.head[0] = n_movers;
    sc.head[2] = live;
  }
}

__global__ void __launch_bounds__(COPY_T) k_compact_apply(Cache c) {
  pdl_wait();
  const Scratch sc = scratch_of(c);
  const int live = sc.head[2];
  if (sc.head[0] == 0) return;
  const int64_t entries = (int64_t)c.seqs * c.max_pages;
  for (int64_t i = (int64_t)blockIdx.x * COPY_T + threadIdx.x; i < entries; i += (int64_t)gridDim.x * COPY_T) {
    const int p = c.table[i];
    if (p >= live && p < c.pages) c.table[i] = sc.list[p - live];
  }
  copy_pages(c, sc);
}

// One warp per new token: its sequence by a search of starts, its slot through the table, then 16-byte copies of its key and
// value heads. Bound by memory (read once, written once). The first 8 pieces a lane are loaded before the look-ups, a chain
// of five dependent loads that otherwise stands before every byte (four prompts of up to 16,384 tokens, 8 heads of 128, with
// their allocation: 90 us before, 70 now, 56 of them the bytes at the copy's rate).
struct WriteArgs {
  const uint16_t *k, *v;
  int64_t rows, k_row, k_head, v_row, v_head;
  int32_t kv_heads, dim;
  const int32_t *starts, *ids;
  int32_t n;
  uint16_t *kl, *vl;
  int64_t page_stride, head_stride, token_stride;
  uint32_t per_mul, per_shift;   // i / (dim / 8)
};
constexpr int BATCH = 8;
__global__ void __launch_bounds__(256) k_write(Cache c, WriteArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t r = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= a.rows) return;
  const int per = a.dim >> 3, chunks = a.kv_heads * per, total = 2 * chunks;
  const uint16_t *kr = a.k + r * a.k_row, *vr = a.v + r * a.v_row;
  auto head_of = [&](int q) { return (int)((__umulhi((uint32_t)q, a.per_mul) + (uint32_t)q) >> a.per_shift); };
  uint4 x[BATCH];
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * 32, q = i < chunks ? i : i - chunks, h = head_of(q), e = (q - h * per) * 8;
      if (i < total) x[u] = __ldcs((const uint4*)(i < chunks ? kr + h * a.k_head + e : vr + h * a.v_head + e));
    }
  };
  load(lane);
  int lo = 0, hi = a.n;                                  // the last b with starts[b] <= r
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.starts[mid] <= r) lo = mid;
    else hi = mid;
  }
  const int64_t b0 = a.starts[lo], b1 = a.starts[lo + 1];
  if (r < b0 || r >= b1) return;                         // rows outside every sequence
  const int s = a.ids ? a.ids[lo] : lo;
  if (s < 0 || s >= c.seqs) {
    if (lane == 0) set_err(c.err, SSB_ERR_SEQUENCE);
    return;
  }
  if (scratch_of(c).refused[s >> 5] >> (s & 31) & 1) {   // no room was made for the row
    if (lane == 0) set_err(c.err, SSB_ERR_NO_ROOM);
    return;
  }
  const int64_t pos = c.lengths[s] - (b1 - b0) + (r - b0);
  if (pos < 0 || pos >= (int64_t)c.max_pages * c.page_size) {
    if (lane == 0) set_err(c.err, SSB_ERR_SEQUENCE);
    return;
  }
  const int j = (int)pos / c.page_size, slot = (int)pos - j * c.page_size;
  const int page = c.table[(int64_t)s * c.max_pages + j];
  if (page < 0 || page >= c.pages || c.refs[page] != 1) {
    if (lane == 0) set_err(c.err, page < 0 || page >= c.pages ? SSB_ERR_PAGE_RANGE : SSB_ERR_SHARED_PAGE);
    return;
  }
  const int64_t to = (int64_t)page * a.page_stride + slot * a.token_stride;
  for (int i0 = lane; i0 < total; i0 += 32 * BATCH) {
    if (i0 != lane) load(i0);
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int i = i0 + u * 32, q = i < chunks ? i : i - chunks, h = head_of(q), e = (q - h * per) * 8;
      if (i < total) *(uint4*)((i < chunks ? a.kl : a.vl) + to + h * a.head_stride + e) = x[u];
    }
  }
}

int cache_of(const ssb_kv_cache* c, Cache* o) {
  SSB_CHECK_ARG(c && c->pool && c->lengths && c->refs && c->free_words && c->table && c->scratch);
  SSB_CHECK_ARG(c->pages > 0 && c->pages <= MAX_PAGES && c->seqs > 0 && c->seqs <= 65536 && c->max_pages > 0 &&
                c->page_size > 0 && (int64_t)c->max_pages * c->page_size <= 0x7FFFFFFFll);
  SSB_CHECK_ARG(c->page_bytes > 0 && c->page_bytes % 16 == 0 && ((uintptr_t)c->pool & 15) == 0);
  *o = Cache{(uint8_t*)c->pool, c->page_bytes, c->pages, c->page_size, c->seqs, c->max_pages,
             c->lengths, c->refs, c->free_words, c->table, c->err, c->scratch};
  return SSB_OK;
}

}  // namespace

extern "C" int ssb_kv_scratch_ints(int32_t pages, int32_t seqs) {
  SSB_CHECK_ARG(pages > 0 && pages <= MAX_PAGES && seqs > 0 && seqs <= 65536);
  return (int)scratch_ints(pages, seqs);
}

extern "C" int ssb_kv_extend(const ssb_kv_cache* cc, const int32_t* ids, const int32_t* counts, int32_t n,
                             void* stream) {
  Cache c;
  if (int rc = cache_of(cc, &c)) return rc;
  SSB_CHECK_ARG(n >= 0 && n <= c.seqs);
  if (n == 0) return SSB_OK;
  SSB_CHECK_ARG(ids && counts);
  const size_t smem = (size_t)((c.seqs + 31) / 32) * 4;
  static std::atomic<uint64_t> done{0};
  if (int rc = ssb_setup_kernel(done, "kv_extend", k_extend, BITMAP)) return rc;
  return ssb_launch(k_extend, dim3(1), dim3(PLAN_T), smem, (cudaStream_t)stream, false, c, ids, counts, n);
}

extern "C" int ssb_kv_fork(const ssb_kv_cache* cc, const int32_t* parents, const int32_t* children, int32_t n,
                           void* stream) {
  Cache c;
  if (int rc = cache_of(cc, &c)) return rc;
  SSB_CHECK_ARG(n >= 0 && n <= c.seqs);
  if (n == 0) return SSB_OK;
  SSB_CHECK_ARG(parents && children);
  const size_t smem = (size_t)((c.seqs + 31) / 32) * 4;
  static std::atomic<uint64_t> done{0};
  if (int rc = ssb_setup_kernel(done, "kv_fork", k_fork_plan, BITMAP)) return rc;
  const int64_t looks = (int64_t)n * ((c.max_pages + LOOK - 1) / LOOK), sms = ssb_sm_count();
  const unsigned plans = (unsigned)(looks < sms * LOOKS ? (looks + LOOKS - 1) / LOOKS : sms);
  int rc = ssb_launch(k_fork_plan, dim3(plans), dim3(PLAN_T), smem, (cudaStream_t)stream, false, c, parents, children, n);
  if (rc) return rc;
  const int64_t tasks = (int64_t)n * ((c.page_bytes + PIECE - 1) / PIECE), most = (int64_t)ssb_sm_count() * 8;
  return ssb_launch(k_fork_apply, dim3((unsigned)(tasks < most ? tasks : most)), dim3(COPY_T), 0, (cudaStream_t)stream,
                    true, c, parents, children);
}

extern "C" int ssb_kv_free(const ssb_kv_cache* cc, const int32_t* ids, const int32_t* first, const int32_t* last,
                           int32_t n, void* stream) {
  Cache c;
  if (int rc = cache_of(cc, &c)) return rc;
  SSB_CHECK_ARG(n >= 0 && n <= 65536 && (first == nullptr) == (last == nullptr));
  if (n == 0) return SSB_OK;
  SSB_CHECK_ARG(ids);
  SSB_CHECK_ARG(c.max_pages <= 65535 * 1024);
  static std::atomic<uint64_t> done{0};
  if (int rc = ssb_setup_kernel(done, "kv_free", k_free, 0)) return rc;
  return ssb_launch(k_free, dim3((unsigned)n, (unsigned)((c.max_pages + 1023) / 1024)), dim3(256), 0,
                    (cudaStream_t)stream, false, c, ids, first, last);
}

extern "C" int ssb_kv_compact(const ssb_kv_cache* cc, void* stream) {
  Cache c;
  if (int rc = cache_of(cc, &c)) return rc;
  static std::atomic<uint64_t> done{0};
  if (int rc = ssb_setup_kernel(done, "kv_compact", k_compact_plan, 0)) return rc;
  int rc = ssb_launch(k_compact_plan, dim3(1), dim3(PLAN_T), 0, (cudaStream_t)stream, false, c);
  if (rc) return rc;
  return ssb_launch(k_compact_apply, dim3((unsigned)ssb_sm_count() * 8), dim3(COPY_T), 0, (cudaStream_t)stream, true, c);
}

extern "C" int ssb_kv_write(const ssb_kv_cache* cc, const ssb_kv_rows* w, void* stream) {
  Cache c;
  if (int rc = cache_of(cc, &c)) return rc;
  SSB_CHECK_ARG(w && w->rows >= 0 && w->rows < (1ll << 31) && w->n >= 0 && w->kv_heads > 0 && w->dim > 0);
  if (w->dim % 8) return SSB_EUNSUPPORTED;
  if (w->rows == 0 || w->n == 0) return SSB_OK;
  SSB_CHECK_ARG(w->k && w->v && w->starts && w->k_layer && w->v_layer);
  const int64_t bits = w->k_row_stride | w->k_head_stride | w->v_row_stride | w->v_head_stride | w->page_stride |
                       w->head_stride | w->token_stride;
  SSB_CHECK_ARG(bits % 8 == 0);
  SSB_CHECK_ARG((((uintptr_t)w->k | (uintptr_t)w->v | (uintptr_t)w->k_layer | (uintptr_t)w->v_layer) & 15) == 0);
  SSB_CHECK_ARG((int64_t)w->kv_heads * w->dim < (1ll << 30));
  WriteArgs a{w->k, w->v, w->rows, w->k_row_stride, w->k_head_stride, w->v_row_stride, w->v_head_stride, w->kv_heads, w->dim,
              w->starts, w->ids, w->n, w->k_layer, w->v_layer, w->page_stride, w->head_stride, w->token_stride, 0, 0};
  while ((8ll << a.per_shift) < w->dim) ++a.per_shift;    // round-up reciprocal, for i < 2^31
  a.per_mul = (uint32_t)((1ll << 32) * ((1ll << a.per_shift) - w->dim / 8) / (w->dim / 8) + 1);
  static std::atomic<uint64_t> done{0};
  if (int rc = ssb_setup_kernel(done, "kv_write", k_write, 0)) return rc;
  return ssb_launch(k_write, dim3((unsigned)((w->rows + 7) / 8)), dim3(256), 0, (cudaStream_t)stream, false, c, a);
}
