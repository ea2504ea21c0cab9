// Attention over the paged key-value cache for prompts: causal, ragged, with a sliding window and sinks.
//
// The rows of one key head are (query token, head of its group) pairs, flattened; an item is MB = 128 NT of them
// against the tokens they can see, in tiles of T tokens. Per tile, on the tensor cores (tcgen05, fp32 in TMEM):
// S = Q K^T from shared memory, and O += P V with P read from TMEM, where the softmax has put it.
// What bounds it: the two products are 4 T MB D operations and the softmax T MB exponentials per tile; at head size
// 128 the tensor cores and the 16 exponentials per clock of an SM need the same time, so both have to run all the time.
// Hence two row tiles of 128 (NT = 2; one at head size 256, whose accumulator fills half of TMEM) and two to four buffers
// of S for each: the S of the next tile is computed under the softmax of this one, so neither waits for the latency of the other
// (about 350 cycles from an instruction's issue to a waiting thread).
//
// The running maximum is only raised when a row's maximum grows by more than STEP (log2 domain; a published form of the online
// softmax): p stays below 2^STEP times what it is for the maximum itself, and rescaling the accumulator in TMEM becomes rare.
// bf16 holds all these weights with 8 bits; for fp16 see below_max, which leaves 11 bits down to 2^-21 of the largest weight
// and an error of 2^-32 of it below. A smaller STEP would leave more and costs time (fp16, 32K tokens, window 4096, 32 / 8
// heads of 128: 2.01 ms at 8, 2.13 at 6, 2.23 at 4, 2.63 at 0; without the shift 1.99).
//
// Warps: NT groups of four for the softmax (one thread per row; TMEM lane = row), four that bring Q, K and V into
// 128-byte-swizzled tiles (TMA boxes where pages allow, else row by row with cp.async; rows that no query sees become zeros) and
// hand out the units, and one per row tile and product that issues its matrix instructions. Nothing orders products of
// different threads, shapes or accumulators but the waits here. S is read into registers once and P takes its place; a
// buffer is free for the next S when the product that read P has ended.
//
// Tiles of 64 tokens: two buffers of S for two row tiles of head size 128 fill TMEM. Instructions of 64 columns cost 48
// cycles for 32 columns' worth of work (operands read from shared memory), so the products of a pair of tiles take 2570
// cycles per 128 tokens instead of 2050; single-buffered tiles of 128, where each S waits for the product before it, took
// 4600 (32K tokens, 32 heads, 8 key heads, window 4096: 2.16 ms against 1.91). At size 256 two chunks of 2,048 tokens after
// 14K and 3K take 0.61 ms: each tile brings 64 KB of K and V for one row tile, 8 TB/s out of L2 through a ring of only five
// slots, and shared memory moves 192 KB for it. Without the exponentials it takes as long, with half of Q K^T left out 0.52
// (10 TB/s); the scores of two tiles in one instruction of 128 columns hold two slots at once: 0.68. These are single bursts at
// full clocks (1.08 and 1.05 PFLOP/s); call after call, under the power cap, the two cases take 2.26 and 0.70 ms (0.92 and 0.90).
//
// Balance: k_prefill_plan lists the items, longest first within a sequence, cut into pieces that shrink with the work left
// (an item of w tiles with R tiles left, itself included, and C blocks: pieces of about max(R / C, total / 16 C)); blocks
// take units from the list by a counter; k_prefill_join sums an item's pieces in order, so the outcome does not depend on who
// took which. Where there are many more items than blocks only those of the last wave or so are cut. With about 64 to 140 items
// all of them are, and the pieces wanted can pass the 4 C slots that there are: then an item near the end of the list stays
// whole, and one block works alone for longest (restated on the CPU: 1,024 tokens after 100,000, 32 heads, 8 key heads, size 128,
// 128 items: 617 pieces wanted, 2,863 tiles in the longest block where an even split has 1,359).
#include "paged_attn.cuh"

#include "affine.cuh"
#include "tc_common.cuh"

namespace attn {
namespace {

template <int D>
struct Cfg {
  static constexpr int NT = D == 256 ? 1 : 2, MB = 128 * NT, T = 64;
  static constexpr int SLOTS = D == 64 ? 16 : D == 128 ? 10 : 5;
  static constexpr int CPR = D / 8, SLOT = T * D * 2, QB = MB * D * 2, CTL = 512;
  static constexpr int SMEM = QB + SLOTS * SLOT + CTL, THREADS = (NT + 2) * 128;
  // TMEM columns: the accumulators, then as many buffers of S / P a row tile as fit
  static constexpr int S_COL = NT * D, NBUF = (512 - S_COL) / (NT * T);
  static_assert(NBUF >= 2 && NT * NBUF <= 6, "TMEM");
};
constexpr int PLAN_T = 1024, LAG = 1;
constexpr int STEP = 8;          // how far (log2) a row's maximum runs ahead of the one that its weights are taken against

struct __align__(16) Unit {
  int b, h, r0, rows;          // sequence, key head, first flat row, rows
  int i0, i1, len, q;          // tiles of the unit, sequence length, query tokens
  int q0, row, slot, pad;      // first query token, table row, piece slot (-1: a whole item)
};
struct __align__(16) Joint {
  int h, r0, rows, q0, slot, pieces, pad0, pad1;
};

// Tiles of K and V lie in shared memory as groups of 8 tokens, in each of them 64 dims after 64 dims, as 8 rows of 128 swizzled
// bytes: [T / 8][D / 64][8][128 B]. So the tokens of a page, with all their dims, are one run of it and come as one box
// (with a box for every 64 dims, 2 KB each at pages of 16 tokens, head size 256 was bound by the number of boxes).
//
// Tensor maps of a call: q [rows, heads, dim] in boxes of 128 flat rows x 64; k and v as [page and head, page / 8, dim / 64, 8, 64]
// in boxes of page_rows tokens x dim.
struct Maps {
  CUtensorMap q, k, v;
};

struct Work {
  int* item0;                  // [n + 1] first item of each sequence
  int* ctl;                    // [0] units taken, [1] units, [2] joints
  Unit* units;
  Joint* joints;
  int max_units, max_slots;
  int page_rows, q_boxes;      // tokens of a K / V box, 0: by cp.async; whether Q comes in boxes
  int page_heads;              // steps of the key head's stride from page to page
};

SSB_DEV int block_scan(int v, int* part, int* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    int u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) part[w] = inc;
  __syncthreads();
  if (w == 0) {
    const int p = part[lane];
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
SSB_DEV long long block_scan_ll(long long v, long long* part, long long* total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    long long u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();
  if (lane == 31) part[w] = inc;
  __syncthreads();
  if (w == 0) {
    const long long p = part[lane];
    long long q = p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      long long u = __shfl_up_sync(0xFFFFFFFFu, q, o);
      if (lane >= o) q += u;
    }
    part[lane] = q - p;
    if (lane == 31) part[32] = q;
  }
  __syncthreads();
  *total = part[32];
  return part[w] + inc - v;
}

struct ItemAt {
  int b, h, r0, rows, tiles, len, q, q0, row;
};
// Item i: sequences in order, key heads inside, row blocks from the last one (the longest) down.
template <int MB, int T>
SSB_DEV ItemAt item_at(const Args& a, const Work& w, int i) {
  int lo = 0, hi = a.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (w.item0[mid] <= i) lo = mid;
    else hi = mid;
  }
  const Seq s = seq_of(a, lo);
  const int flat = s.q * a.group, nb = (flat + MB - 1) / MB, k = i - w.item0[lo];
  ItemAt t;
  t.b = lo;
  t.h = k / nb;
  t.r0 = (nb - 1 - (k - t.h * nb)) * MB;
  t.rows = min(MB, flat - t.r0);
  const int p = s.len - s.q;
  t.tiles = range_of(a, p + t.r0 / a.group, p + (t.r0 + t.rows - 1) / a.group, T).tiles;
  t.len = s.len;
  t.q = s.q;
  t.q0 = (int)s.q0;
  t.row = s.row;
  return t;
}

template <int MB, int T>
__global__ void __launch_bounds__(PLAN_T) k_prefill_plan(Args a, Work w, int blocks) {
  __shared__ int part[33];
  __shared__ long long lpart[33];
  pdl_wait();
  pdl_trigger();
  int items = 0;
  for (int b0 = 0; b0 < a.n; b0 += PLAN_T) {
    const int b = b0 + threadIdx.x;
    int c = 0;
    if (b < a.n) {
      const Seq s = seq_of(a, b);
      if (s.row < 0 && s.q > 0) set_err(a.err, SSB_ERR_SEQUENCE);
      c = a.kv_heads * ((s.q * a.group + MB - 1) / MB);
    }
    int total;
    const int ex = block_scan(c, part, &total);
    if (b < a.n) w.item0[b] = items + ex;
    items += total;
  }
  if (threadIdx.x == 0) w.item0[a.n] = items;
  __syncthreads();
  items = min(items, w.max_units);                      // starts that overlap would list more: never out of bounds
  long long all = 0;
  for (int i = threadIdx.x; i < items; i += PLAN_T) all += item_at<MB, T>(a, w, i).tiles;
  long long sum;
  block_scan_ll(all, lpart, &sum);
  const long long least = max(sum / (16ll * blocks), 2ll);
  long long before = 0;
  int units = 0, slots = 0, joints = 0;
  for (int i0 = 0; i0 < items; i0 += PLAN_T) {
    const int i = i0 + threadIdx.x;
    ItemAt t = {};
    if (i < items) t = item_at<MB, T>(a, w, i);
    long long total;
    const long long ex = block_scan_ll(t.tiles, lpart, &total);
    const long long left = sum - before - ex;
    before += total;
    const long long most = max(left / blocks, least);
    int k = i < items ? (int)((t.tiles + most - 1) / most) : 0;
    int n_s, n_j, n_u;
    const int at = slots + block_scan(k > 1 ? k : 0, part, &n_s);
    const bool cut = k > 1 && at + k <= w.max_slots;
    if (k > 1 && !cut) k = 1;
    const int j = joints + block_scan(cut, part, &n_j), u = units + block_scan(k, part, &n_u);
    if (cut) w.joints[j] = Joint{t.h, t.r0, t.rows, t.q0, at, k, 0, 0};
    for (int x = 0; x < k; ++x)
      w.units[u + x] = Unit{t.b, t.h, t.r0, t.rows, (int)((long long)t.tiles * x / k), (int)((long long)t.tiles * (x + 1) / k),
                            t.len, t.q, t.q0, t.row, cut ? at + x : -1, 0};
    slots += n_s;
    joints += n_j;
    units += n_u;
  }
  if (threadIdx.x == 0) {
    w.ctl[0] = 0;
    w.ctl[1] = units;
    w.ctl[2] = joints;
  }
}

SSB_DEV bool ready(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity & 1)
      : "memory");
  return done;
}
// Waits for phase `parity`; false after SSB_WAIT_NS. try_wait: a waiting thread sleeps instead of taking issue slots from the
// softmax; no suspend-time hint: the roles hand tiles to one another several times per microsecond.
SSB_DEV bool wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  uint64_t t0 = 0;
  uint32_t i = 0;
#pragma unroll 1
  for (;;) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(addr), "r"(parity & 1)
        : "memory");
    if (done) return true;
    if (++i & 63u) continue;                         // the global timer is slow to read
    const uint64_t t = globaltimer_ns();
    if (t0 == 0) t0 = t;
    else if (t - t0 > SSB_WAIT_NS) return false;
  }
}
// The same by a whole warp that goes on to warp-wide instructions (TMEM, shuffles): the lanes may leave the wait one by one,
// and the vote brings them together again, so that either all of them go on or all of them give up. A full-mask instruction
// that some lanes have given up on would never end.
SSB_DEV bool warp_wait(uint64_t* bar, uint32_t parity) { return __all_sync(0xFFFFFFFFu, wait(bar, parity)); }

using OneLane = std::false_type;
using WholeWarp = std::true_type;

// Shared-memory descriptors as (low word, constant high word): moving inside a tile adds to the low word only. That keeps
// the one thread that issues the products off the critical path -- with descriptors built from scratch it took about 100
// cycles an instruction, more than the instruction itself.
SSB_DEV uint32_t desc_lo(uint32_t smem_addr, uint32_t lead) { return (smem_addr >> 4) | (lead >> 4) << 16; }
constexpr uint32_t desc_hi(uint32_t group) { return (group >> 4) | 1u << 14 | 2u << 29; }   // bytes between groups of 8 rows
// K-major tile (rows of 64 elements of the summed index); `lead` is not used by the swizzled form.
constexpr uint32_t LEAD_K = 16;

// One box of a 3-D / 5-D tensor map; the bytes are counted on `bar`.
SSB_DEV void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
SSB_DEV void tma_load_5d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, int v, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::
          "r"(dst),
      "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
      : "memory");
}

// D[tmem] (+)= A[smem] * B[smem]^T.
SSB_DEV void umma_ss(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc,
                     uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n mov.b64 da, {%1, %2};\n mov.b64 db, {%3, %4};\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n}\n" ::"r"(tmem_d),
      "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: the A rows are TMEM lanes, two 16-bit elements of a row per column.
SSB_DEV void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n mov.b64 db, {%2, %3};\n setp.ne.b32 p, %5, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n}\n" ::"r"(tmem_d),
      "r"(tmem_a), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
template <typename E>
__host__ __device__ constexpr uint32_t idesc_of(int m, int n, bool b_mn);
template <>
constexpr uint32_t idesc_of<__nv_bfloat16>(int m, int n, bool b_mn) {
  return idesc_bf16_f32(m, n) | (b_mn ? 1u << 16 : 0u);
}
template <>
constexpr uint32_t idesc_of<__half>(int m, int n, bool b_mn) {
  return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

SSB_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
SSB_DEV void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
SSB_DEV void tmem_ld16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr));
}
// N columns of this thread's TMEM lane, all loads in flight together. The empty statements keep uses behind the wait.
template <int N>
SSB_DEV void tmem_ld_row(uint32_t taddr, float* v) {
#pragma unroll
  for (int c = 0; c < N; c += 16) tmem_ld16(taddr + c, v + c);
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < N; c += 8)
    asm volatile("" : "+f"(v[c]), "+f"(v[c + 1]), "+f"(v[c + 2]), "+f"(v[c + 3]), "+f"(v[c + 4]), "+f"(v[c + 5]), "+f"(v[c + 6]),
                 "+f"(v[c + 7]));
}
// Bit x: token t0 + x (x < 32) is visible to the query at position p.
SSB_DEV uint32_t bits_below(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }
SSB_DEV uint32_t seen_bits(const Args& a, int p, int t0) {
  uint32_t m = bits_below(p + 1 - t0);
  if (a.window) m &= ~bits_below(window_start(a, p) - t0) | bits_below(a.sinks - t0);
  return m;
}
SSB_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename E, int D>
__global__ void __launch_bounds__(Cfg<D>::THREADS, 1) k_prefill(const __grid_constant__ Maps maps, Args a, Work w) {
  using C = Cfg<D>;
  constexpr int NT = C::NT, T = C::T, CPR = C::CPR, SLOTS = C::SLOTS, NBUF = C::NBUF;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* sq = smem;
  uint8_t* ring = smem + C::QB;
  uint64_t* bar = (uint64_t*)(ring + SLOTS * C::SLOT);
  uint64_t *q_full = bar, *q_empty = bar + 1, *u_full = bar + 2, *u_empty = bar + 4, *drained = bar + 6,
           *s_full = bar + 10, *p_full = bar + 16, *o_done = bar + 22, *full = bar + 28, *empty = full + SLOTS;
  int* u_slot = (int*)(empty + SLOTS);             // unit numbers handed out, two in flight
  uint32_t* tmem_slot = (uint32_t*)(u_slot + 2);
  int* failed = (int*)(tmem_slot + 1);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (smem_u32(smem) & 1023u) {                     // the swizzled tiles need it; the same for every thread
    if (tid == 0) set_err(a.err, SSB_ERR_MISALIGNED);
    return;
  }
  constexpr int PROD = NT * 4, MMA = PROD + 4;    // first warps of the roles

  if (warp == MMA) tmem_alloc(tmem_slot, 512);
  if (tid == 0) {
    mbar_init(q_full, 128);
    mbar_init(q_empty, NT);
    for (int i = 0; i < 2; ++i) {
      mbar_init(u_full + i, 1);
      mbar_init(u_empty + i, NT * 128 + 128 + 2 * NT);
    }
    for (int i = 0; i < 4; ++i) mbar_init(drained + i, 1);
    for (int i = 0; i < NT * NBUF; ++i) {            // [row tile][buffer]
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(full + i, 128);
      mbar_init(empty + i, NT);
    }
    *failed = 0;
    fence_mbar_init();
  }
  pdl_wait();
  pdl_trigger();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  auto give_up = [&] { atomicExch(failed, 1); };
  int un = 0;                                       // units this thread has seen
  // The next unit, or false at the end of the list (or when a wait gave up). `by_warp`: called by all lanes of a warp.
  auto next_unit = [&](Unit& u, auto by_warp) {
    const int s = un & 1;
    if (!(by_warp.value ? warp_wait(u_full + s, (un >> 1) & 1) : wait(u_full + s, (un >> 1) & 1))) {
      give_up();
      return false;
    }
    const int i = *(volatile int*)(u_slot + s);
    mbar_arrive(u_empty + s);
    ++un;
    if (i < 0) return false;
    u = w.units[i];
    return true;
  };
  auto range_for = [&](const Unit& u) {
    const int p = u.len - u.q;
    return range_of(a, p + u.r0 / a.group, p + (u.r0 + u.rows - 1) / a.group, T);
  };

  if (warp >= MMA + 2 * NT || (warp >= MMA && lane > 0)) {
    // the rest of the issuing warps
  } else if (warp >= MMA) {
    // One warp per row tile and product: a thread that waits on a barrier between two products leaves the tensor cores
    // idle for about 170 cycles (its queue is short), unless another thread's products fill the gap.
    constexpr uint32_t ID_S = idesc_of<E>(128, T, false), ID_O = idesc_of<E>(128, D, true);
    const int t = (warp - MMA) % NT;
    const bool scores = warp < MMA + NT;
    const uint32_t q_lo = desc_lo(smem_u32(sq) + t * 128 * 128, LEAD_K), k_lo = desc_lo(smem_u32(ring), LEAD_K),
                   v_lo = desc_lo(smem_u32(ring), 1024);
    constexpr uint32_t GROUP = D / 64 * 1024, HI_Q = desc_hi(1024), HI_KV = desc_hi(GROUP);
    // A commit costs the tensor cores about 40 cycles. With a long ring its slots are given back by plain arrivals, when a
    // later wait shows that the product has ended; with a short one (size 256) that would be too late.
    constexpr bool FREE_BY_COMMIT = SLOTS < 8;
    Unit u;
    uint32_t kv = 0, qn = 0, tn = 0;                // slots, units and tiles so far
    bool ok = true;
    auto need = [&](uint64_t* b, uint32_t parity) { ok = ok && wait(b, parity); };
    while (ok && next_unit(u, OneLane())) {
      if (scores) need(q_full, qn++);
#pragma unroll 1
      for (int i = u.i0; i < u.i1 && ok; ++i, ++tn, kv += 2) {
        const uint32_t buf = NBUF * t + tn % NBUF, use = tn / NBUF, sd = tmem + C::S_COL + buf * T;
        if (scores) {
          const uint32_t slot = kv % SLOTS;
          need(full + slot, kv / SLOTS);
          if (use) need(o_done + buf, use - 1);     // the product that read P from this buffer
          if (!ok) break;
          if (!FREE_BY_COMMIT && use) mbar_arrive(empty + (kv + 1 - 2 * NBUF) % SLOTS);      // and its values
          tc_fence_after();
          const uint32_t kd = k_lo + slot * (C::SLOT >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t kk = kd + (((k / 4) * 1024 + (k % 4) * 32) >> 4);
            umma_ss(sd, q_lo + (((k / 4) * (C::MB * 128) + (k % 4) * 32) >> 4), HI_Q, kk, HI_KV, ID_S, k > 0);
          }
          umma_commit(s_full + buf);
          if (FREE_BY_COMMIT) umma_commit(empty + slot);
        } else {
          const uint32_t slot = (kv + 1) % SLOTS;
          need(full + slot, (kv + 1) / SLOTS);
          need(p_full + buf, use);
          if (!ok) break;
          if (!FREE_BY_COMMIT) mbar_arrive(empty + kv % SLOTS);                       // S has been read: so have the keys
          tc_fence_after();
          const uint32_t vd = v_lo + slot * (C::SLOT >> 4), od = tmem + t * D;
#pragma unroll
          for (int k = 0; k < T / 16; ++k) umma_ts(od, sd + k * 8, vd + (k * 2 * GROUP >> 4), HI_KV, ID_O, i > u.i0 || k > 0);
          umma_commit(o_done + buf);
          if (FREE_BY_COMMIT) umma_commit(empty + slot);
        }
      }
      if (scores && ok) umma_commit(q_empty);
    }
    if (!ok) give_up();
    umma_commit(drained + (warp - MMA));            // nothing of this thread's may run when TMEM goes
    if (!wait(drained + (warp - MMA), 0)) give_up();
  } else if (warp >= PROD) {
    const int pt = tid - PROD * 32, pw = pt >> 5;
    Unit u;
    uint32_t kv = 0, qn = 0;
    bool ok = true;
    // The first of these threads also hands out the units, one ahead of its own use.
    const int units = w.ctl[1];
    uint32_t given = 0;
    auto give_unit = [&] {
      if (pt) return true;
      const uint32_t slot = given & 1;
      if (given >= 2 && !wait(u_empty + slot, (given >> 1) - 1)) return false;
      const int i = atomicAdd(w.ctl, 1);
      *(volatile int*)(u_slot + slot) = i < units ? i : -1;
      mbar_arrive(u_full + slot);
      ++given;
      return true;
    };
    // Every decision to go on or to give up is a vote of the warp: the shuffles below need all of its lanes.
    ok = __all_sync(0xFFFFFFFFu, give_unit());
    while (ok && next_unit(u, WholeWarp())) {
      if (!__all_sync(0xFFFFFFFFu, give_unit())) {
        ok = false;
        break;
      }
      const Range rg = range_for(u);
      const int p = u.len - u.q, p_lo = p + u.r0 / a.group, p_hi = p + (u.r0 + u.rows - 1) / a.group;
      const uint16_t *kh = a.k + u.h * a.sh, *vh = a.v + u.h * a.sh;
      const int32_t* trow = a.table + (int64_t)max(u.row, 0) * a.max_pages;
      if (qn && !warp_wait(q_empty, (qn - 1) & 1)) {
        ok = false;
        break;
      }
      ++qn;
      const bool boxes = w.q_boxes != 0;
      if (boxes) {
        constexpr int N = NT * (D / 64);               // one box per row tile and 64 columns
        if (pt < N) {
          const int t = pt % NT, c = pt / NT;
          mbar_expect_tx(q_full, 128 * 128);
          tma_load_3d(smem_u32(sq) + c * (C::MB * 128) + t * (128 * 128), &maps.q, c * 64, u.h * a.group,
                      u.q0 + (u.r0 + t * 128) / a.group, q_full);
        } else {
          mbar_arrive(q_full);
        }
      } else {
        constexpr int RPP = 128 / CPR;                 // rows a pass
        const int c = pt % CPR;
        const uint32_t dst = smem_u32(sq) + (c >> 3) * (C::MB * 128);
        const uint16_t* base = a.q + (int64_t)u.q0 * a.q_tok + (int64_t)u.h * a.group * a.q_head + c * 8;
#pragma unroll 4
        for (int r = pt / CPR; r < C::MB; r += RPP) {
          const int f = u.r0 + r, t = (int)((__umulhi((uint32_t)f, a.group_mul) + (uint32_t)f) >> a.group_shift);
          const int64_t off = t * a.q_tok + (f - t * a.group) * a.q_head;
          cp_async16(dst + swz128(r, c & 7), base + (r < u.rows ? off : 0), r < u.rows ? 16 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      // tokens of this warp: rows [pw * T / 4, (pw + 1) * T / 4) of a tile; lane l holds the offset of row l
      auto offset_of = [&](int i) -> long long {
        if (i >= u.i1 || lane >= T / 4) return -1;
        const int t = tile_token(rg, i, T) + pw * (T / 4) + lane;
        if (!seen_by_any(a, t, p_lo, p_hi)) return -1;
        const int j = page_of(a, t), page = trow[j];
        if (page < 0 || page >= a.pages) {
          set_err(a.err, SSB_ERR_PAGE_RANGE);
          return -1;
        }
        return (long long)page * a.sp + (long long)(t - j * a.page_size) * a.st;
      };
      uint32_t first = kv;                            // oldest slot that is not handed over yet
      bool q_given = boxes;
      auto hand_over = [&](uint32_t upto) {           // the copies of the slots before `upto` have landed
        fence_proxy_async_smem();
        if (!q_given && first < upto) {
          q_given = true;
          mbar_arrive(q_full);
        }
        for (; first < upto; ++first) mbar_arrive(full + first % SLOTS);
      };
      // A tile whose tokens are all seen by some query comes as boxes, one page's tokens each, box pt by thread pt; others,
      // and pages that do not divide a tile, row by row, with zeros for what nobody sees.
      const int n_boxes = w.page_rows ? T / w.page_rows : 0;
      auto boxed = [&](int i) {
        const int t = tile_token(rg, i, T);
        return w.page_rows && t + T - 1 <= p_hi && (a.window == 0 || p_lo - t < a.window || t + T <= a.sinks);
      };
      auto box_page = [&](int i) {                    // page of this thread's box
        return i < u.i1 && pt < n_boxes ? trow[page_of(a, tile_token(rg, i, T) + pt * w.page_rows)] : 0;
      };
      bool as_box = boxed(u.i0);
      long long off = as_box ? -1 : offset_of(u.i0);
      int page = as_box ? box_page(u.i0) : 0;
      for (int i = u.i0; i < u.i1 && ok; ++i) {
        asm volatile("" : "+r"(page), "+l"(off));     // loaded a tile ago; their checks stay behind this point
        const bool box_next = i + 1 < u.i1 && boxed(i + 1);
        const long long off_next = box_next ? -1 : offset_of(i + 1);
        const int page_next = box_next ? box_page(i + 1) : 0;
        if (as_box) {
          if (first < kv || !q_given) {               // copies on their way go first
            cp_async_wait_all();
            hand_over(kv);
            if (!q_given) {
              q_given = true;
              mbar_arrive(q_full);
            }
          }
          const int t0 = tile_token(rg, i, T) + pt * w.page_rows, in_page = t0 - page_of(a, t0) * a.page_size;
          const uint32_t at = pt * w.page_rows * (D * 2);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (kv >= SLOTS && !warp_wait(empty + kv % SLOTS, kv / SLOTS - 1)) {
              ok = false;
              break;
            }
            uint64_t* bar_full = full + kv % SLOTS;
            if (pt >= n_boxes) {
              mbar_arrive(bar_full);
            } else if (page >= 0 && page < a.pages) {
              mbar_expect_tx(bar_full, w.page_rows * (D * 2));
              tma_load_5d(smem_u32(ring + (kv % SLOTS) * C::SLOT) + at, x ? &maps.v : &maps.k, 0, 0, 0, in_page >> 3,
                          page * w.page_heads + u.h, bar_full);
            } else {                                  // a missing page reads as zeros
              set_err(a.err, SSB_ERR_PAGE_RANGE);
              uint4* z = (uint4*)(ring + (kv % SLOTS) * C::SLOT + at);
              for (int y = 0; y < w.page_rows * (D / 8); ++y) z[y] = make_uint4(0, 0, 0, 0);
              fence_proxy_async_smem();
              mbar_arrive(bar_full);
            }
            ++kv;
          }
          first = kv;
        } else {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (kv >= SLOTS && !__all_sync(0xFFFFFFFFu, ready(empty + kv % SLOTS, kv / SLOTS - 1))) {
              cp_async_wait_all();                     // nothing to issue: hand over what is on its way first
              hand_over(kv);
              if (!warp_wait(empty + kv % SLOTS, kv / SLOTS - 1)) {
                ok = false;
                break;
              }
            }
            const uint32_t dst = smem_u32(ring + (kv % SLOTS) * C::SLOT);
            const uint16_t* base = x ? vh : kh;
            constexpr int RPP = 32 / CPR > 0 ? 32 / CPR : 1, PASSES = (T / 4) * CPR / 32;
#pragma unroll 4
            for (int v = 0; v < PASSES; ++v) {
              const int r = v * RPP + lane / CPR, c = lane % CPR;
              const long long o = __shfl_sync(0xFFFFFFFFu, off, r);
              const uint32_t row = pw * (T / 4) + r;
              cp_async16(dst + (row >> 3) * (D * 16) + (c >> 3) * 1024 + swz128(row & 7, c & 7), base + (o < 0 ? 0 : o) + c * 8,
                         o < 0 ? 0 : 16);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            ++kv;
            if (kv - first > LAG) {
              asm volatile("cp.async.wait_group %0;" ::"n"(LAG) : "memory");
              hand_over(kv - LAG);
            }
          }
        }
        off = off_next;
        page = page_next;
        as_box = box_next;
      }
      cp_async_wait_all();
      if (ok) hand_over(kv);
    }
    cp_async_wait_all();
    // No copy of this block's may be on its way when it ends (after a wait that gave up, one could be).
    if (qn) ok = wait(q_full, qn - 1) && ok;
    for (uint32_t n = kv > SLOTS ? kv - SLOTS : 0; n < kv; ++n) ok = wait(full + n % SLOTS, n / SLOTS) && ok;
    if (!ok) give_up();
  } else {
    const int t = warp >> 2, row = tid & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(warp & 3) << 21);
    Unit u;
    uint32_t tn = 0;
    bool ok = true;
    while (ok && next_unit(u, WholeWarp())) {
      const Range rg = range_for(u);
      const int p = u.len - u.q, f0 = u.r0 + t * 128, last = u.r0 + u.rows - 1;
      // rows past the last have zero queries or, where Q came in boxes, another sequence's; they are never written
      const int pos = p + min(f0 + row, last) / a.group;
      const int t_lo = p + min(f0, last) / a.group, t_hi = p + min(f0 + 127, last) / a.group;
      float m = -INFINITY, l = 0.f;
      for (int i = u.i0; i < u.i1; ++i, ++tn) {
        const uint32_t buf = NBUF * t + tn % NBUF, sc = lane_base + C::S_COL + buf * T;
        if (!warp_wait(s_full + buf, tn / NBUF)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int tok = tile_token(rg, i, T);
        float v[T];
        tmem_ld_row<T>(sc, v);
        if (!seen_by_all(a, tok, tok + T, t_lo, t_hi)) {
#pragma unroll
          for (int c = 0; c < T; c += 16) {
            const uint32_t bits = seen_bits(a, pos, tok + c);
#pragma unroll
            for (int x = 0; x < 16; ++x)
              if (!(bits >> x & 1)) v[c + x] = -INFINITY;
          }
        }
        float m4[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int x = 4; x < T; x += 8) {
#pragma unroll
          for (int y = 0; y < 4; ++y)
            m4[y] = x + 4 + y < T ? fmaxf(m4[y], fmaxf(v[x + y], v[x + 4 + y])) : fmaxf(m4[y], v[x + y]);
        }
        const float mx = below_max<E, STEP>(fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2);
        if (i == u.i0) {
          m = mx;
        } else {
          const bool raise = mx > m + STEP;
          if (__any_sync(0xFFFFFFFFu, raise)) {
            // the product of the tile before adds to the sum
            if (!warp_wait(o_done + NBUF * t + (tn - 1) % NBUF, (tn - 1) / NBUF)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const float f = raise ? ex2(m - mx) : 1.f;
            if (raise) m = mx;
            l *= f;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld_row<16>(lane_base + t * D + c, o);
              uint32_t r[16];
#pragma unroll
              for (int x = 0; x < 16; ++x) r[x] = __float_as_uint(o[x] * f);
              tmem_st16(lane_base + t * D + c, r);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.f : m;
        const float2 sc2 = make_float2(a.scale_log2, a.scale_log2), mu2 = make_float2(-mu, -mu);
        float2 l2 = make_float2(0.f, 0.f), l3 = l2;
#pragma unroll
        for (int c = 0; c < T; c += 16) {
          uint32_t r[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            float2 e = __ffma2_rn(make_float2(v[c + 2 * x], v[c + 2 * x + 1]), sc2, mu2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            if (x & 1) l3 = __fadd2_rn(l3, e);
            else l2 = __fadd2_rn(l2, e);
            r[x] = pack2<E>(e.x, e.y);
          }
          tmem_st8(sc + c / 2, r);               // P takes the place of S, which is in registers
        }
        l += (l2.x + l2.y) + (l3.x + l3.y);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full + buf);
      }
      if (!ok || !warp_wait(o_done + NBUF * t + (tn - 1) % NBUF, (tn - 1) / NBUF)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int fr = f0 + row;
      const bool in = t * 128 + row < u.rows;
      const int tk = fr / a.group, hg = fr - tk * a.group;
      const int64_t orow = (u.q0 + (int64_t)tk) * a.heads + u.h * a.group + hg;
      const int64_t prow = (int64_t)u.slot * C::MB + t * 128 + row;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        float v[32];
        __syncwarp();                                  // the rows past the last skip the stores
        tmem_ld_row<32>(lane_base + t * D + c, v);
        if (in && u.slot < 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *(uint4*)(a.out + orow * D + c + 8 * x) =
                make_uint4(pack2<E>(v[8 * x] * inv, v[8 * x + 1] * inv), pack2<E>(v[8 * x + 2] * inv, v[8 * x + 3] * inv),
                           pack2<E>(v[8 * x + 4] * inv, v[8 * x + 5] * inv), pack2<E>(v[8 * x + 6] * inv, v[8 * x + 7] * inv));
        } else if (in) {
#pragma unroll
          for (int x = 0; x < 8; ++x)
            *(float4*)(a.acc + prow * D + c + 4 * x) = make_float4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
        }
      }
      if (in) {
        if (u.slot >= 0) a.ml[prow] = make_float2(m, l);
        else if (a.lse) a.lse[orow] = (m + log2f(l)) * LN2;
      }
    }
    if (!ok) give_up();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == MMA) tmem_dealloc(tmem, 512);
  if (tid == 0 && *failed) set_err(a.err, SSB_ERR_TIMEOUT);
}

// Sums the pieces of the items that were cut: grid (joints at most, MB / 8), eight rows a block, D / 4 threads a row.
template <typename E, int D>
__global__ void __launch_bounds__(2 * D) k_prefill_join(Args a, Work w) {
  pdl_wait();
  if ((int)blockIdx.x >= w.ctl[2]) return;
  const Joint j = w.joints[blockIdx.x];
  const int r = blockIdx.y * 8 + threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
  if (r >= j.rows) return;
  const int64_t at = (int64_t)j.slot * Cfg<D>::MB + r;
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < j.pieces; ++i) m = fmaxf(m, a.ml[at + (int64_t)i * Cfg<D>::MB].x);
  const float u = m == -INFINITY ? 0.f : m;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < j.pieces; ++i) {
    const int64_t s = at + (int64_t)i * Cfg<D>::MB;
    const float2 e = a.ml[s];
    const float f = ex2(e.x - u);
    const float4 x = *(const float4*)(a.acc + s * D + c * 4);
    l += e.y * f;
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  const int fr = j.r0 + r, t = fr / a.group, g = fr - t * a.group;
  const int64_t row = (j.q0 + (int64_t)t) * a.heads + j.h * a.group + g;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  *(uint2*)(a.out + row * D + c * 4) = make_uint2(pack2<E>(o.x * inv, o.y * inv), pack2<E>(o.z * inv, o.w * inv));
  if (a.lse && c == 0) a.lse[row] = (m + log2f(l)) * LN2;
}

struct Layout {
  int64_t item0, ctl, units, joints, ml, acc, bytes;
  int max_units, max_slots;
};
int64_t up(int64_t x) { return (x + 127) / 128 * 128; }
Layout layout_of(int dim, int n, int64_t rows, int heads, int kv_heads) {
  const int mb = dim == 256 ? 128 : 256, blocks = ssb_sm_count();
  Layout l;
  const int64_t items = (rows * (heads / kv_heads) / mb + n) * kv_heads;
  l.max_slots = 4 * blocks;
  l.max_units = (int)items;
  l.item0 = 0;
  l.ctl = up((int64_t)(n + 1) * 4);
  l.units = l.ctl + 128;
  l.joints = l.units + up((items + l.max_slots) * (int64_t)sizeof(Unit));
  l.ml = l.joints + up(l.max_slots / 2 * (int64_t)sizeof(Joint));
  l.acc = l.ml + up((int64_t)l.max_slots * mb * 8);
  l.bytes = l.acc + (int64_t)l.max_slots * mb * dim * 4;
  return l;
}

// The driver's tensor-map encoder, looked up through the runtime.
using EncodeFn = decltype(&cuTensorMapEncodeTiled);
EncodeFn encode_fn() {
  static EncodeFn fn = []() -> EncodeFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return nullptr;
    }
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}
bool encode(CUtensorMap* m, bool bf16, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  for (int i = 0; i + 1 < rank; ++i)                 // what the encoder refuses goes by cp.async
    if (strides[i] == 0 || strides[i] >= (1ull << 40)) return false;
  EncodeFn f = encode_fn();
  return f && f(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims,
                strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Boxes need pages that divide a tile or are divided by it, in groups of 8 tokens, page strides that are whole numbers of
// head strides (page and head are one index of the map), and a group that divides the 128 rows of a row tile.
void make_maps(Maps& m, Work& w, const Args& a, bool bf16, int dim, int tile) {
  w.page_rows = w.q_boxes = w.page_heads = 0;
  if (a.page_size >= 8 && (a.page_size & (a.page_size - 1)) == 0 && a.st > 0 && a.sh > 0 && a.sp > 0 && a.sp % a.sh == 0 &&
      ((int64_t)a.pages * (a.sp / a.sh) + a.kv_heads) < 0x7FFFFFFF) {
    const int rows = a.page_size < tile ? a.page_size : tile;
    const cuuint64_t steps = (cuuint64_t)(a.sp / a.sh);
    const cuuint64_t dims[5] = {64, 8, (cuuint64_t)dim / 64, (cuuint64_t)a.page_size / 8,
                                (cuuint64_t)(a.pages - 1) * steps + (cuuint64_t)a.kv_heads};
    const cuuint64_t strides[4] = {(cuuint64_t)a.st * 2, 128, (cuuint64_t)a.st * 16, (cuuint64_t)a.sh * 2};
    const cuuint32_t box[5] = {64, 8, (cuuint32_t)dim / 64, (cuuint32_t)rows / 8, 1};
    if (encode(&m.k, bf16, 5, a.k, dims, strides, box) && encode(&m.v, bf16, 5, a.v, dims, strides, box)) {
      w.page_rows = rows;
      w.page_heads = (int)steps;
    }
  }
  if (128 % a.group == 0) {
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)a.heads, (cuuint64_t)a.rows};
    const cuuint64_t strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_tok * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(128 / a.group)};
    w.q_boxes = a.q_head > 0 && a.q_tok > 0 && encode(&m.q, bf16, 3, a.q, dims, strides, box);
  }
}

template <typename E, int D>
int launch(Args& a, uint8_t* ws, const Layout& l, cudaStream_t stream) {
  using C = Cfg<D>;
  Work w;
  w.item0 = (int*)(ws + l.item0);
  w.ctl = (int*)(ws + l.ctl);
  w.units = (Unit*)(ws + l.units);
  w.joints = (Joint*)(ws + l.joints);
  w.max_units = l.max_units;
  w.max_slots = l.max_slots;
  a.ml = (float2*)(ws + l.ml);
  a.acc = (float*)(ws + l.acc);
  auto kern = k_prefill<E, D>;
  static std::atomic<uint64_t> done{0};
  int rc = ssb_setup_kernel(done, "attn_prefill", kern, C::SMEM);
  if (rc) return rc;
  Maps maps = {};
  make_maps(maps, w, a, sizeof(E) == 2 && idesc_of<E>(128, 64, false) == idesc_of<__nv_bfloat16>(128, 64, false), D, C::T);
  const int blocks = ssb_sm_count();
  rc = ssb_launch(k_prefill_plan<C::MB, C::T>, dim3(1), dim3(PLAN_T), 0, stream, false, a, w, blocks);
  if (rc) return rc;
  rc = ssb_launch(kern, dim3(blocks), dim3(C::THREADS), C::SMEM, stream, true, maps, a, w);
  if (rc) return rc;
  return ssb_launch(k_prefill_join<E, D>, dim3(l.max_slots / 2, C::MB / 8), dim3(2 * D), 0, stream, true, a, w);
}

}  // namespace

int64_t prefill_workspace(int dim, int n, int64_t rows, int heads, int kv_heads) {
  return layout_of(dim, n, rows, heads, kv_heads).bytes;
}

int prefill_launch(Args& a, int dim, bool bf16, void* ws, void* stream) {
  const Layout l = layout_of(dim, a.n, a.rows, a.heads, a.kv_heads);
  uint8_t* p = (uint8_t*)ws;
  cudaStream_t st = (cudaStream_t)stream;
  if (bf16)
    return dim == 64 ? launch<__nv_bfloat16, 64>(a, p, l, st)
                     : dim == 128 ? launch<__nv_bfloat16, 128>(a, p, l, st) : launch<__nv_bfloat16, 256>(a, p, l, st);
  return dim == 64 ? launch<__half, 64>(a, p, l, st)
                   : dim == 128 ? launch<__half, 128>(a, p, l, st) : launch<__half, 256>(a, p, l, st);
}

}  // namespace attn
