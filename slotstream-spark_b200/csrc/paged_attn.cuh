// Shared pieces of the attention kernels over the paged key-value cache: arguments, sequences, visible-tile ranges, the
// rounding of the weights.
//
// Work is a list of items -- (sequence, key head, block of query rows) -- each a run of tiles of the tokens it can
// see. How they are divided:
// - few rows, long items (paged_attn.cu, k_attn_rows<DIRECT = false>): the total number of tiles evenly over the blocks,
//   whatever the lengths: block c takes tiles [c * chunk, (c + 1) * chunk) of the concatenated items. An item inside one
//   block is finished there; one that crosses blocks leaves (max, sum, accumulator) pieces in the workspace, which
//   k_attn_join sums in block order.
// - few rows, short items (DIRECT): a cluster of one to eight blocks an item, joined in rank order through shared memory.
// - prompts (paged_prefill.cu): a planned list of whole items and pieces of items, taken by a counter; k_prefill_join sums
//   the pieces of an item in their order.
// In each case what is summed with what depends on the lengths alone, so results do not change from run to run.
#pragma once
#include <type_traits>

#include "common.cuh"
#include "registry.h"

namespace attn {

struct Args {
  const uint16_t* q;
  int64_t q_seq, q_tok, q_head;       // strides in elements; q_seq unused for ragged rows
  const uint16_t *k, *v;
  int64_t sp, sh, st;                 // page, head, token strides
  int64_t rows;                       // query tokens
  const int32_t* starts;              // ragged rows; nullptr: q_len rows of every sequence
  int32_t n, q_len, heads, kv_heads, group;
  int32_t page_size, pages, table_rows, max_pages;
  uint32_t page_mul, page_shift;      // t / page_size for t < 2^31: (mulhi(t, mul) + t) >> shift
  uint32_t group_mul, group_shift;    // the same for the group
  const int32_t *table, *lengths, *ids;
  int32_t window, sinks;
  float scale_log2;                   // scale * log2(e)
  uint16_t* out;
  float* lse;
  int32_t* err;
  int4* desc;                         // items to join (see k_attn_join)
  int desc_by_item;
  float2* ml;                         // (max, sum) of the pieces' rows, log2 domain: [2 * blocks, RB], or [slots, MB] for prompts
  float* acc;                         // their accumulators, D floats a row
};

SSB_DEV int page_of(const Args& a, int t) { return (int)((__umulhi((uint32_t)t, a.page_mul) + (uint32_t)t) >> a.page_shift); }

// One sequence of the batch: its queries are the newest tokens, so row i sits at position len - q + i.
struct Seq {
  int row;          // table row; < 0 when the id is out of range (reads as empty)
  int len, q;
  int64_t q0;       // first query token (row of out)
};
SSB_DEV Seq seq_of(const Args& a, int b) {
  Seq s;
  s.row = a.ids ? a.ids[b] : b;
  if (a.starts) {
    const int64_t r0 = max(a.starts[b], 0), r1 = min((int64_t)a.starts[b + 1], a.rows);
    s.q0 = r0;
    s.q = (int)max(r1 - r0, (int64_t)0);
  } else {
    s.q0 = (int64_t)b * a.q_len;
    s.q = a.q_len;
  }
  s.len = 0;
  if (s.row < 0 || s.row >= a.table_rows) s.row = -1;
  else s.len = (int)min((int64_t)max(a.lengths[s.row], 0), (int64_t)a.max_pages * a.page_size);
  return s;
}

// First token inside the window of a query at position p. Queries before the sequence's start have negative positions and
// see nothing; taken as position 0, the difference stays inside 32 bits for any window.
SSB_DEV int window_start(const Args& a, int p) { return max(max(p, 0) - a.window + 1, 0); }

// The tiles of T tokens that rows at positions p_min .. p_max can see: the sinks' first, then the window's. A range
// without a visible token has one (fully masked) tile, so that its rows are still written.
struct Range {
  int sink_tiles, first, tiles;
};
SSB_DEV Range range_of(const Args& a, int p_min, int p_max, int T) {
  Range r;
  const int end = p_max < 0 ? 0 : p_max / T + 1;
  r.first = a.window ? window_start(a, p_min) / T : 0;
  r.first = min(r.first, end);
  r.sink_tiles = min((a.sinks + T - 1) / T, r.first);
  r.tiles = max(r.sink_tiles + end - r.first, 1);
  return r;
}
SSB_DEV int tile_token(const Range& r, int i, int T) { return (i < r.sink_tiles ? i : i - r.sink_tiles + r.first) * T; }

SSB_DEV bool seen(const Args& a, int t, int p) { return t <= p && (a.window == 0 || p - t < a.window || t < a.sinks); }
// Some row between p_min and p_max sees t.
SSB_DEV bool seen_by_any(const Args& a, int t, int p_min, int p_max) {
  return t <= p_max && (a.window == 0 || p_min - t < a.window || t < a.sinks);
}
// Every row between p_min and p_max sees all of [t0, t1).
SSB_DEV bool seen_by_all(const Args& a, int t0, int t1, int p_min, int p_max) {
  return t1 - 1 <= p_min && (a.window == 0 || p_max - t0 < a.window || t1 <= a.sinks);
}

template <typename E>
SSB_DEV uint32_t pack2(float lo, float hi);
template <>
SSB_DEV uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
SSB_DEV uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
SSB_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LN2 = 0.6931471805599453f;

// The weights p = 2^(s - m) are rounded to E for the second product. fp16 has no normal numbers below 2^-14, and a long context
// is made of weights that small as soon as one token stands out by 10 nats; so for it m is kept 15 - STEP below the maximum
// (STEP: how far the maximum may run ahead of m), which puts the largest weight at 2^15, just inside the type. o and l carry
// the factor alike and m + log2 l does not see it. Weights then keep 11 bits down to 2^(STEP - 29) of the largest and an
// absolute 2^(STEP - 40) of it below. Where scores are so large that m would lose the 15 to rounding, m is the maximum itself.
template <typename E, int STEP>
SSB_DEV float below_max(float max) {
  constexpr float LIFT = std::is_same<E, __half>::value ? 15.f - STEP : 0.f;
  return LIFT == 0.f || fabsf(max) >= 1048576.f ? max : max - LIFT;
}

// csrc/paged_prefill.cu
int64_t prefill_workspace(int dim, int n, int64_t rows, int heads, int kv_heads);
int prefill_launch(Args& a, int dim, bool bf16, void* ws, void* stream);

}  // namespace attn
