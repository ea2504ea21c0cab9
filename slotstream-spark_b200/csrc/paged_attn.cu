// Attention over the paged key-value cache for few query rows per key head: decode steps and speculative verifies.
//
// Per item (sequence, key head, block of RB query rows): s = q k^T, online softmax (running maximum and sum, fp32,
// log2 domain), o = p v. Up to 16 rows of one key head -- query tokens x heads of its group -- share every key and value
// read, so up to there each cached byte is read once per key head: the kernel is bound by reading the cache. More rows (a
// verify of four tokens of a group of eight, say) are several items, and each of them reads the cache again. Tensor cores
// (mma.sync m16n8k16, fp32 accumulation) do both products, since RB x D x 2 multiply-adds per cached element pair
// would otherwise take more issue slots than the loads leave; tcgen05's 128-row tiles would be mostly padding here. The
// products are taken transposed -- S^T = K Q^T, O^T = V^T P^T -- so that the query rows are the instruction's 8 columns
// and nothing is padded to 16 for groups of up to eight rows (at 131,072 tokens and head size 256, 84 us with rows padded to
// 16, 57 us now).
//
// A block has NW warps that work alone: each walks every NW-th sub-tile of TW tokens through its own ring of cp.async
// units (no block barrier inside an item), and the warps' (max, sum, accumulator) are joined through shared
// memory at the end of the item. p is rounded to the inputs' type for the second product (half an ulp: relative 2^-8 for bf16,
// 2^-11 for fp16 down to 2^-29 of the largest weight and 2^-40 of that one below, see below_max; as the library's other
// tensor-core inputs); its sum is taken before the rounding, in fp32.
#include "paged_attn.cuh"

#include <cooperative_groups.h>

#include "affine.cuh"
#include "tc_common.cuh"

namespace attn {
namespace {

SSB_DEV void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
SSB_DEV void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Transposes an 8 x 8 matrix of 16-bit elements held two a thread.
SSB_DEV uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename E>
SSB_DEV void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1);
template <>
SSB_DEV void mma16816<__nv_bfloat16>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
SSB_DEV void mma16816<__half>(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte chunk c of row r of a [rows][D] 16-bit tile: chunks are XORed with the row inside groups of eight, so that
// the eight rows of an ldmatrix fall into different banks.
template <int D>
SSB_DEV uint32_t swz(int r, int c) {
  return (uint32_t)(r * (D * 2) + ((c ^ (r & 7)) << 4));
}

constexpr int NW = 4;
template <int D>
constexpr int TW = D == 256 ? 16 : 32;            // tokens of a warp's sub-tile
template <int D>
constexpr int UNIT = TW<D> * D * 2;               // keys, or values, of one sub-tile
template <int D>
constexpr int NU = D == 64 ? 6 : 3;               // units in a warp's ring: 24 KB, all but one in flight
template <int D, int RB>
constexpr int SMEM = RB * D * 2 + NW * NU<D> * UNIT<D>;
constexpr int BLOCKS_PER_SM = 2;

template <typename E, int D, int RB, bool DIRECT>
__global__ void __launch_bounds__(NW * 32, BLOCKS_PER_SM) k_attn_rows(Args a, int cluster) {
  constexpr int T = NW * TW<D>, CPR = D / 8, NB = RB / 8;       // tokens of a tile, 16-byte chunks and blocks of 8 rows
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scan[NW];
  __shared__ long long place[2];                   // the sequence where this block starts, and its first tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* sq = smem;
  uint8_t* ring = smem + RB * D * 2 + warp * NU<D> * UNIT<D>;
  pdl_wait();
  pdl_trigger();                                   // the join's blocks may come up; they wait for this grid's end

  // ---- this block's share: tiles of all sequences, divided evenly. One scan of the sequences' weights for each NW * 32 of
  // them; where they all fit in one, it gives the total and the place of this block's first tile at once.
  auto weight_of = [&](int b) -> long long {
    if (b >= a.n) return 0;
    const Seq s = seq_of(a, b);
    const long long items = (long long)a.kv_heads * ((s.q * a.group + RB - 1) / RB);
    return DIRECT ? items : items * range_of(a, s.len - s.q, s.len - 1, T).tiles;
  };
  auto scan_block = [&](long long w, long long* sum) {      // inclusive
    long long inc = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      if (v < warp) before += scan[v];
      all += scan[v];
    }
    *sum = all;
    return before + inc;
  };
  if (!DIRECT && !a.desc_by_item && tid == 0) a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  long long w0 = weight_of(tid), total;
  const long long inc0 = scan_block(w0, &total);
  const long long first_total = total;
  if (a.n > NW * 32) {
    long long more = 0;
    for (int b = tid + NW * 32; b < a.n; b += NW * 32) more += weight_of(b);
    long long rest;
    scan_block(more, &rest);
    total += rest;
  }
  // DIRECT: an item a cluster, whose blocks share its tiles (all of a cluster returns here, or none does)
  const int rank = DIRECT ? blockIdx.x % cluster : 0;
  const long long chunk = DIRECT ? 1 : max((total + gridDim.x - 1) / gridDim.x, 1ll);
  const long long lo = DIRECT ? blockIdx.x / cluster : chunk * blockIdx.x, hi = min(lo + chunk, total);
  if (lo >= hi) return;
  // the sequence that holds tile `lo`, and its first tile
  if (lo >= inc0 - w0 && lo < inc0) {
    place[0] = tid;
    place[1] = inc0 - w0;
  }
  long long seen_total = first_total;
  for (int b0 = NW * 32; lo >= seen_total; b0 += NW * 32) {
    long long sum;
    const long long w = weight_of(b0 + tid), inc = seen_total + scan_block(w, &sum);
    if (lo >= inc - w && lo < inc) {
      place[0] = b0 + tid;
      place[1] = inc - w;
    }
    seen_total += sum;
  }
  __syncthreads();
  int b = (int)place[0];
  long long begin = place[1];

  long long at = lo;
  Seq s = seq_of(a, b);
  while (at < hi) {
    const Range rg = range_of(a, s.len - s.q, s.len - 1, T);
    const int nb = (s.q * a.group + RB - 1) / RB;
    const long long unit = DIRECT ? 1 : rg.tiles, weight = a.kv_heads * nb * unit;
    if (at >= begin + weight) {
      begin += weight;
      s = seq_of(a, ++b);
      continue;
    }
    // ---- one item, or the part of it inside this block
    const int item = (int)((at - begin) / unit), h = item / nb, rb = item - h * nb;
    const long long item0 = begin + item * unit;
    const int i0 = DIRECT ? (int)((long long)rg.tiles * rank / cluster) : (int)(at - item0);
    const int i1 = DIRECT ? (int)((long long)rg.tiles * (rank + 1) / cluster) : (int)min((long long)rg.tiles, hi - item0);
    const int r0 = rb * RB, rows = min(RB, s.q * a.group - r0);
    const int p_first = s.len - s.q, p_lo = p_first + r0 / a.group, p_hi = p_first + (r0 + rows - 1) / a.group;

    const uint16_t *kh = a.k + h * a.sh, *vh = a.v + h * a.sh;
    const int32_t* trow = a.table + (int64_t)max(s.row, 0) * a.max_pages;
    // Element offset of token t inside a layer's keys or values, -1 where it reads as zeros.
    auto offset_of = [&](int t) -> long long {
      if (!seen_by_any(a, t, p_lo, p_hi)) return -1;
      const int j = page_of(a, t), page = trow[j];
      if (page < 0 || page >= a.pages) {
        set_err(a.err, SSB_ERR_PAGE_RANGE);
        return -1;
      }
      return (long long)page * a.sp + (long long)(t - j * a.page_size) * a.st;
    };
    // Unit n of this part: keys (n even) or values (n odd) of tile i0 + n / 2. Lane l holds the offset of token l; values
    // are issued right after their keys and use the same.
    const int n_units = 2 * (i1 - i0);
    long long mine_off = -1;
    auto issue = [&](int n) {
      if (n < n_units) {
        if ((n & 1) == 0) mine_off = lane < TW<D> ? offset_of(tile_token(rg, i0 + (n >> 1), T) + warp * TW<D> + lane) : -1;
        const uint32_t dst = smem_u32(ring + n % NU<D> * UNIT<D>);
        const uint16_t* base = n & 1 ? vh : kh;
#pragma unroll
        for (int u = 0; u < TW<D> * CPR / 32; ++u) {
          const int r = (u * 32 + lane) / CPR, c = (u * 32 + lane) % CPR;
          const long long off = __shfl_sync(0xFFFFFFFFu, mine_off, r);
          cp_async16(dst + swz<D>(r, c), base + (off < 0 ? 0 : off) + c * 8, off < 0 ? 0 : 16);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto landed = [&] {                              // the oldest unit in flight is there, for every lane
      asm volatile("cp.async.wait_group %0;" ::"n"(NU<D> - 2) : "memory");
      __syncwarp();
    };

#pragma unroll
    for (int n = 0; n < NU<D> - 1; ++n) issue(n);
    for (int i = tid; i < RB * CPR; i += NW * 32) {
      const int r = i / CPR, c = i - r * CPR;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows) {
        const int t = (r0 + r) / a.group, g = (r0 + r) - t * a.group;
        const int64_t qt = a.starts ? (s.q0 + t) * a.q_tok : (int64_t)b * a.q_seq + t * a.q_tok;
        v = __ldg((const uint4*)(a.q + qt + (h * a.group + g) * a.q_head + c * 8));
      }
      *(uint4*)(sq + swz<D>(r, c)) = v;
    }
    __syncthreads();

    // Rows are the columns of both products (see the top): a thread holds rows 8 n + 2 (lane % 4) and the next of every
    // n < NB, as columns of S^T (tokens lane / 4 and + 8 of a group of 16) and of O^T (dims lane / 4 and + 8 of 16).
    constexpr int MT = TW<D> / 16, KS = D / 16;
    constexpr bool Q_IN_REGS = KS * NB <= 16;
    float acc[KS][NB][4];
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int n = 0; n < NB; ++n) acc[j][n][0] = acc[j][n][1] = acc[j][n][2] = acc[j][n][3] = 0.f;
    float m[NB][2], l[NB][2];
    int pos[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        m[n][y] = -INFINITY;
        l[n][y] = 0.f;
        // rows past the item's last have zero queries and are never written: they take the last one's position
        pos[n][y] = p_first + (r0 + min(n * 8 + (lane & 3) * 2 + y, rows - 1)) / a.group;
      }
    auto load_q = [&](int kk, int n, uint32_t* b) {  // two steps of 16 dims: b[0..1] of kk, b[2..3] of kk + 1
      ldsm4(smem_u32(sq) + swz<D>(n * 8 + (lane & 7), 2 * kk + (lane >> 3)), b);
    };
    uint32_t qf[Q_IN_REGS ? KS : 2][NB][2];
    if constexpr (Q_IN_REGS) {
#pragma unroll
      for (int kk = 0; kk < KS; kk += 2)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          uint32_t b[4];
          load_q(kk, n, b);
          qf[kk][n][0] = b[0];
          qf[kk][n][1] = b[1];
          qf[kk + 1][n][0] = b[2];
          qf[kk + 1][n][1] = b[3];
        }
    }

    for (int i = i0; i < i1; ++i) {
      const int un = 2 * (i - i0);
      landed();
      const uint32_t ks = smem_u32(ring + un % NU<D> * UNIT<D>);
      const int t0 = tile_token(rg, i, T) + warp * TW<D>;
      float c[MT][NB][4], c2[MT][NB][4];              // even and odd steps: two chains hide the instruction's latency
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) c[x][n][y] = c2[x][n][y] = 0.f;
#pragma unroll
      for (int kk = 0; kk < KS; kk += 2) {
        if constexpr (!Q_IN_REGS) {
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            uint32_t b[4];
            load_q(kk, n, b);
            qf[0][n][0] = b[0];
            qf[0][n][1] = b[1];
            qf[1][n][0] = b[2];
            qf[1][n][1] = b[3];
          }
        }
        constexpr int Q0 = Q_IN_REGS ? 1 : 0;
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          uint32_t ka[4], kb[4];
          ldsm4(ks + swz<D>(x * 16 + (lane & 15), 2 * kk + (lane >> 4)), ka);
          ldsm4(ks + swz<D>(x * 16 + (lane & 15), 2 * kk + 2 + (lane >> 4)), kb);
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            mma16816<E>(c[x][n], ka, qf[Q0 * kk][n][0], qf[Q0 * kk][n][1]);
            mma16816<E>(c2[x][n], kb, qf[Q0 * kk + 1][n][0], qf[Q0 * kk + 1][n][1]);
          }
        }
      }
      __syncwarp();
      issue(un + NU<D> - 1);
      // mask and scale; then the tile's maximum, one rescaling of what is there, and the weights
      float top[NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n) top[n][0] = top[n][1] = -INFINITY;
#pragma unroll
      for (int x = 0; x < MT; ++x) {
        const bool whole = seen_by_all(a, t0 + x * 16, t0 + x * 16 + 16, p_lo, p_hi);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int t = t0 + x * 16 + (lane >> 2) + (y >> 1) * 8;
            const float v = c[x][n][y] + c2[x][n][y];
            c[x][n][y] = whole || seen(a, t, pos[n][y & 1]) ? v * a.scale_log2 : -INFINITY;
            top[n][y & 1] = fmaxf(top[n][y & 1], c[x][n][y]);
          }
      }
      bool up = false;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float v = top[n][y];
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
          top[n][y] = fmaxf(below_max<E, 0>(v), m[n][y]);
          up |= top[n][y] != m[n][y];
        }
      if (__any_sync(0xFFFFFFFFu, up)) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float f = top[n][y] == m[n][y] ? 1.f : ex2(m[n][y] - top[n][y]);
            m[n][y] = top[n][y];
            l[n][y] *= f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              acc[j][n][y] *= f;
              acc[j][n][2 + y] *= f;
            }
          }
      }
      uint32_t p[MT][NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float u0 = m[n][0] == -INFINITY ? 0.f : m[n][0], u1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
#pragma unroll
        for (int x = 0; x < MT; ++x) {
          float* e = c[x][n];
          e[0] = ex2(e[0] - u0);
          e[1] = ex2(e[1] - u1);
          e[2] = ex2(e[2] - u0);
          e[3] = ex2(e[3] - u1);
          l[n][0] += e[0] + e[2];
          l[n][1] += e[1] + e[3];
          p[x][n][0] = transpose8(pack2<E>(e[0], e[1]));   // [8 tokens][8 rows] -> the second product's columns
          p[x][n][1] = transpose8(pack2<E>(e[2], e[3]));
        }
      }
      landed();
      const uint32_t vs = smem_u32(ring + (un + 1) % NU<D> * UNIT<D>);
#pragma unroll
      for (int x = 0; x < MT; ++x)
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          uint32_t va[4];
          ldsm4t(vs + swz<D>(x * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * j + ((lane >> 3) & 1)), va);
#pragma unroll
          for (int n = 0; n < NB; ++n) mma16816<E>(acc[j][n], va, p[x][n][0], p[x][n][1]);
        }
      __syncwarp();
      issue(un + NU<D>);
    }
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        l[n][y] += __shfl_xor_sync(0xFFFFFFFFu, l[n][y], 4);
        l[n][y] += __shfl_xor_sync(0xFFFFFFFFu, l[n][y], 8);
        l[n][y] += __shfl_xor_sync(0xFFFFFFFFu, l[n][y], 16);
      }

    // ---- join the warps: their accumulators go through the (now idle) ring
    cp_async_wait_all();
    __syncthreads();
    float* wacc = (float*)(smem + RB * D * 2);                         // [NW][RB][D]
    float2* wml = (float2*)(wacc + NW * RB * D);                        // [NW][RB]
    static_assert((NW + 1) * RB * (D * 4 + 8) <= NW * NU<D> * UNIT<D>, "the join needs the ring");
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int y = 0; y < 4; ++y)
          wacc[(warp * RB + n * 8 + (lane & 3) * 2 + (y & 1)) * D + j * 16 + (lane >> 2) + (y >> 1) * 8] = acc[j][n][y];
    if (lane < 4)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y) wml[warp * RB + n * 8 + lane * 2 + y] = make_float2(m[n][y], l[n][y]);
    __syncthreads();
    const bool whole_item = DIRECT ? cluster == 1 : i0 == 0 && i1 == rg.tiles;
    const int64_t piece = 2 * (int64_t)blockIdx.x + (i0 == 0);
    float* macc = (float*)(wml + NW * RB);                               // [RB][D], of this block (DIRECT)
    float2* mml = (float2*)(macc + RB * D);                              // [RB]
    auto finish = [&](int r, int c, float4 o, float m, float l) {
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const int t = (r0 + r) / a.group, g = (r0 + r) - t * a.group;
      const int64_t row = (s.q0 + t) * a.heads + h * a.group + g;
      *(uint2*)(a.out + row * D + c) = make_uint2(pack2<E>(o.x * inv, o.y * inv), pack2<E>(o.z * inv, o.w * inv));
      if (a.lse && c == 0) a.lse[row] = (m + log2f(l)) * LN2;
    };
    for (int i = tid; i < rows * (D / 4); i += NW * 32) {
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      float m = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, wml[w * RB + r].x);
      const float u = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float2 e = wml[w * RB + r];
        const float f = ex2(e.x - u);
        const float4 x = *(const float4*)(wacc + (w * RB + r) * D + c);
        l += e.y * f;
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
      }
      if (whole_item) {
        finish(r, c, o, m, l);
      } else if (DIRECT) {
        *(float4*)(macc + r * D + c) = o;
        if (c == 0) mml[r] = make_float2(m, l);
      } else {
        *(float4*)(a.acc + (piece * RB + r) * D + c) = o;
        if (c == 0) a.ml[piece * RB + r] = make_float2(m, l);
      }
    }
    if (DIRECT && cluster > 1) {                     // join the cluster's blocks through their shared memory, in rank order
      cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
      cl.sync();
      for (int i = tid * cluster + rank; i < rows * (D / 4); i += NW * 32 * cluster) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k = 0; k < cluster; ++k) m = fmaxf(m, cl.map_shared_rank(mml, k)[r].x);
        const float u = m == -INFINITY ? 0.f : m;
        for (int k = 0; k < cluster; ++k) {
          const float2 e = cl.map_shared_rank(mml, k)[r];
          const float f = ex2(e.x - u);
          const float4 x = *(const float4*)(cl.map_shared_rank(macc, k) + r * D + c);
          l += e.y * f;
          o.x += x.x * f;
          o.y += x.y * f;
          o.z += x.z * f;
          o.w += x.w * f;
        }
        finish(r, c, o, m, l);
      }
      cl.sync();                                     // nobody leaves while another reads its memory
    }
    if (tid == 0) {
      if (s.row < 0) set_err(a.err, SSB_ERR_SEQUENCE);
      if (!DIRECT && i0 == 0 && (!whole_item || a.desc_by_item))
        a.desc[a.desc_by_item ? b * a.kv_heads * nb + item : blockIdx.x] =
            make_int4(whole_item ? -1 : b, item, blockIdx.x | rows << 24, (int)((item0 + rg.tiles - 1) / chunk));
    }
    if (DIRECT) return;
    __syncthreads();
    at = item0 + i1;
  }
}

// Joins the pieces of the items that cross blocks: grid (descriptors, RB), one row per block. Descriptors are one an item
// where those are fewer, else one a block (of the item whose first piece it holds): (sequence or -1, item, first block and
// rows, last block). The pieces are slot 2c + 1 of the first block and the even slots of the blocks after it, summed in that
// order. JT threads: 1024 where items have many pieces.
template <typename E, int D, int ROWS, int JT>
__global__ void __launch_bounds__(JT) k_attn_join(Args a) {
  pdl_wait();
  const int4 d = a.desc[blockIdx.x];
  const int r = blockIdx.y, c0 = d.z & 0xFFFFFF;
  if (d.x < 0 || r >= d.z >> 24) return;
  constexpr int LANES = D / 4, G = JT / LANES;        // threads of a row, groups that share the pieces
  __shared__ float4 part[G][LANES];
  __shared__ float factor[JT], warp_m[JT / 32], warp_l[JT / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = d.w - c0 + 1, c = tid % LANES, g = tid / LANES;
  auto slot = [&](int i) { return (i == 0 ? 2 * (int64_t)c0 + 1 : 2 * (int64_t)(c0 + i)) * ROWS + r; };
  float m = -INFINITY;
  for (int i = tid; i < n; i += JT) m = fmaxf(m, a.ml[slot(i)].x);
  m = warp_max(m);
  if (lane == 0) warp_m[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JT / 32; ++w) m = fmaxf(m, warp_m[w]);
  const float u = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += JT) {
    __syncthreads();
    if (i0 + tid < n) {
      const float2 e = a.ml[slot(i0 + tid)];
      factor[tid] = ex2(e.x - u);
      l += e.y * factor[tid];
    }
    __syncthreads();
    const int k = min(n - i0, JT);
#pragma unroll 8
    for (int i = g; i < k; i += G) {
      const float f = factor[i];
      const float4 x = *(const float4*)(a.acc + slot(i0 + i) * D + c * 4);
      o.x += x.x * f;
      o.y += x.y * f;
      o.z += x.z * f;
      o.w += x.w * f;
    }
  }
  l = warp_sum(l);
  if (lane == 0) warp_l[warp] = l;
  part[g][c] = o;
  __syncthreads();
  if (g) return;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < JT / 32; ++w) l += warp_l[w];
#pragma unroll
  for (int x = 1; x < G; ++x) {
    const float4 y = part[x][c];
    o.x += y.x;
    o.y += y.y;
    o.z += y.z;
    o.w += y.w;
  }
  const Seq s = seq_of(a, d.x);
  const int nb = (s.q * a.group + ROWS - 1) / ROWS, h = d.y / nb, row_in = (d.y - h * nb) * ROWS + r;
  const int t = row_in / a.group, hg = row_in - t * a.group;
  const int64_t row = (s.q0 + t) * a.heads + h * a.group + hg;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  *(uint2*)(a.out + row * D + c * 4) = make_uint2(pack2<E>(o.x * inv, o.y * inv), pack2<E>(o.z * inv, o.w * inv));
  if (a.lse && c == 0) a.lse[row] = (m + log2f(l)) * LN2;
}

int row_blocks() { return ssb_sm_count() * BLOCKS_PER_SM; }

struct Layout {
  int64_t desc, ml, acc, bytes;
};
Layout layout_of(int blocks, int rows, int dim) {
  Layout l;
  l.desc = 0;
  l.ml = ((int64_t)blocks * 16 + 127) / 128 * 128;
  l.acc = l.ml + ((int64_t)2 * blocks * rows * 8 + 127) / 128 * 128;
  l.bytes = l.acc + (int64_t)2 * blocks * rows * dim * 4;
  return l;
}

// Blocks that share an item when each item is taken whole in one launch (0: all tiles split evenly over the GPU, joined by a
// second launch). That saves the second launch and the pieces' way through memory, at the price of an uneven split, so it is
// for items of few tiles, counted from the longest sequence that the table (or the window) allows: clusters grow until a block
// has at most DIRECT_GOOD tiles or the GPU is full; more than DIRECT_MOST tiles a block, or more than DIRECT_WAVES fillings
// of the GPU, go the other way. Device time, whole items against split (16 heads, 2 key heads, head size 256): 16 sequences of
// 1,000 tokens 12.8 against 13.9 us, 64 of 500 19.7 against 22.7, one of 2,000 12.5 against 11.2 (but one launch less, 4 us
// of host time, which a captured call does not have: there the rule loses the 1.3 us); 24 heads, 8 key heads, head size 64,
// 256 sequences of 500: 70 against 59.
constexpr int DIRECT_GOOD = 4, DIRECT_MOST = 8, DIRECT_WAVES = 4;
int tiles_at_most(const Args& a, int tile) {
  int64_t len = (int64_t)a.max_pages * a.page_size;
  if (a.window) {
    const int64_t q = a.starts ? a.rows : a.q_len, seen = (int64_t)a.window + q + a.sinks + 2 * tile;
    len = len < seen ? len : seen;
  }
  return (int)((len + tile - 1) / tile);
}
int direct_cluster(int tiles, int64_t items) {
  int c = 1;
  while (c < 8 && tiles > DIRECT_GOOD * c && items * 2 * c <= row_blocks()) c *= 2;
  return tiles > DIRECT_MOST * c || items * c > (int64_t)DIRECT_WAVES * row_blocks() ? 0 : c;
}
int64_t items_of(const Args& a, int rb) {
  return a.starts ? (a.rows * a.group / rb + a.n) * a.kv_heads
                  : (int64_t)a.n * a.kv_heads * ((a.q_len * a.group + rb - 1) / rb);
}
constexpr int tile_of(int dim) { return NW * (dim == 64 ? TW<64> : dim == 128 ? TW<128> : TW<256>); }

// Items of 8 rows where that holds every row of a key head, else of 16: the second 8 cost registers and instructions.
int rows_per_item(const Args& a) { return a.q_len * a.group <= 8 && !a.starts ? 8 : 16; }

// Prompts go to this kernel too where it takes every item whole and the call is at most SMALL_TILES tiles a block: the
// tcgen05 kernel's plan, tensor maps and 128-row tiles cost more there. Device time, this one against that one: 5 ragged
// prompts of up to 129 tokens (8 heads, 2 key heads, size 64) 7.7 against 20.4 us; one of 256 tokens (32 heads, 8 key heads,
// size 128; 5 tiles a block) 20.9 against 25.3; one of 512 (17 tiles a block) 55 against 37.
constexpr int SMALL_TILES = 8;
bool small_prompt(const Args& a, int dim) {
  const int tiles = tiles_at_most(a, tile_of(dim));
  const int64_t items = items_of(a, 16);
  return direct_cluster(tiles, items) && items * tiles <= (int64_t)SMALL_TILES * row_blocks();
}

int64_t workspace(const Args& a, int dim) {
  if (a.starts && !small_prompt(a, dim)) return prefill_workspace(dim, a.n, a.rows, a.heads, a.kv_heads);
  const int rb = rows_per_item(a);
  return direct_cluster(tiles_at_most(a, tile_of(dim)), items_of(a, rb)) ? 0 : layout_of(row_blocks(), rb, dim).bytes;
}

template <typename E, int D, int RB>
int launch_rows(Args& a, uint8_t* ws, cudaStream_t stream) {
  const int64_t items = items_of(a, RB);
  if (const int c = direct_cluster(tiles_at_most(a, NW * TW<D>), items)) {
    auto kern = k_attn_rows<E, D, RB, true>;
    static std::atomic<uint64_t> done{0};
    if (int rc = ssb_setup_kernel(done, "attn_decode", kern, SMEM<D, RB>)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * c));
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = SMEM<D, RB>;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, c);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return (int)e;
  }
  const int blocks = row_blocks();
  const Layout l = layout_of(blocks, RB, D);
  a.desc = (int4*)(ws + l.desc);
  a.ml = (float2*)(ws + l.ml);
  a.acc = (float*)(ws + l.acc);
  a.desc_by_item = items <= blocks;                   // the split is for decode calls only: the same items a sequence
  auto kern = k_attn_rows<E, D, RB, false>;
  static std::atomic<uint64_t> done{0};
  int rc = ssb_setup_kernel(done, "attn_decode", kern, SMEM<D, RB>);
  if (rc) return rc;
  rc = ssb_launch(kern, dim3(blocks), dim3(NW * 32), SMEM<D, RB>, stream, false, a, 1);
  if (rc) return rc;
  const dim3 grid((unsigned)(a.desc_by_item ? items : blocks), RB);
  if (items * 8 <= blocks) return ssb_launch(k_attn_join<E, D, RB, 1024>, grid, dim3(1024), 0, stream, true, a);
  return ssb_launch(k_attn_join<E, D, RB, 256>, grid, dim3(256), 0, stream, true, a);
}

template <typename E>
int launch_dim(Args& a, int dim, uint8_t* ws, cudaStream_t st) {
  const bool few = rows_per_item(a) == 8;
  if (dim == 64) return few ? launch_rows<E, 64, 8>(a, ws, st) : launch_rows<E, 64, 16>(a, ws, st);
  if (dim == 128) return few ? launch_rows<E, 128, 8>(a, ws, st) : launch_rows<E, 128, 16>(a, ws, st);
  return few ? launch_rows<E, 256, 8>(a, ws, st) : launch_rows<E, 256, 16>(a, ws, st);
}

int launch_checked(Args& a, int dim, bool bf16, void* ws, int64_t ws_bytes, void* stream) {
  const int64_t need = workspace(a, dim);
  SSB_CHECK_ARG(need == 0 || (ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= need));
  if (a.starts && !small_prompt(a, dim)) return prefill_launch(a, dim, bf16, ws, stream);
  return bf16 ? launch_dim<__nv_bfloat16>(a, dim, (uint8_t*)ws, (cudaStream_t)stream)
              : launch_dim<__half>(a, dim, (uint8_t*)ws, (cudaStream_t)stream);
}

// t / d = (mulhi(t, mul) + t) >> shift for t < 2^31 (round-up reciprocal of a 32-bit division).
void reciprocal(int32_t d, uint32_t* mul, uint32_t* shift) {
  uint32_t s = 0;
  while ((1ull << s) < (uint64_t)d) ++s;
  *shift = s;
  *mul = (uint32_t)(((1ull << 32) * ((1ull << s) - (uint64_t)d)) / (uint64_t)d + 1);
}

// Checks and the fields that both entry points share.
int fill(Args& a, const ssb_attn_args& x) {
  SSB_CHECK_ARG(x.type == SSB_BF16 || x.type == SSB_F16);
  SSB_CHECK_ARG(x.n >= 0 && x.heads > 0 && x.kv_heads > 0 && x.heads % x.kv_heads == 0 && x.page_size > 0 && x.pages > 0 &&
                x.table_rows > 0 && x.max_pages > 0 && x.window >= 0 && x.sinks >= 0 && x.scale > 0.f && x.scale <= 3.4e38f);
  SSB_CHECK_ARG((int64_t)x.max_pages * x.page_size <= 0x7FFFFFFFll - 1024 && x.sinks <= 0x7FFFFFFF - 1024);
  if (x.dim != 64 && x.dim != 128 && x.dim != 256) return SSB_EUNSUPPORTED;
  SSB_CHECK_ARG((x.page_stride | x.head_stride | x.token_stride | x.q_tok_stride | x.q_head_stride) % 8 == 0);
  SSB_CHECK_ARG((((uintptr_t)x.q | (uintptr_t)x.k | (uintptr_t)x.v | (uintptr_t)x.out) & 15) == 0);
  a.q = (const uint16_t*)x.q;
  a.q_tok = x.q_tok_stride;
  a.q_head = x.q_head_stride;
  a.k = (const uint16_t*)x.k;
  a.v = (const uint16_t*)x.v;
  a.sp = x.page_stride;
  a.sh = x.head_stride;
  a.st = x.token_stride;
  a.n = x.n;
  a.heads = x.heads;
  a.kv_heads = x.kv_heads;
  a.group = x.heads / x.kv_heads;
  a.page_size = x.page_size;
  a.pages = x.pages;
  a.table = x.table;
  a.table_rows = x.table_rows;
  a.max_pages = x.max_pages;
  a.lengths = x.lengths;
  a.ids = x.ids;
  a.window = x.window;
  a.sinks = x.window ? x.sinks : 0;
  a.scale_log2 = x.scale * 1.4426950408889634f;
  a.out = (uint16_t*)x.out;
  a.lse = x.lse;
  a.err = x.err;
  reciprocal(x.page_size, &a.page_mul, &a.page_shift);
  reciprocal(a.group, &a.group_mul, &a.group_shift);
  return SSB_OK;
}

}  // namespace
}  // namespace attn

using namespace attn;

extern "C" int ssb_attn_workspace(const ssb_attn_args* x, int32_t prefill, int64_t* bytes) {
  SSB_CHECK_ARG(x && bytes && x->n >= 0 && x->kv_heads > 0 && x->heads > 0 && x->heads % x->kv_heads == 0);
  SSB_CHECK_ARG(x->page_size > 0 && x->max_pages > 0 && x->window >= 0 && x->sinks >= 0 && x->rows >= 0 && x->q_len >= 0);
  if (x->dim != 64 && x->dim != 128 && x->dim != 256) return SSB_EUNSUPPORTED;
  Args a = {};
  a.n = x->n;
  a.heads = x->heads;
  a.kv_heads = x->kv_heads;
  a.group = x->heads / x->kv_heads;
  a.page_size = x->page_size;
  a.max_pages = x->max_pages;
  a.window = x->window;
  a.sinks = x->window ? x->sinks : 0;
  const int32_t some = 0;
  if (prefill) a.starts = &some;                     // only whether there are any matters here
  else a.q_len = x->q_len;
  a.rows = prefill ? x->rows : (int64_t)x->n * x->q_len;
  SSB_CHECK_ARG(a.rows * a.group < (1ll << 30));
  *bytes = a.n && a.rows ? workspace(a, x->dim) : 0;
  return SSB_OK;
}

extern "C" int ssb_attn_decode(const ssb_attn_args* x, void* stream) {
  Args a = {};
  SSB_CHECK_ARG(x);
  if (int rc = fill(a, *x)) return rc;
  SSB_CHECK_ARG(x->q_len >= 0 && x->q_seq_stride % 8 == 0);
  if ((int64_t)x->q_len * a.group > 128) return SSB_EUNSUPPORTED;
  a.rows = (int64_t)x->n * x->q_len;
  SSB_CHECK_ARG(a.rows * a.group < (1ll << 30));
  if (a.rows == 0) return SSB_OK;
  SSB_CHECK_ARG(x->q && x->k && x->v && x->table && x->lengths && x->out);
  a.q_seq = x->q_seq_stride;
  a.q_len = x->q_len;
  return launch_checked(a, x->dim, x->type == SSB_BF16, x->ws, x->ws_bytes, stream);
}

extern "C" int ssb_attn_prefill(const ssb_attn_args* x, void* stream) {
  Args a = {};
  SSB_CHECK_ARG(x);
  if (int rc = fill(a, *x)) return rc;
  SSB_CHECK_ARG(x->rows >= 0 && x->rows * a.group < (1ll << 30));
  if (x->n == 0 || x->rows == 0) return SSB_OK;
  SSB_CHECK_ARG(x->q && x->k && x->v && x->table && x->lengths && x->starts && x->out);
  a.starts = x->starts;
  a.rows = x->rows;
  return launch_checked(a, x->dim, x->type == SSB_BF16, x->ws, x->ws_bytes, stream);
}
