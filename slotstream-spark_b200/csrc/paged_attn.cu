// Attention over the paged key-value cache for few query rows per key head: decode steps and speculative verifies.
//
// Per item (sequence, key head, block of RB query rows): s = q k^T, online softmax (running maximum and sum, fp32,
// log2 domain), o = p v. The rows of one key head -- query tokens x heads of its group -- share every key and value
// read, so each cached byte is read once per key head: the kernel is bound by reading the cache. Tensor cores
// (mma.sync m16n8k16, fp32 accumulation) do both products, since RB x D x 2 multiply-adds per cached element pair
// would otherwise take more issue slots than the loads leave; tcgen05's 128-row tiles would be mostly padding here.
//
// A block has NW warps that work alone: each walks every NW-th sub-tile of TW tokens through its own ring of NS
// cp.async stages (no block barrier inside an item), and the warps' (max, sum, accumulator) are joined through shared
// memory at the end of the item. p is rounded to the inputs' type for the second product (relative 2^-8 for bf16,
// 2^-11 for fp16, as the library's other tensor-core inputs); its sum is taken before the rounding, in fp32.
#include "paged_attn.cuh"

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

constexpr int NW = 4, RB = 16, NS = 3;
template <int D>
constexpr int TW = D == 64 ? 32 : 16;
template <int D>
constexpr int STAGE = TW<D> * D * 2 * 2;          // keys and values of one sub-tile
template <int D>
constexpr int SMEM = RB * D * 2 + NW * NS * STAGE<D>;
template <int D>
constexpr int BLOCKS_PER_SM = D == 256 ? 1 : 2;

template <typename E, int D>
__global__ void __launch_bounds__(NW * 32, BLOCKS_PER_SM<D>) k_attn_rows(Args a) {
  constexpr int T = NW * TW<D>, CPR = D / 8;       // tokens of a tile, 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scan[NW + 1];
  __shared__ long long plan[3];                    // chunk, then the item where this block starts: its start, b
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* sq = smem;
  uint8_t* ring = smem + RB * D * 2 + warp * NS * STAGE<D>;
  pdl_wait();

  // ---- this block's share: tiles of all sequences, divided evenly
  auto tiles_of = [&](int b, int* items, int* tiles) {
    const Seq s = seq_of(a, b);
    *items = a.kv_heads * ((s.q * a.group + RB - 1) / RB);
    *tiles = range_of(a, s.len - s.q, s.len - 1, T).tiles;
  };
  long long mine = 0;
  for (int b = tid; b < a.n; b += NW * 32) {
    int items, tiles;
    tiles_of(b, &items, &tiles);
    mine += (long long)items * tiles;
  }
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
  if (lane == 0) scan[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    long long t = 0;
    for (int w = 0; w < NW; ++w) t += scan[w];
    const long long ch = (t + gridDim.x - 1) / gridDim.x;
    plan[0] = ch < 2 ? 2 : ch;
    plan[1] = t;
    a.desc[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
  __syncthreads();
  const long long chunk = plan[0], total = plan[1];
  const long long lo = chunk * blockIdx.x, hi = min(lo + chunk, total);
  if (lo >= hi) return;
  // the sequence that holds tile `lo`
  int b = 0;
  long long begin = 0;
  for (int b0 = 0;; b0 += NW * 32) {
    int items = 0, tiles = 0;
    if (b0 + tid < a.n) tiles_of(b0 + tid, &items, &tiles);
    long long w = (long long)items * tiles, inc = w;
    for (int o = 1; o < 32; o <<= 1) {
      long long u = __shfl_up_sync(0xFFFFFFFFu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) scan[warp] = inc;
    if (tid == 0) scan[NW] = -1;
    __syncthreads();
    long long pre = begin;
    for (int v = 0; v < warp; ++v) pre += scan[v];
    if (lo >= pre + inc - w && lo < pre + inc) {
      plan[1] = pre + inc - w;
      scan[NW] = b0 + tid;
    }
    __syncthreads();
    if (scan[NW] >= 0) {
      b = (int)scan[NW];
      begin = plan[1];
      break;
    }
    for (int v = 0; v < NW; ++v) begin += scan[v];
    __syncthreads();
  }

  long long at = lo;
  Seq s = seq_of(a, b);
  while (at < hi) {
    const Range rg = range_of(a, s.len - s.q, s.len - 1, T);
    const int nb = (s.q * a.group + RB - 1) / RB;
    const long long weight = (long long)a.kv_heads * nb * rg.tiles;
    if (at >= begin + weight) {
      begin += weight;
      s = seq_of(a, ++b);
      continue;
    }
    // ---- one item, or the part of it inside this block
    const int item = (int)((at - begin) / rg.tiles), h = item / nb, rb = item - h * nb;
    const long long item0 = begin + (long long)item * rg.tiles;
    const int i0 = (int)(at - item0), i1 = (int)min((long long)rg.tiles, hi - item0);
    const int r0 = rb * RB, rows = min(RB, s.q * a.group - r0);
    const int p_first = s.len - s.q, p_lo = p_first + r0 / a.group, p_hi = p_first + (r0 + rows - 1) / a.group;

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
    auto issue = [&](int i, int slot) {
      uint8_t* st = ring + slot * STAGE<D>;
      const int t0 = tile_token(rg, i, T) + warp * TW<D>;
      long long mine_off = lane < TW<D> ? offset_of(t0 + lane) : -1;
#pragma unroll
      for (int u = 0; u < TW<D> * CPR / 32; ++u) {
        const int r = (u * 32 + lane) / CPR, c = (u * 32 + lane) % CPR;
        const long long off = __shfl_sync(0xFFFFFFFFu, mine_off, r);
        const uint32_t n = off < 0 ? 0 : 16;
        const uint16_t* src = kh + (off < 0 ? 0 : off) + c * 8;
        const uint16_t* srv = vh + (off < 0 ? 0 : off) + c * 8;
        cp_async16(smem_u32(st) + swz<D>(r, c), src, n);
        cp_async16(smem_u32(st) + STAGE<D> / 2 + swz<D>(r, c), srv, n);
      }
    };

    float acc[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const int ra = lane >> 2, rb8 = ra + 8;
    // rows past the item's last have zero queries and are never written: they take the last one's position
    const int pa = p_first + (r0 + min(ra, rows - 1)) / a.group, pb = p_first + (r0 + min(rb8, rows - 1)) / a.group;

#pragma unroll
    for (int u = 0; u < NS - 1; ++u) {
      if (i0 + u < i1) issue(i0 + u, u);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    for (int i = i0; i < i1; ++i) {
      const int slot = (i - i0) % NS;
      asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
      __syncwarp();
      const uint32_t ks = smem_u32(ring + slot * STAGE<D>), vs = ks + STAGE<D> / 2;
      const int t0 = tile_token(rg, i, T) + warp * TW<D>;
#pragma unroll
      for (int hf = 0; hf < TW<D> / 16; ++hf) {
        float c[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t qa[4], kb[4];
          ldsm4(smem_u32(sq) + swz<D>(lane & 15, 2 * kk + (lane >> 4)), qa);
          ldsm4(ks + swz<D>(hf * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)), kb);
          mma16816<E>(c[0], qa, kb[0], kb[1]);
          mma16816<E>(c[1], qa, kb[2], kb[3]);
        }
        const int t1 = t0 + hf * 16;
        const bool whole = seen_by_all(a, t1, t1 + 16, p_lo, p_hi);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int t = t1 + x * 8 + (lane & 3) * 2 + y;
            c[x][y] = whole || seen(a, t, pa) ? c[x][y] * a.scale_log2 : -INFINITY;
            c[x][2 + y] = whole || seen(a, t, pb) ? c[x][2 + y] * a.scale_log2 : -INFINITY;
          }
        float ma = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1]));
        float mb = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
        ma = fmaxf(ma, __shfl_xor_sync(0xFFFFFFFFu, ma, 1));
        mb = fmaxf(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, 1));
        ma = fmaxf(m0, fmaxf(ma, __shfl_xor_sync(0xFFFFFFFFu, ma, 2)));
        mb = fmaxf(m1, fmaxf(mb, __shfl_xor_sync(0xFFFFFFFFu, mb, 2)));
        if (__any_sync(0xFFFFFFFFu, ma != m0 || mb != m1)) {
          const float fa = ma == m0 ? 1.f : ex2(m0 - ma), fb = mb == m1 ? 1.f : ex2(m1 - mb);
          l0 *= fa;
          l1 *= fb;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            acc[j][0] *= fa;
            acc[j][1] *= fa;
            acc[j][2] *= fb;
            acc[j][3] *= fb;
          }
          m0 = ma;
          m1 = mb;
        }
        const float ua = m0 == -INFINITY ? 0.f : m0, ub = m1 == -INFINITY ? 0.f : m1;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          c[x][0] = ex2(c[x][0] - ua);
          c[x][1] = ex2(c[x][1] - ua);
          c[x][2] = ex2(c[x][2] - ub);
          c[x][3] = ex2(c[x][3] - ub);
          l0 += c[x][0] + c[x][1];
          l1 += c[x][2] + c[x][3];
        }
        const uint32_t p[4] = {pack2<E>(c[0][0], c[0][1]), pack2<E>(c[0][2], c[0][3]), pack2<E>(c[1][0], c[1][1]),
                               pack2<E>(c[1][2], c[1][3])};
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t vb[4];
          ldsm4t(vs + swz<D>(hf * 16 + (lane & 15), 2 * j + (lane >> 4)), vb);
          mma16816<E>(acc[2 * j], p, vb[0], vb[1]);
          mma16816<E>(acc[2 * j + 1], p, vb[2], vb[3]);
        }
      }
      __syncwarp();
      if (i + NS - 1 < i1) issue(i + NS - 1, (i - i0 + NS - 1) % NS);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 1);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 1);
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, 2);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, 2);

    // ---- join the warps: their accumulators go through the (now idle) ring
    cp_async_wait_all();
    __syncthreads();
    float* wacc = (float*)(smem + RB * D * 2);                         // [NW][RB][D]
    float2* wml = (float2*)(wacc + NW * RB * D);                        // [NW][RB]
    static_assert(NW * RB * D * 4 + NW * RB * 8 <= NW * NS * STAGE<D>, "the join needs the ring");
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      *(float2*)(wacc + (warp * RB + ra) * D + j * 8 + (lane & 3) * 2) = make_float2(acc[j][0], acc[j][1]);
      *(float2*)(wacc + (warp * RB + rb8) * D + j * 8 + (lane & 3) * 2) = make_float2(acc[j][2], acc[j][3]);
    }
    if ((lane & 3) == 0) {
      wml[warp * RB + ra] = make_float2(m0, l0);
      wml[warp * RB + rb8] = make_float2(m1, l1);
    }
    __syncthreads();
    const bool whole_item = i0 == 0 && i1 == rg.tiles;
    const int64_t piece = 2 * (int64_t)blockIdx.x + (i0 == 0);
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
        const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
        const int t = (r0 + r) / a.group, g = (r0 + r) - t * a.group;
        const int64_t row = (s.q0 + t) * a.heads + h * a.group + g;
        *(uint2*)(a.out + row * D + c) = make_uint2(pack2<E>(o.x * inv, o.y * inv), pack2<E>(o.z * inv, o.w * inv));
        if (a.lse && c == 0) a.lse[row] = (m + log2f(l)) * LN2;
      } else {
        *(float4*)(a.acc + (piece * RB + r) * D + c) = o;
        if (c == 0) a.ml[piece * RB + r] = make_float2(m, l);
      }
    }
    if (tid == 0) {
      if (s.row < 0) set_err(a.err, SSB_ERR_SEQUENCE);
      if (i0 == 0 && !whole_item)
        a.desc[blockIdx.x] = make_int4(b, item, (int)((item0 + rg.tiles - 1) / chunk), rows);
    }
    __syncthreads();
    at = item0 + i1;
  }
}

// Joins the pieces of the items that cross blocks: grid (blocks of the first kernel, RB), one row per block; desc[c] =
// (sequence, item, last block, rows) when block c holds an item's first piece. Its pieces are slot 2c + 1 and the even
// slots of the blocks after c, summed in that order.
template <typename E, int D, int ROWS>
__global__ void __launch_bounds__(128) k_attn_join(Args a) {
  pdl_wait();
  const int4 d = a.desc[blockIdx.x];
  const int r = blockIdx.y;
  if (d.x < 0 || r >= d.w) return;
  constexpr int LANES = D / 4, G = 128 / LANES;       // threads of a row, groups that share the pieces
  __shared__ float4 part[G][LANES];
  __shared__ float2 pml[G];
  const int c0 = blockIdx.x, n = d.z - c0 + 1, c = threadIdx.x % LANES, g = threadIdx.x / LANES;
  auto slot = [&](int i) { return (i == 0 ? 2 * (int64_t)c0 + 1 : 2 * (int64_t)(c0 + i)) * ROWS + r; };
  float m = -INFINITY;
  for (int i = 0; i < n; ++i) m = fmaxf(m, a.ml[slot(i)].x);
  const float u = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = g; i < n; i += G) {
    const float2 e = a.ml[slot(i)];
    const float f = ex2(e.x - u);
    const float4 x = *(const float4*)(a.acc + slot(i) * D + c * 4);
    l += e.y * f;
    o.x += x.x * f;
    o.y += x.y * f;
    o.z += x.z * f;
    o.w += x.w * f;
  }
  part[g][c] = o;
  if (c == 0) pml[g] = make_float2(l, 0.f);
  __syncthreads();
  if (g) return;
  for (int x = 1; x < G; ++x) {
    const float4 y = part[x][c];
    l += pml[x].x;
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

int sm_count() {
  int dev = 0, sms = 148;
  cudaGetDevice(&dev);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

int blocks_of(int dim) { return sm_count() * (dim == 256 ? BLOCKS_PER_SM<256> : BLOCKS_PER_SM<128>); }

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

template <typename E, int D>
int launch_rows(Args& a, uint8_t* ws, cudaStream_t stream) {
  const int blocks = blocks_of(D);
  const Layout l = layout_of(blocks, RB, D);
  a.desc = (int4*)(ws + l.desc);
  a.ml = (float2*)(ws + l.ml);
  a.acc = (float*)(ws + l.acc);
  auto kern = k_attn_rows<E, D>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM<D>);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return (int)e;
  }
  ssb_note_smem("attn_decode", kern, SMEM<D>);
  int rc = ssb_launch(kern, dim3(blocks), dim3(NW * 32), SMEM<D>, stream, false, a);
  if (rc) return rc;
  return ssb_launch(k_attn_join<E, D, RB>, dim3(blocks, RB), dim3(128), 0, stream, true, a);
}

template <typename E>
int launch_dim(Args& a, int dim, uint8_t* ws, cudaStream_t st) {
  if (dim == 64) return launch_rows<E, 64>(a, ws, st);
  if (dim == 128) return launch_rows<E, 128>(a, ws, st);
  return launch_rows<E, 256>(a, ws, st);
}

// t / d = (mulhi(t, mul) + t) >> shift for t < 2^31 (round-up reciprocal of a 32-bit division).
void reciprocal(int32_t d, uint32_t* mul, uint32_t* shift) {
  uint32_t s = 0;
  while ((1ull << s) < (uint64_t)d) ++s;
  *shift = s;
  *mul = (uint32_t)(((1ull << 32) * ((1ull << s) - (uint64_t)d)) / (uint64_t)d + 1);
}

// Checks and the fields that both entry points share.
int fill(Args& a, const void* q, int32_t q_type, const void* k, const void* v, int64_t page_stride,
         int64_t head_stride, int64_t token_stride, int32_t n, int32_t heads, int32_t kv_heads, int32_t dim,
         int32_t page_size, int32_t pages, const int32_t* table, int32_t table_rows, int32_t max_pages,
         const int32_t* lengths, const int32_t* ids, int32_t window, int32_t sinks, float scale, void* out, float* lse,
         int32_t* err) {
  SSB_CHECK_ARG(q_type == SSB_BF16 || q_type == SSB_F16);
  SSB_CHECK_ARG(n >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && page_size > 0 && pages > 0 &&
                table_rows > 0 && max_pages > 0 && window >= 0 && sinks >= 0 && scale > 0.f && scale <= 3.4e38f);
  SSB_CHECK_ARG((int64_t)max_pages * page_size <= 0x7FFFFFFFll - 1024 && sinks <= 0x7FFFFFFF - 1024);
  if (dim != 64 && dim != 128 && dim != 256) return SSB_EUNSUPPORTED;
  SSB_CHECK_ARG((page_stride | head_stride | token_stride) % 8 == 0);
  SSB_CHECK_ARG((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15) == 0);
  a.q = (const uint16_t*)q;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.sp = page_stride;
  a.sh = head_stride;
  a.st = token_stride;
  a.n = n;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.group = heads / kv_heads;
  a.page_size = page_size;
  a.pages = pages;
  a.table = table;
  a.table_rows = table_rows;
  a.max_pages = max_pages;
  a.lengths = lengths;
  a.ids = ids;
  a.window = window;
  a.sinks = window ? sinks : 0;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  a.lse = lse;
  a.err = err;
  reciprocal(page_size, &a.page_mul, &a.page_shift);
  reciprocal(a.group, &a.group_mul, &a.group_shift);
  return SSB_OK;
}

}  // namespace
}  // namespace attn

using namespace attn;

static int64_t workspace(int dim, int n, int64_t rows, int heads, int kv_heads, bool prefill) {
  return prefill ? prefill_workspace(dim, n, rows, heads, kv_heads) : layout_of(blocks_of(dim), RB, dim).bytes;
}

extern "C" int ssb_attn_workspace(int32_t dim, int32_t n, int64_t rows, int32_t heads, int32_t kv_heads,
                                  int32_t prefill, int64_t* bytes) {
  SSB_CHECK_ARG(bytes && n >= 0 && rows >= 0 && kv_heads > 0 && heads > 0 && heads % kv_heads == 0);
  SSB_CHECK_ARG(rows * (heads / kv_heads) < (1ll << 30));
  if (dim != 64 && dim != 128 && dim != 256) return SSB_EUNSUPPORTED;
  *bytes = workspace(dim, n, rows, heads, kv_heads, prefill != 0);
  return SSB_OK;
}

extern "C" int ssb_attn_decode(const void* q, int32_t q_type, int64_t q_seq_stride, int64_t q_tok_stride,
                               int64_t q_head_stride, const void* k, const void* v, int64_t page_stride,
                               int64_t head_stride, int64_t token_stride, int32_t n, int32_t q_len, int32_t heads,
                               int32_t kv_heads, int32_t dim, int32_t page_size, int32_t pages, const int32_t* table,
                               int32_t table_rows, int32_t max_pages, const int32_t* lengths, const int32_t* ids,
                               int32_t window, int32_t sinks, float scale, void* out, float* lse, void* ws,
                               int64_t ws_bytes, int32_t* err, void* stream) {
  Args a = {};
  if (int rc = fill(a, q, q_type, k, v, page_stride, head_stride, token_stride, n, heads, kv_heads, dim, page_size,
                    pages, table, table_rows, max_pages, lengths, ids, window, sinks, scale, out, lse, err))
    return rc;
  SSB_CHECK_ARG(q_len >= 0 && (q_seq_stride | q_tok_stride | q_head_stride) % 8 == 0);
  if ((int64_t)q_len * (heads / kv_heads) > 128) return SSB_EUNSUPPORTED;
  if (n == 0 || q_len == 0) return SSB_OK;
  SSB_CHECK_ARG(q && k && v && table && lengths && out && ws);
  SSB_CHECK_ARG(((uintptr_t)ws & 15) == 0 && ws_bytes >= layout_of(blocks_of(dim), RB, dim).bytes);
  a.q_seq = q_seq_stride;
  a.q_tok = q_tok_stride;
  a.q_head = q_head_stride;
  a.q_len = q_len;
  a.rows = (int64_t)n * q_len;
  return q_type == SSB_BF16 ? launch_dim<__nv_bfloat16>(a, dim, (uint8_t*)ws, (cudaStream_t)stream)
                            : launch_dim<__half>(a, dim, (uint8_t*)ws, (cudaStream_t)stream);
}

extern "C" int ssb_attn_prefill(const void* q, int32_t q_type, int64_t q_tok_stride, int64_t q_head_stride,
                                const void* k, const void* v, int64_t page_stride, int64_t head_stride,
                                int64_t token_stride, int64_t rows, const int32_t* starts, int32_t n, int32_t heads,
                                int32_t kv_heads, int32_t dim, int32_t page_size, int32_t pages, const int32_t* table,
                                int32_t table_rows, int32_t max_pages, const int32_t* lengths, const int32_t* ids,
                                int32_t window, int32_t sinks, float scale, void* out, float* lse, void* ws,
                                int64_t ws_bytes, int32_t* err, void* stream) {
  Args a = {};
  if (int rc = fill(a, q, q_type, k, v, page_stride, head_stride, token_stride, n, heads, kv_heads, dim, page_size,
                    pages, table, table_rows, max_pages, lengths, ids, window, sinks, scale, out, lse, err))
    return rc;
  SSB_CHECK_ARG(rows >= 0 && rows * (heads / kv_heads) < (1ll << 30) && (q_tok_stride | q_head_stride) % 8 == 0);
  if (n == 0 || rows == 0) return SSB_OK;
  SSB_CHECK_ARG(q && k && v && table && lengths && starts && out && ws);
  SSB_CHECK_ARG(((uintptr_t)ws & 15) == 0 && ws_bytes >= workspace(dim, n, rows, heads, kv_heads, true));
  a.q_tok = q_tok_stride;
  a.q_head = q_head_stride;
  a.starts = starts;
  a.rows = rows;
  return prefill_launch(a, dim, q_type == SSB_BF16, ws, stream);
}
