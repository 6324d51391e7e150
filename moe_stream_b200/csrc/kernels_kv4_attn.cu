// kernels_kv4_attn.cu — attention of the newest tokens of each sequence over the paged 4-bit K/V cache.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  k, v = o + d (16 + c) per 32 dims
//
// Bound by memory: each (token, kv head) is 1.25 head_dim bytes that are read once, for all query heads of the
// group and all query tokens (the rows).  One row tile holds 8 NT rows.
//
// Work.  A job is (sequence, kv head, row tile); its keys are cut into tiles of TT = 4096 / head_dim tokens (5 KB).
// The tiles of all jobs form one list that is cut into equal ranges, one per block, so sequences of any
// lengths fill the GPU without the host knowing them.  The 4 warps of a block take the tiles of a range in
// turn, each with its own ring of two stages filled by bulk copies, its own running maximum and sum; they are
// joined at the end of a job's part.  A job inside one range is finished there; the others leave their
// numerators and sums in the workspace, which a second kernel joins.
//
// Scores (keys x rows, m16n8k16): a code is turned into the number 16 + c by one shift and one mask-and-or, so
// per group of 32 dims the product of q and (16 + c) is exact in the tensor core's f32, and
//   s += d P + o Q,  P = sum q (16 + c),  Q = sum q
// in f32.  Values: v = fma(16 + c, d, o) in f16 pairs of two keys, the probabilities in f16 (bf16 would
// cost 8 times their rounding) transposed by movmatrix from the score layout.  The running maximum is raised
// only when a score exceeds it by more than 2^8: then p <= 256 stays far inside f16.
#include <math_constants.h>

#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"

namespace ms {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStages = 2;
constexpr int kTileBytes = 5120;          // 16 * 20 * 16 for every head_dim
// blocks of an SM: 3 leave 168 registers a thread; 256 dims, or 16 rows of 128, need more than that
__host__ __device__ constexpr int blocks_per_sm(int hd, int nt) { return hd * nt >= 256 ? 2 : 3; }
constexpr int kMinTiles = kWarps;         // tiles of a range at least: one per warp
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;            // scores (log2) above the running maximum that are let through

// ---- the list of tiles ----
struct Plan {
  int jobs;          // of one sequence: kv heads x row tiles
  int row_tiles;
  int64_t total;     // tiles of all jobs
  int64_t chunk;     // tiles of one block's range
};
struct SeqTiles {
  int len;           // tokens (checked)
  int lo;            // first key of any query
  int first;         // index of the first tile
  int n;             // tiles of one job, at least 1 (a sequence without tokens still gets its zeros)
};
template <int TT>
__device__ __forceinline__ SeqTiles seq_tiles(const ms_kv4_cache& c, const ms_kv4_attn& a, int seq) {
  SeqTiles s;
  const int len = a.lens[seq], cap = c.max_pages * c.page_tokens;
  s.len = len < 0 ? 0 : min(len, cap);
  s.lo = a.window > 0 ? max(0, s.len - a.n_query - a.window + 1) : 0;   // the first query's first key
  s.first = s.lo / TT;
  s.n = max(1, (s.len + TT - 1) / TT - s.first);
  return s;
}
// whole warp: the plan, and (before >= 0) the tiles of the jobs of the sequences in front of `before`
template <int TT>
__device__ __forceinline__ Plan make_plan(const ms_kv4_cache& c, const ms_kv4_attn& a, int row_tiles, int ranges, int before,
                                          int64_t* in_front) {
  const int lane = threadIdx.x & 31;
  int64_t all = 0, front = 0;
  for (int i = lane; i < c.n_seqs; i += 32) {
    const int n = seq_tiles<TT>(c, a, i).n;
    all += n;
    if (i < before) front += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    front += __shfl_xor_sync(0xffffffffu, front, o);
  }
  Plan p;
  p.row_tiles = row_tiles;
  p.jobs = c.kv_heads * row_tiles;
  p.total = all * p.jobs;
  p.chunk = max((int64_t)kMinTiles, (p.total + ranges - 1) / ranges);
  *in_front = front * p.jobs;
  return p;
}
// whole warp: the sequence that tile u of the list belongs to, and the first tile of that sequence
template <int TT>
__device__ __forceinline__ int find_seq(const ms_kv4_cache& c, const ms_kv4_attn& a, const Plan& p, int64_t u, int64_t* base) {
  const int lane = threadIdx.x & 31;
  int64_t at = 0;
  for (int b = 0; b < c.n_seqs; b += 32) {
    const int64_t n = b + lane < c.n_seqs ? (int64_t)seq_tiles<TT>(c, a, b + lane).n * p.jobs : 0;
    int64_t inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, u < at + inc);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *base = at + __shfl_sync(0xffffffffu, inc - n, l);
      return b + l;
    }
    at += __shfl_sync(0xffffffffu, inc, 31);
  }
  *base = at;
  return c.n_seqs;
}

// partial of one block and one of its two cut jobs: [rows][HD] numerators, then m and l of the rows
template <int HD, int ROWS>
__host__ __device__ constexpr int partial_floats() { return ROWS * HD + 2 * ROWS; }

// ---- tensor-core pieces ----
template <class T>
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// pair n of a word (nibbles at bits 4 n and 4 n + 16) as the two numbers 16 + c: the code in the top bits
// of the mantissa of 16.0
template <class T, int N>
__device__ __forceinline__ uint32_t codes2(uint32_t w);
#define MS_CODES2(T, N, SHIFTED, MASK, BASE) \
  template <>                                \
  __device__ __forceinline__ uint32_t codes2<T, N>(uint32_t w) { return ((SHIFTED) & MASK) | BASE; }
MS_CODES2(__half, 0, w << 6, 0x03C003C0u, 0x4C004C00u)
MS_CODES2(__half, 1, w << 2, 0x03C003C0u, 0x4C004C00u)
MS_CODES2(__half, 2, w >> 2, 0x03C003C0u, 0x4C004C00u)
MS_CODES2(__half, 3, w >> 6, 0x03C003C0u, 0x4C004C00u)
MS_CODES2(__nv_bfloat16, 0, w << 3, 0x00780078u, 0x41804180u)
MS_CODES2(__nv_bfloat16, 1, w >> 1, 0x00780078u, 0x41804180u)
MS_CODES2(__nv_bfloat16, 2, w >> 5, 0x00780078u, 0x41804180u)
MS_CODES2(__nv_bfloat16, 3, w >> 9, 0x00780078u, 0x41804180u)
#undef MS_CODES2

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <int HD, int NT>
struct Smem {
  static constexpr int kPitch = HD + 4;   // floats between rows of the joining buffer
  alignas(128) uint8_t stage[kWarps][kStages][kTileBytes];
  alignas(16) float o[kWarps][8 * NT][kPitch];
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  uint64_t full[kWarps][kStages];
  uint32_t have[kWarps][kStages];         // blocks of the tile that were copied
};

template <class T, int HD, int NT>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(HD, NT)) kv4_attn_kernel(const ms_kv4_cache c, const ms_kv4_attn a, int row_tiles,
                                                                        uint32_t* err) {
  constexpr int G = HD / 32, TB = 256 / HD, TT = 16 * TB, BLK = 20 * HD, ROWS = 8 * NT;
  constexpr int MT = HD / 16;              // 16-row tiles of the value product
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<HD, NT>& sm = *reinterpret_cast<Smem<HD, NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  pdl_launch_dependents();
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  int64_t unused;
  const Plan plan = make_plan<TT>(c, a, row_tiles, gridDim.x, 0, &unused);
  const int64_t u0 = (int64_t)blockIdx.x * plan.chunk, u1 = min(u0 + plan.chunk, plan.total);
  if (u0 >= u1) return;
  const int rep = a.heads / c.kv_heads, rows = a.n_query * rep;
  const float c2 = a.scale * kLog2e;

  // ---- the ring: tiles u0 + warp, + kWarps, ... ----
  struct Cursor {
    int seq;
    int64_t base;    // first tile of the sequence
    SeqTiles s;
  };
  Cursor pre;
  pre.seq = find_seq<TT>(c, a, plan, u0, &pre.base);
  pre.s = seq_tiles<TT>(c, a, pre.seq);
  Cursor cur = pre;
  auto seek = [&](Cursor& k, int64_t u) {
    while (u >= k.base + (int64_t)k.s.n * plan.jobs) {
      k.base += (int64_t)k.s.n * plan.jobs;
      ++k.seq;
      k.s = seq_tiles<TT>(c, a, k.seq);
    }
  };
  const int per_page = max(1, c.page_tokens / TT), pages = max(1, TT / c.page_tokens);   // tiles of a page / pages of a tile
  auto fetch = [&](int64_t u, int stage) {
    seek(pre, u);
    const int at = (int)(u - pre.base), job = at / pre.s.n, tile = pre.s.first + at % pre.s.n, head = job / row_tiles;
    // lane p brings page p of the tile: all of its blocks that the tile covers
    const int token = tile * TT + lane * c.page_tokens, j = token / c.page_tokens;
    const bool want = lane < pages && token < pre.s.len && token + c.page_tokens > pre.s.lo;
    int page = -1;
    if (want) page = c.block_table[(int64_t)pre.seq * c.max_pages + j];
    const bool ok = page >= 0 && page < c.n_pages;
    if (want && !ok) atomicOr(err, EF_BAD_INDEX);
    const int n_blk = pages > 1 ? c.page_tokens / 16 : TB;      // blocks this lane copies
    const unsigned mask = __ballot_sync(0xffffffffu, ok);
    if (lane == 0) {
      uint32_t have = 0;
      for (int p = 0; p < pages; ++p)
        if (mask >> p & 1) have |= ((1u << n_blk) - 1) << (p * n_blk);
      sm.have[warp][stage] = have;
      mbar_expect_tx(&sm.full[warp][stage], __popc(mask) * n_blk * BLK);
    }
    __syncwarp();
    if (ok) {
      const int64_t blk = ((int64_t)page * c.kv_heads + head) * (c.page_tokens / 16) + (pages > 1 ? 0 : (tile % per_page) * TB);
      bulk_g2s(sm.stage[warp][stage] + lane * n_blk * BLK, (const uint8_t*)c.pages + blk * BLK, n_blk * BLK, &sm.full[warp][stage]);
    }
  };
  int64_t next = u0 + warp;                // next tile to fetch
  int filled = 0, used = 0;                // tiles fetched and consumed by this warp
  for (; filled < kStages && next < u1; ++filled, next += kWarps) fetch(next, filled % kStages);

  int64_t u = u0;                          // begin of the current job's part
  while (u < u1) {
    seek(cur, u);
    const int at = (int)(u - cur.base), job = at / cur.s.n, head = job / row_tiles, row0 = (job % row_tiles) * ROWS;
    const int64_t j0 = cur.base + (int64_t)job * cur.s.n, j1 = j0 + cur.s.n, part1 = min(j1, u1);
    const int len = cur.s.len;
    if (threadIdx.x == 0 && u == j0 && job == 0 && a.lens[cur.seq] != len) atomicOr(err, EF_BAD_INDEX);

    // ---- queries: lane (g, t) holds dims 32 w + 8 t .. + 7 of row g of each row block ----
    uint32_t q[NT][G][4];
    float qs[NT][G][2];                    // sums over the group's dims of rows 2 t and 2 t + 1
    int last[NT][2];                       // last key of rows 2 t, 2 t + 1 (-1: no such row)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const T* src = (const T*)a.q + (((int64_t)cur.seq * a.n_query + r / rep) * a.heads + head * rep + r % rep) * HD;
#pragma unroll
      for (int w = 0; w < G; ++w) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) v = *reinterpret_cast<const uint4*>(src + 32 * w + 8 * t);
        q[n][w][0] = v.x; q[n][w][1] = v.y; q[n][w][2] = v.z; q[n][w][3] = v.w;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2<T>(q[n][w][i]);
          s += f.x + f.y;
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        qs[n][w][0] = __shfl_sync(0xffffffffu, s, 8 * t);
        qs[n][w][1] = __shfl_sync(0xffffffffu, s, 8 * t + 4);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = row0 + 8 * n + 2 * t + i;
        last[n][i] = rr < rows ? len - a.n_query + rr / rep : -1;
      }
    }
    // keys that every row of the tile sees: [lo_all, hi_all]
    const int t_first = row0 / rep, t_last = min(rows - 1, row0 + ROWS - 1) / rep;
    const int hi_all = len - a.n_query + t_first, lo_all = a.window > 0 ? len - a.n_query + t_last - a.window + 1 : 0;
    const int window = a.window > 0 ? a.window : 0x7fffffff;

    float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) { m[n][i] = -CUDART_INF_F; l[n][i] = 0.f; }
    }

    // this warp's tiles of the part
    for (int64_t x = u0 + warp + (int64_t)used * kWarps; x < part1; x += kWarps) {
      const int stage = used % kStages;
      const bool landed = mbar_wait(&sm.full[warp][stage], (used / kStages) & 1, err, EF_TIMEOUT_FULL);
      const uint32_t have = landed ? sm.have[warp][stage] : 0u;
      const uint8_t* tile = sm.stage[warp][stage];
      const int key0 = (cur.s.first + (int)(x - j0)) * TT;
      const bool whole = key0 >= lo_all && key0 + TT - 1 <= hi_all && have == (1u << TB) - 1;

      // scores: s[b][n] = {key g: rows 2 t, 2 t + 1; key g + 8: the same rows}
      float s[TB][NT][4];
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        const uint8_t* blk = tile + b * BLK;
        uint32_t k0[G], k1[G], s0[G], s1[G];
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(blk) + (g * 4 + t) * G;
        const uint32_t* ks = reinterpret_cast<const uint32_t*>(blk + kv4_k_scales(HD)) + g * G;
        if (G == 2) {
          *reinterpret_cast<uint2*>(k0) = *reinterpret_cast<const uint2*>(kw);
          *reinterpret_cast<uint2*>(k1) = *reinterpret_cast<const uint2*>(kw + 32 * G);
          *reinterpret_cast<uint2*>(s0) = *reinterpret_cast<const uint2*>(ks);
          *reinterpret_cast<uint2*>(s1) = *reinterpret_cast<const uint2*>(ks + 8 * G);
        } else {
#pragma unroll
          for (int w = 0; w < G; w += 4) {
            *reinterpret_cast<uint4*>(k0 + w) = *reinterpret_cast<const uint4*>(kw + w);
            *reinterpret_cast<uint4*>(k1 + w) = *reinterpret_cast<const uint4*>(kw + 32 * G + w);
            *reinterpret_cast<uint4*>(s0 + w) = *reinterpret_cast<const uint4*>(ks + w);
            *reinterpret_cast<uint4*>(s1 + w) = *reinterpret_cast<const uint4*>(ks + 8 * G + w);
          }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[b][n][e] = 0.f;
#pragma unroll
        for (int w = 0; w < G; ++w) {
          const uint32_t a0 = codes2<T, 0>(k0[w]), a1 = codes2<T, 0>(k1[w]), a2 = codes2<T, 1>(k0[w]), a3 = codes2<T, 1>(k1[w]);
          const uint32_t a4 = codes2<T, 2>(k0[w]), a5 = codes2<T, 2>(k1[w]), a6 = codes2<T, 3>(k0[w]), a7 = codes2<T, 3>(k1[w]);
          const float2 d0 = unpack2<__half>(s0[w]), d1 = unpack2<__half>(s1[w]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float p[4] = {0.f, 0.f, 0.f, 0.f};
            mma_16816<T>(p, a0, a1, a2, a3, q[n][w][0], q[n][w][1]);
            mma_16816<T>(p, a4, a5, a6, a7, q[n][w][2], q[n][w][3]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              s[b][n][i] = fmaf(d0.x, p[i], fmaf(d0.y, qs[n][w][i], s[b][n][i]));
              s[b][n][2 + i] = fmaf(d1.x, p[2 + i], fmaf(d1.y, qs[n][w][i], s[b][n][2 + i]));
            }
          }
        }
      }
      // to log2, masked where a key is no row's business
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[b][n][e] *= c2;
            if (!whole) {
              const int key = key0 + 16 * b + g + (e >= 2 ? 8 : 0), la = last[n][e & 1];
              if (key > la || la - key >= window || !(have >> b & 1)) s[b][n][e] = -CUDART_INF_F;
            }
          }
      // raise the maximum only where a score is far above it
      bool far = false;
#pragma unroll
      for (int b = 0; b < TB; ++b)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) far |= s[b][n][e] > m[n][e & 1] + kRaise;
      if (__any_sync(0xffffffffu, far)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = m[n][i];
#pragma unroll
            for (int b = 0; b < TB; ++b) top = fmaxf(top, fmaxf(s[b][n][i], s[b][n][2 + i]));
#pragma unroll
            for (int x2 = 4; x2 < 32; x2 <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x2));
            const float f = top == -CUDART_INF_F ? 1.f : exp2_fast(m[n][i] - top);
            m[n][i] = top;
            l[n][i] *= f;
#pragma unroll
            for (int k = 0; k < MT; ++k) { o[n][k][i] *= f; o[n][k][2 + i] *= f; }
          }
      }
      // probabilities: column g of the transposed fragments holds keys 2 t, 2 t + 1 (p0) and 2 t + 8, 2 t + 9 (p1)
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        uint32_t p0[NT], p1[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float mm = m[n][e & 1] == -CUDART_INF_F ? 0.f : m[n][e & 1];
            p[e] = exp2_fast(s[b][n][e] - mm);
            l[n][e & 1] += p[e];
          }
          p0[n] = transpose8x8(pack2<__half>(p[0], p[1]));
          p1[n] = transpose8x8(pack2<__half>(p[2], p[3]));
        }
        // values: lane (g, t) brings the dims of chunk g for token pairs t and t + 4
        const uint8_t* blk = tile + b * BLK;
        uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;   // halves of the two pairs that are keys of the sequence
        if (!whole) {
          const int k = key0 + 16 * b + 2 * t, lim = have >> b & 1 ? len : 0;
          keep0 = (k < lim ? 0xFFFFu : 0u) | (k + 1 < lim ? 0xFFFF0000u : 0u);
          keep1 = (k + 8 < lim ? 0xFFFFu : 0u) | (k + 9 < lim ? 0xFFFF0000u : 0u);
        }
        auto values = [&](int first, const uint32_t* w0, const uint32_t* w1, int words, uint2 sc0, uint2 sc1) {
          sc0.x &= keep0; sc0.y &= keep0; sc1.x &= keep1; sc1.y &= keep1;
#pragma unroll
          for (int i = 0; i < words; ++i) {
            const uint32_t a0 = hfma2(codes2<__half, 0>(w0[i]), sc0.x, sc0.y), a1 = hfma2(codes2<__half, 1>(w0[i]), sc0.x, sc0.y);
            const uint32_t a2 = hfma2(codes2<__half, 0>(w1[i]), sc1.x, sc1.y), a3 = hfma2(codes2<__half, 1>(w1[i]), sc1.x, sc1.y);
            const uint32_t a4 = hfma2(codes2<__half, 2>(w0[i]), sc0.x, sc0.y), a5 = hfma2(codes2<__half, 3>(w0[i]), sc0.x, sc0.y);
            const uint32_t a6 = hfma2(codes2<__half, 2>(w1[i]), sc1.x, sc1.y), a7 = hfma2(codes2<__half, 3>(w1[i]), sc1.x, sc1.y);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_16816<__half>(o[n][first + 2 * i], a0, a1, a2, a3, p0[n], p1[n]);
              mma_16816<__half>(o[n][first + 2 * i + 1], a4, a5, a6, a7, p0[n], p1[n]);
            }
          }
        };
        const uint8_t *vc = blk + kv4_v_codes(HD), *vs = blk + kv4_v_scales(HD);
        if (HD == 64) {
          uint32_t w0[2], w1[2];
          *reinterpret_cast<uint2*>(w0) = *reinterpret_cast<const uint2*>(vc + (t * 4 + kv4_v_chunk<HD>(g >> 1, t)) * 16 + (g & 1) * 8);
          *reinterpret_cast<uint2*>(w1) = *reinterpret_cast<const uint2*>(vc + ((t + 4) * 4 + kv4_v_chunk<HD>(g >> 1, t + 4)) * 16 + (g & 1) * 8);
          values(0, w0, w1, 2, *reinterpret_cast<const uint2*>(vs + (t * G + (g >> 2)) * 8),
                 *reinterpret_cast<const uint2*>(vs + ((t + 4) * G + (g >> 2)) * 8));
        } else {
#pragma unroll
          for (int h = 0; h < HD / 128; ++h) {
            uint32_t w0[4], w1[4];
            const int C = g + 8 * h;
            *reinterpret_cast<uint4*>(w0) = *reinterpret_cast<const uint4*>(vc + (t * (HD / 16) + kv4_v_chunk<HD>(C, t)) * 16);
            *reinterpret_cast<uint4*>(w1) = *reinterpret_cast<const uint4*>(vc + ((t + 4) * (HD / 16) + kv4_v_chunk<HD>(C, t + 4)) * 16);
            values(8 * h, w0, w1, 4, *reinterpret_cast<const uint2*>(vs + (t * G + (C >> 1)) * 8),
                   *reinterpret_cast<const uint2*>(vs + ((t + 4) * G + (C >> 1)) * 8));
          }
        }
      }
      ++used;
      __syncwarp();                        // the stage is free
      if (next < u1) {
        fetch(next, stage);
        ++filled;
        next += kWarps;
      }
    }

    // ---- join the warps ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x2 = 4; x2 < 32; x2 <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x2);
        const int r = 8 * n + 2 * t + i;
        if (g == 0) { sm.m[warp][r] = m[n][i]; sm.l[warp][r] = l[n][i]; }
#pragma unroll
        for (int k = 0; k < MT; ++k) {     // tile k, rows g and g + 8: dims 2 k and 2 k + 1 of the lane's chunk
          const int d = HD == 64 ? 8 * g + 2 * k : 128 * (k >> 3) + 16 * g + 2 * (k & 7);
          *reinterpret_cast<float2*>(&sm.o[warp][r][d]) = make_float2(o[n][k][i], o[n][k][2 + i]);
        }
      }
    __syncthreads();
    const bool done = u == j0 && part1 == j1;
    const int slot = u == j0 ? 1 : 0;      // the job begins here, or began in an earlier range
    float* part = (float*)a.work + ((int64_t)blockIdx.x * 2 + slot) * partial_floats<HD, ROWS>();
    for (int i = threadIdx.x; i < ROWS * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, rr = row0 + r;
      if (rr >= rows) break;
      float top = sm.m[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
      const int h = head * rep + rr % rep;
      float base = top;
      if (done && a.sinks) base = fmaxf(top, a.sinks[h] * kLog2e);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = done && a.sinks ? exp2_fast(a.sinks[h] * kLog2e - base) : 0.f;
      if (top != -CUDART_INF_F) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(sm.m[w][r] - base);
          const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
          v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
          sum += f * sm.l[w][r];
        }
      }
      if (done) {
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
        T* dst = (T*)a.out + (((int64_t)cur.seq * a.n_query + rr / rep) * a.heads + h) * HD + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
      } else {
        *reinterpret_cast<float4*>(part + r * HD + d) = v;
        if (d == 0) { part[ROWS * HD + r] = top; part[ROWS * HD + ROWS + r] = sum; }
      }
    }
    __syncthreads();                       // the buffers may be written again
    u = part1;
  }
}

// one block per (job, row): joins the parts that the ranges left of a job
template <class T, int HD, int NT>
__global__ void __launch_bounds__(kThreads) kv4_join_kernel(const ms_kv4_cache c, const ms_kv4_attn a, int row_tiles, int ranges) {
  constexpr int TT = 4096 / HD, ROWS = 8 * NT, COLS = HD / 4, GROUPS = kThreads / COLS;
  __shared__ float4 acc[kThreads];
  __shared__ float ls[GROUPS];
  const int jobs = c.kv_heads * row_tiles, seq = blockIdx.x / jobs, job = blockIdx.x % jobs, r = blockIdx.y;
  const int rep = a.heads / c.kv_heads, rr = (job % row_tiles) * ROWS + r;
  int64_t base;
  const Plan plan = make_plan<TT>(c, a, row_tiles, ranges, seq, &base);
  const int64_t n = seq_tiles<TT>(c, a, seq).n, j0 = base + job * n, j1 = j0 + n;
  const int64_t c0 = j0 / plan.chunk, c1 = (j1 - 1) / plan.chunk;
  pdl_wait_prior();                        // every block waits: this grid must not end before the first one
  if (c0 == c1 || rr >= a.n_query * rep) return;   // finished by its block, or no such row
  const int h = (job / row_tiles) * rep + rr % rep;
  auto part = [&](int64_t b) { return (const float*)a.work + (b * 2 + (b == c0 ? 1 : 0)) * partial_floats<HD, ROWS>(); };
  // the maximum first, so that the join is one sum in a fixed order
  float top = -CUDART_INF_F;
  for (int64_t b = c0 + (threadIdx.x & 31); b <= c1; b += 32) top = fmaxf(top, part(b)[ROWS * HD + r]);
  top = warp_max(top);
  float m = a.sinks ? fmaxf(top, a.sinks[h] * kLog2e) : top;
  if (m == -CUDART_INF_F) m = 0.f;
  const int col = threadIdx.x % COLS, grp = threadIdx.x / COLS;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int64_t b = c0 + grp; b <= c1; b += GROUPS) {
    const float* p = part(b);
    const float f = exp2_fast(p[ROWS * HD + r] - m);
    const float4 x = *reinterpret_cast<const float4*>(p + r * HD + 4 * col);
    v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
    l += f * p[ROWS * HD + ROWS + r];
  }
  acc[threadIdx.x] = v;
  if (col == 0) ls[grp] = l;
  __syncthreads();
  if (grp) return;
  l = a.sinks ? exp2_fast(a.sinks[h] * kLog2e - m) : 0.f;
  v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float4 x = acc[i * COLS + col];
    v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
    l += ls[i];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* dst = (T*)a.out + (((int64_t)seq * a.n_query + rr / rep) * a.heads + h) * HD + 4 * col;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
}

// 8 rows a tile fill the tensor core's columns once; with more rows a tile of 16 reads each key once for them.
// 256 dims hold 64 accumulators a lane for 8 rows already.
int rows_of(int head_dim, int rows) { return rows > 8 && head_dim <= 128 ? 16 : 8; }
int ranges_of(const DevCtx& d, int hd, int nt) { return d.sm_count * blocks_per_sm(hd, nt); }

template <class T, int HD, int NT>
cudaError_t start(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_attn& a, cudaStream_t s) {
  const int rows = a.n_query * (a.heads / c.kv_heads), row_tiles = (rows + 8 * NT - 1) / (8 * NT);
  const int smem = sizeof(Smem<HD, NT>);
  cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<T, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  kv4_attn_kernel<T, HD, NT><<<ranges_of(d, HD, NT), kThreads, smem, s>>>(c, a, row_tiles, d.err);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.n_seqs * c.kv_heads * row_tiles, min(rows, 8 * NT));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, HD, NT>, c, a, row_tiles, ranges_of(d, HD, NT));
}

template <class T>
cudaError_t start_hd(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_attn& a, cudaStream_t s) {
  const bool wide = rows_of(c.head_dim, a.n_query * (a.heads / c.kv_heads)) == 16;
  if (c.head_dim == 64) return wide ? start<T, 64, 2>(d, c, a, s) : start<T, 64, 1>(d, c, a, s);
  if (c.head_dim == 128) return wide ? start<T, 128, 2>(d, c, a, s) : start<T, 128, 1>(d, c, a, s);
  return start<T, 256, 1>(d, c, a, s);
}

}  // namespace

size_t kv4_attn_workspace(const DevCtx& d, const ms_kv4_cache& c, int n_query, int heads) {
  const int rows = rows_of(c.head_dim, n_query * (heads / c.kv_heads));
  return (size_t)ranges_of(d, c.head_dim, rows / 8) * 2 * (rows * c.head_dim + 2 * rows) * 4;
}

cudaError_t launch_kv4_attention(const DevCtx& d, const ms_kv4_cache& c, const ms_kv4_attn& a, cudaStream_t s) {
  if (c.n_seqs == 0) return cudaSuccess;
  return a.type == MS_Q_F16 ? start_hd<__half>(d, c, a, s) : start_hd<__nv_bfloat16>(d, c, a, s);
}

}  // namespace ms
