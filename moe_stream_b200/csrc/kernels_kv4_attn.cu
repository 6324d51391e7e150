// kernels_kv4_attn.cu — attention of the newest tokens of each sequence over the paged 4-bit K/V cache.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q . k_j - m),  k, v = o + d (16 + c) per 32 dims
//
// Bound by memory: each (token, kv head) is 1.25 head_dim bytes that are read once, for all query heads of the
// group and all query tokens (the rows).  One row tile holds 8 NT rows.
//
// Work.  A job is (sequence, kv head, row tile); its keys are cut into tiles of TT = 4096 / head_dim tokens (5 KB).
// The tiles of all jobs form one list that is cut into equal ranges, one per block, so sequences of any
// lengths fill the GPU without the host knowing them; each job adds kExtra empty tiles to the list, the time that
// a block spends on the queries and the join of a job.  The 4 warps of a block take the tiles of a range in
// turn, each with its own ring of two stages filled by bulk copies, its own running maximum and sum; they are
// joined at the end of a job's part.  A job inside one range is finished there; the others leave their
// numerators and sums in the workspace, which a second kernel joins.
//
// Scores (keys x rows, m16n8k16 in f16).  The rows of q are scaled by a power of two to a largest value in [1, 2),
// which makes bf16 rows exact in f16 but for dims below 2^-14 of the largest (off by 2^-25 of it).  A code becomes
// 16 + c or 256 + c by a mask-and-or after one shift for two of them.  With P = sum q x over a group of 32 dims as
// the tensor core adds it, Q = sum q and R = -240 times the sum of the q of the 256 + c dims,
//   s = sum over the groups of (d R + o Q) + d P.
// The first part is one more product of the stored (d, o) pairs with R and Q, each cut into two f16 (22 bits);
// the second is one f32 multiply-add a group.  Values: v = fma(16 + c, d, o) in f16 pairs of two keys, the probabilities in f16 (bf16 would
// cost 8 times their rounding; with f16 outputs, where it shows, their rests in a second product) transposed by
// movmatrix from the score layout.  The probabilities are taken against the running maximum less kBelow (7): the largest is
// 2^7, so those that f16 rounds to a multiple of 2^-24 lie below 2^-21 of it and are off by 2^-32 of it at most (against the
// maximum itself, keys below 2^-25 of it would have counted in the sum and not in the output: 4,000 keys at 2^-25.5 behind
// one of 1 lost all of their share).  The maximum is raised only when a lane's probabilities of a tile add up to more than
// 2^15, 2^8 times the largest: p stays inside f16, and most tiles need no reduction over the lanes.
//
// Measured: 32 sequences of 7,845 tokens on average, 4 heads of 128 dims (161 MB): 44 us, 3.7 TB/s; one of 131,072
// tokens, 8 heads of 64 dims (84 MB, f16): 28 us; one of 4,097 tokens: 9 us.  Bulk copies alone stream the first
// in 30 us, about what the loop takes; 3 us go by before the first copy (lengths, split, page numbers), the blocks end up to
// 4 us apart, and the second kernel takes 3 to 4 us.  The loop issues 330 instructions a warp for 16 tokens of 128 dims and
// keeps the issue slots half busy.
#include <type_traits>

#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv4.cuh"
#include "phases.h"

namespace ms {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStages = 2;
constexpr int kTileBytes = 5120;          // 16 * 20 * 16 for every head_dim
// blocks of an SM: 3 leave 168 registers a thread; 256 dims, or 16 rows of 128, need more than that.  (4 blocks, with
// a few values spilled, have more warps but more starts, joins and parts: 47 us for 3's 44 on a batch of 32
// sequences of 7,845 tokens on average, 4 heads of 128 dims.)
__host__ __device__ constexpr int blocks_per_sm(int hd, int nt) { return hd * nt >= 256 ? 2 : 3; }
constexpr int kMinTiles = kWarps;         // tiles of a range at least: one per warp
constexpr int kExtra = 8;                 // empty tiles behind those of a job
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -1e30f;           // the running maximum before any key
constexpr float kBelow = 7.0f;            // powers of two that the probabilities' base lies below the maximum
constexpr float kRaise = 32768.0f;        // sum of a lane's probabilities of a tile that raises the maximum

// ---- the list of tiles ----
struct Plan {        // (the callers check that all tiles of a cache's capacity are below 2^31)
  int jobs;          // of one sequence: kv heads x row tiles
  int total;         // tiles of all jobs, the empty ones counted
  int chunk;         // tiles of one block's range
};
struct SeqTiles {
  int len;           // tokens (checked)
  int lo;            // first key of any query
  int first;         // index of the first tile
  int n;             // tiles of one job, at least 1 (a sequence without tokens still gets its zeros)
  __device__ __forceinline__ int units() const { return n + kExtra; }
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
// whole warp: the plan, and the tiles of the jobs of the sequences in front of `before`
template <int TT>
__device__ __forceinline__ Plan make_plan(const ms_kv4_cache& c, const ms_kv4_attn& a, int row_tiles, int ranges, int before,
                                          int* in_front) {
  const int lane = threadIdx.x & 31;
  int all = 0, front = 0;
  for (int i = lane; i < c.n_seqs; i += 32) {
    const int n = seq_tiles<TT>(c, a, i).units();
    all += n;
    if (i < before) front += n;
  }
  all = __reduce_add_sync(0xffffffffu, all);
  front = __reduce_add_sync(0xffffffffu, front);
  Plan p;
  p.jobs = c.kv_heads * row_tiles;
  p.total = all * p.jobs;
  p.chunk = max(kMinTiles, (int)(((unsigned)p.total + ranges - 1) / (unsigned)ranges));
  *in_front = front * p.jobs;
  return p;
}

// a tile of the list; every lane of a warp holds the same one
struct Cursor {
  int seq, job, tile;   // tile counts from s.first; from s.n on it is empty
  SeqTiles s;
};
template <int TT>
__device__ __forceinline__ Cursor find_tile(const ms_kv4_cache& c, const ms_kv4_attn& a, const Plan& p, int u) {
  const int lane = threadIdx.x & 31;
  Cursor k;
  int at = 0;
  for (int b = 0; b < c.n_seqs; b += 32) {
    const int n = b + lane < c.n_seqs ? seq_tiles<TT>(c, a, b + lane).units() * p.jobs : 0;
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, u < at + inc);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int in = u - at - __shfl_sync(0xffffffffu, inc - n, l);
      k.seq = b + l;
      k.s = seq_tiles<TT>(c, a, k.seq);
      k.job = in / k.s.units();
      k.tile = in - k.job * k.s.units();
      return k;
    }
    at += __shfl_sync(0xffffffffu, inc, 31);
  }
  return k;             // not reached: u < total
}
template <int TT>
__device__ __forceinline__ void advance(const ms_kv4_cache& c, const ms_kv4_attn& a, int jobs, Cursor& k, int n) {
  k.tile += n;
  while (k.tile >= k.s.units()) {
    k.tile -= k.s.units();
    if (++k.job == jobs) {
      k.job = 0;
      if (++k.seq == c.n_seqs) return;   // behind the list
      k.s = seq_tiles<TT>(c, a, k.seq);
    }
  }
}

// partial of one block and one of its two cut jobs: [rows][HD] numerators, then m and l of the rows
template <int HD, int ROWS>
__host__ __device__ constexpr int partial_floats() { return ROWS * HD + 2 * ROWS; }

// ---- tensor-core pieces ----
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                    float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// K = 8: A rows g and g + 8, k = 2 t and 2 t + 1
__device__ __forceinline__ void mma_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}
// the four pairs of a word (nibbles at bits 4 n and 4 n + 16) as f16 numbers: pairs 0 and 2 as 256 + c, pairs 1
// and 3 as 16 + c, the code in the mantissa bits that weigh 1 to 8
// (a three-input logic instruction takes one constant: the other two stay in registers)
struct Bases {
  uint32_t b256 = 0x5C005C00u, b16 = 0x4C004C00u;
  __device__ __forceinline__ Bases() { asm volatile("" : "+r"(b256), "+r"(b16)); }
};
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mask_or(uint32_t x, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(base));
  return r;
}
__device__ __forceinline__ void codes(uint32_t w, const Bases& k, uint32_t (&x)[4]) {
  const uint32_t lo = w << 2, hi = w >> 6;
  x[0] = mask_or<0x003C003Cu>(lo, k.b256);
  x[1] = mask_or<0x03C003C0u>(lo, k.b16);
  x[2] = mask_or<0x003C003Cu>(hi, k.b256);
  x[3] = mask_or<0x03C003C0u>(hi, k.b16);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t minus240(uint32_t a) {   // 256 + c -> 16 + c, exact
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xDB80DB80u));
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
  static constexpr int kPitch = HD + 4;   // floats between rows of the joining buffers
  alignas(128) uint8_t stage[kWarps][kStages][kTileBytes];
  alignas(16) float o[kWarps / 2][8 * NT][kPitch];
  float m[kWarps][8 * NT], l[kWarps][8 * NT];
  uint64_t full[kWarps][kStages];
  uint32_t have[kWarps][kStages];         // blocks of the tile that were copied
  int issued[kWarps];                     // tiles that the warp has fetched
};

// what a warp keeps of a job
template <int HD, int NT>
struct Rows {
  static constexpr int G = HD / 32, MT = HD / 16;
  uint32_t q[NT][G][4];    // lane (g, t): dims 32 w + 8 t .. + 7 of row g
  // (R, Q) of row g as pairs: group 4 j + t in corr[j][0] and what f16 left of it in [1]; with 2 groups, lanes
  // t = 0, 1 hold the groups and t = 2, 3 the rests
  static constexpr int CORR = (G + 3) / 4;
  uint32_t corr[NT][CORR][2];
  float c2[NT][2];         // log2(e) scale times the row's power of two
  int last[NT][2];         // the row's last key (-1: no such row)
  float o[NT][MT][4], m[NT][2], l[NT][2];   // m: the base of the probabilities, kBelow under the running maximum
};

// one tile: scores, probabilities, value product.  MASKED: some keys are not every row's
template <int HD, int NT, bool MASKED, bool RESTS>
__device__ __forceinline__ void take_tile(Rows<HD, NT>& R, const Bases& K, const uint8_t* tile, int key0, int len, int window,
                                          uint32_t have) {
  constexpr int G = HD / 32, TB = 256 / HD, BLK = 20 * HD, MT = HD / 16;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
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
    if (G == 2) {
      const uint32_t a0 = ks[(t & 1)], a1 = ks[8 * G + (t & 1)];
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_k8(s[b][n], a0, a1, R.corr[n][0][0]);
    } else {
#pragma unroll
      for (int j = 0; j < G / 4; ++j) {
        const uint32_t a0 = ks[4 * j + t], a1 = ks[8 * G + 4 * j + t];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          if (j == 0) mma(s[b][n], a0, a1, a0, a1, R.corr[n][j][0], R.corr[n][j][1], 0.f, 0.f, 0.f, 0.f);
          else mma_add(s[b][n], a0, a1, a0, a1, R.corr[n][j][0], R.corr[n][j][1]);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < G; ++w) {
      uint32_t x0[4], x1[4];
      codes(k0[w], K, x0);
      codes(k1[w], K, x1);
      const float d0 = h2f_bits((uint16_t)s0[w]), d1 = h2f_bits((uint16_t)s1[w]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float p[4];
        mma(p, x0[0], x1[0], x0[1], x1[1], R.q[n][w][0], R.q[n][w][1], 0.f, 0.f, 0.f, 0.f);
        mma_add(p, x0[2], x1[2], x0[3], x1[3], R.q[n][w][2], R.q[n][w][3]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[b][n][i] = fmaf(d0, p[i], s[b][n][i]);
          s[b][n][2 + i] = fmaf(d1, p[2 + i], s[b][n][2 + i]);
        }
      }
    }
    if (MASKED) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 16 * b + g + (e >= 2 ? 8 : 0), la = R.last[n][e & 1];
          if (key > la || la - key >= window || !(have >> b & 1)) s[b][n][e] = -INFINITY;
        }
    }
  }
  // probabilities against the running base; when they grow too large it is raised first
  float p[TB][NT][4];
  auto exps = [&]() {
    bool far = false;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          p[b][n][i] = exp2_fast(fmaf(s[b][n][i], R.c2[n][i], -R.m[n][i]));
          p[b][n][2 + i] = exp2_fast(fmaf(s[b][n][2 + i], R.c2[n][i], -R.m[n][i]));
          sum += p[b][n][i] + p[b][n][2 + i];
        }
        far |= sum > kRaise;
        R.l[n][i] += sum;
      }
    return far;
  };
  float l0[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) { l0[n][0] = R.l[n][0]; l0[n][1] = R.l[n][1]; }
  if (__any_sync(0xffffffffu, exps())) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < TB; ++b) top = fmaxf(top, fmaxf(s[b][n][i], s[b][n][2 + i]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(fmaf(top, R.c2[n][i], -kBelow), R.m[n][i]);
        const float f = exp2_fast(R.m[n][i] - top);
        R.m[n][i] = top;
        R.l[n][i] = l0[n][i] * f;
#pragma unroll
        for (int k = 0; k < MT; ++k) { R.o[n][k][i] *= f; R.o[n][k][2 + i] *= f; }
      }
    exps();
  }
  // values: lane (g, t) brings the dims of chunk g for token pairs t and t + 4 (rows of the product); the
  // transposed probabilities hold keys 2 t, 2 t + 1 (p0) and 2 t + 8, 2 t + 9 (p1) of row g (columns)
#pragma unroll
  for (int b = 0; b < TB; ++b) {
    uint32_t p0[NT], p1[NT], r0[NT], r1[NT];               // r: what f16 left of p
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint32_t x = pack2<__half>(p[b][n][0], p[b][n][1]), y = pack2<__half>(p[b][n][2], p[b][n][3]);
      p0[n] = transpose8x8(x);
      p1[n] = transpose8x8(y);
      if (RESTS) {
        const float2 fx = unpack2<__half>(x), fy = unpack2<__half>(y);
        r0[n] = transpose8x8(pack2<__half>(p[b][n][0] - fx.x, p[b][n][1] - fx.y));
        r1[n] = transpose8x8(pack2<__half>(p[b][n][2] - fy.x, p[b][n][3] - fy.y));
      }
    }
    const uint8_t* blk = tile + b * BLK;
    uint32_t keep0 = 0xFFFFFFFFu, keep1 = 0xFFFFFFFFu;   // halves of the two pairs that are tokens of the sequence
    if (MASKED) {
      const int k = key0 + 16 * b + 2 * t, lim = have >> b & 1 ? len : 0;
      keep0 = (k < lim ? 0xFFFFu : 0u) | (k + 1 < lim ? 0xFFFF0000u : 0u);
      keep1 = (k + 8 < lim ? 0xFFFFu : 0u) | (k + 9 < lim ? 0xFFFF0000u : 0u);
    }
    auto values = [&](int first, const uint32_t* w0, const uint32_t* w1, int words, uint2 sc0, uint2 sc1) {
      if (MASKED) { sc0.x &= keep0; sc0.y &= keep0; sc1.x &= keep1; sc1.y &= keep1; }
#pragma unroll
      for (int i = 0; i < words; ++i) {
        uint32_t x0[4], x1[4];
        codes(w0[i], K, x0);
        codes(w1[i], K, x1);
        const uint32_t a0 = hfma2(minus240(x0[0]), sc0.x, sc0.y), a1 = hfma2(x0[1], sc0.x, sc0.y);
        const uint32_t a2 = hfma2(minus240(x1[0]), sc1.x, sc1.y), a3 = hfma2(x1[1], sc1.x, sc1.y);
        const uint32_t a4 = hfma2(minus240(x0[2]), sc0.x, sc0.y), a5 = hfma2(x0[3], sc0.x, sc0.y);
        const uint32_t a6 = hfma2(minus240(x1[2]), sc1.x, sc1.y), a7 = hfma2(x1[3], sc1.x, sc1.y);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_add(R.o[n][first + 2 * i], a0, a1, a2, a3, p0[n], p1[n]);
          mma_add(R.o[n][first + 2 * i + 1], a4, a5, a6, a7, p0[n], p1[n]);
          if (RESTS) {
            mma_add(R.o[n][first + 2 * i], a0, a1, a2, a3, r0[n], r1[n]);
            mma_add(R.o[n][first + 2 * i + 1], a4, a5, a6, a7, r0[n], r1[n]);
          }
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
}

template <class T, int HD, int NT>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(HD, NT)) kv4_attn_kernel(const ms_kv4_cache c, const ms_kv4_attn a,
                                                                                  int row_tiles, uint32_t* err) {
  constexpr int G = HD / 32, TB = 256 / HD, TT = 16 * TB, BLK = 20 * HD, ROWS = 8 * NT, MT = HD / 16;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<HD, NT>& sm = *reinterpret_cast<Smem<HD, NT>*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
    sm.issued[warp] = 0;
    fence_mbar_init();
  }
  __syncwarp();
  pdl_wait_prior();
  pdl_launch_dependents();
  int unused;
  const Plan plan = make_plan<TT>(c, a, row_tiles, gridDim.x, 0, &unused);
  if (blockIdx.x >= (plan.total + plan.chunk - 1u) / plan.chunk) return;
  const int u0 = blockIdx.x * plan.chunk, count = min(plan.chunk, plan.total - u0);   // the range
  const int rep = a.heads / c.kv_heads, rows = a.n_query * rep;
  const int shift = 31 - __clz(c.page_tokens);               // page_tokens is a power of two
  const int window = a.window > 0 ? a.window : 0x7fffffff;

  Cursor cur = find_tile<TT>(c, a, plan, u0), pre = cur;
  // ---- the ring: tiles warp, warp + kWarps, ... of the range; `page` is looked up one tile ahead ----
  const bool one_page = (1 << shift) >= TT;                  // a tile lies inside one page (else lane p brings page p of it)
  int page = 0;
  bool want = false;                                         // the lane brings that page (nothing looks at it before the copy)
  auto look_up = [&]() {
    const int token = (pre.s.first + pre.tile) * TT + (one_page ? 0 : lane << shift);
    want = lane < (one_page ? 1 : TT >> shift) && token < pre.s.len && token + c.page_tokens > pre.s.lo;
    if (want) page = c.block_table[(int64_t)pre.seq * c.max_pages + (token >> shift)];
  };
  auto fetch = [&](int k) {                                  // the warp's tile number k
    const int stage = k % kStages;
    const int head = row_tiles > 1 ? pre.job / row_tiles : pre.job;
    const bool ok = want && (unsigned)page < (unsigned)c.n_pages;
    if (want && !ok) atomicOr(err, EF_BAD_INDEX);
    const int n_blk = one_page ? TB : 1 << (shift - 4);      // blocks that a lane copies
    uint32_t have = ok ? ((1u << n_blk) - 1) << (one_page ? 0 : lane * n_blk) : 0u;
    if (!one_page) have = __reduce_or_sync(0xffffffffu, have);
    if (lane == 0) {
      sm.have[warp][stage] = have;
      sm.issued[warp] = k + 1;
      mbar_expect_tx(&sm.full[warp][stage], __popc(have) * BLK);
    }
    if (!one_page) __syncwarp();
    if (ok) {
      const int blk0 = one_page ? (((pre.s.first + pre.tile) * TT) & (c.page_tokens - 1)) >> 4 : 0;
      const int64_t blk = (((int64_t)page * c.kv_heads + head) << (shift - 4)) + blk0;
      bulk_g2s(sm.stage[warp][stage] + lane * n_blk * BLK, (const uint8_t*)c.pages + blk * BLK, n_blk * BLK, &sm.full[warp][stage]);
    }
  };
  int next = warp, used = 0;                                 // next tile to fetch; tiles taken by this warp
  auto step_next = [&](int n) {                              // to the warp's next tile that is not empty
    do {
      advance<TT>(c, a, plan.jobs, pre, n);
      n = kWarps;
    } while (next < count && pre.tile >= pre.s.n && (next += kWarps) < count);
    if (next < count) look_up();
  };
  auto fetch_next = [&](int k) {
    fetch(k);
    next += kWarps;
    step_next(kWarps);
  };
  step_next(warp);
  for (int i = 0; i < kStages && next < count; ++i) fetch_next(i);

  int at = 0;                                                // begin of the current job's part
  while (at < count) {
    const int head = row_tiles > 1 ? cur.job / row_tiles : cur.job, row0 = (cur.job - head * row_tiles) * ROWS;
    const int end = min(count, at + cur.s.n - cur.tile), rest = min(count, at + cur.s.units() - cur.tile);
    if (end <= at) {                                         // only empty tiles
      advance<TT>(c, a, plan.jobs, cur, rest - at);
      at = rest;
      continue;
    }
    const bool begins = cur.tile == 0, done = begins && end - at == cur.s.n;
    const int len = cur.s.len;
    if (threadIdx.x == 0 && begins && cur.job == 0 && a.lens[cur.seq] != len) atomicOr(err, EF_BAD_INDEX);

    constexpr bool RESTS = std::is_same<T, __half>::value;
    const Bases K;
    Rows<HD, NT> R;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g;
      const T* src = (const T*)a.q + (((int64_t)cur.seq * a.n_query + r / rep) * a.heads + head * rep + r % rep) * HD;
      uint4 raw[G];
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < G; ++w) {
        raw[w] = make_uint4(0, 0, 0, 0);
        if (r < rows) raw[w] = *reinterpret_cast<const uint4*>(src + 32 * w + 8 * t);
        const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack2<T>(u[i]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row times 2^(127 - eb); rows of zeros, infinities or NaN as they are
      int eb = (int)(__float_as_uint(top) >> 23);
      eb = eb == 0 || eb == 255 ? 127 : min(eb, 253);
      const float down = __uint_as_float((uint32_t)(254 - eb) << 23);
      const float c2 = a.scale * kLog2e * __uint_as_float((uint32_t)eb << 23);
#pragma unroll
      for (int w = 0; w < G; ++w) {
        const uint32_t u[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
        float s[2] = {0.f, 0.f};                             // of the 256 + c and of the 16 + c dims
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 f = unpack2<T>(u[i]);
          R.q[n][w][i] = pack2<__half>(f.x * down, f.y * down);
          f = unpack2<__half>(R.q[n][w][i]);
          s[i & 1] += f.x + f.y;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);
          s[i] += __shfl_xor_sync(0xffffffffu, s[i], 2);
        }
        const float rr = -240.f * s[0], qq = s[0] + s[1];
        const uint32_t whole = pack2<__half>(rr, qq);
        const float2 f = unpack2<__half>(whole);
        const uint32_t rest = pack2<__half>(rr - f.x, qq - f.y);
        if (G == 2) {
          if (w == 0 || (t & 1)) R.corr[n][0][0] = t < 2 ? whole : rest;
        } else if (t == (w & 3)) {
          R.corr[n][w / 4][0] = whole;
          R.corr[n][w / 4][1] = rest;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int rr = row0 + 8 * n + 2 * t + i;
        R.last[n][i] = rr < rows ? len - a.n_query + rr / rep : -1;
        R.c2[n][i] = fmaxf(__shfl_sync(0xffffffffu, c2, 8 * t + 4 * i), 1e-37f);   // never 0: a masked score stays -inf
        R.m[n][i] = kNone;
        R.l[n][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) R.o[n][i][e] = 0.f;
    }
    // keys that every row of the tile sees: lo_all .. hi_all
    const int t_first = row0 / rep, t_last = min(rows - 1, row0 + ROWS - 1) / rep;
    const int hi_all = len - a.n_query + t_first, lo_all = a.window > 0 ? len - a.n_query + t_last - a.window + 1 : 0;

    bool landed = true;
    for (int x = at + ((warp - at) & (kWarps - 1)); x < end; x += kWarps) {
      const int stage = used % kStages;
      landed = __all_sync(0xffffffffu, mbar_wait(&sm.full[warp][stage], fill_phase(used, kStages) & 1, err, EF_TIMEOUT_FULL));
      if (!landed) break;
      const uint32_t have = sm.have[warp][stage];
      const int key0 = (cur.s.first + cur.tile + x - at) * TT;
      if (key0 >= lo_all && key0 + TT - 1 <= hi_all && have == (1u << TB) - 1)
        take_tile<HD, NT, false, RESTS>(R, K, sm.stage[warp][stage], key0, len, window, have);
      else
        take_tile<HD, NT, true, RESTS>(R, K, sm.stage[warp][stage], key0, len, window, have);
      ++used;
      __syncwarp();                                          // the stage is free
      if (next < count) fetch_next(used + kStages - 1);      // the other stages are full or on their way
    }

    // ---- join the warps: all on the largest maximum, the upper half of them into the lower half ----
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) R.l[n][i] += __shfl_xor_sync(0xffffffffu, R.l[n][i], x);
        if (g == 0) {
          sm.m[warp][8 * n + 2 * t + i] = R.m[n][i];
          sm.l[warp][8 * n + 2 * t + i] = R.l[n][i];
        }
      }
    // where a wait ran out the block leaves, when no copy is under way any more
    if (__syncthreads_or(!landed)) {
      for (; used < sm.issued[warp]; ++used) mbar_wait(&sm.full[warp][used % kStages], fill_phase(used, kStages) & 1, nullptr, 0);
      return;
    }
    // tile k of the product, rows g and g + 8: dims 2 k and 2 k + 1 of the lane's chunk
    auto place = [&](int r, int k) -> float2* {
      const int d = HD == 64 ? 8 * g + 2 * k : 128 * (k >> 3) + 16 * g + 2 * (k & 7);
      return reinterpret_cast<float2*>(&sm.o[warp % (kWarps / 2)][r][d]);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * n + 2 * t + i;
        float top = sm.m[0][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
        const float f = exp2_fast(R.m[n][i] - top);
#pragma unroll
        for (int k = 0; k < MT; ++k) {
          R.o[n][k][i] *= f;
          R.o[n][k][2 + i] *= f;
          if (warp >= kWarps / 2) *place(r, k) = make_float2(R.o[n][k][i], R.o[n][k][2 + i]);
        }
      }
    __syncthreads();
    if (warp < kWarps / 2) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            float2* p = place(8 * n + 2 * t + i, k);
            const float2 x = *p;
            *p = make_float2(x.x + R.o[n][k][i], x.y + R.o[n][k][2 + i]);
          }
    }
    __syncthreads();
    float* part = (float*)a.work + ((int64_t)blockIdx.x * 2 + (begins ? 1 : 0)) * partial_floats<HD, ROWS>();
    for (int i = threadIdx.x; i < ROWS * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, rr = row0 + r;
      if (rr >= rows) break;
      float4 v = *reinterpret_cast<const float4*>(&sm.o[0][r][d]);
#pragma unroll
      for (int w = 1; w < kWarps / 2; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][r][d]);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      float top = sm.m[0][r], sum = 0.f;
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sm.m[w][r]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += exp2_fast(sm.m[w][r] - top) * sm.l[w][r];
      if (done) {
        const int h = head * rep + rr % rep;
        float f = 1.f;
        if (a.sinks && sum != 0.f) {
          const float sink = a.sinks[h] * kLog2e, base = fmaxf(top, sink);
          f = exp2_fast(top - base);
          sum = sum * f + sink_share(sink, base);
        }
        f = sum == 0.f ? 0.f : f / sum;                      // (no keys: zeros)
        T* dst = (T*)a.out + (((int64_t)cur.seq * a.n_query + rr / rep) * a.heads + h) * HD + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(v.x * f, v.y * f), pack2<T>(v.z * f, v.w * f));
      } else {
        *reinterpret_cast<float4*>(part + r * HD + d) = v;
        if (d == 0) { part[ROWS * HD + r] = top; part[ROWS * HD + ROWS + r] = sum; }
      }
    }
    __syncthreads();                                         // the buffers may be written again
    advance<TT>(c, a, plan.jobs, cur, rest - at);
    at = rest;
  }
}

// one block per (job, row): joins the parts that the ranges left of a job
template <class T, int HD, int NT, int FLIGHT>
__global__ void __launch_bounds__(kThreads) kv4_join_kernel(const ms_kv4_cache c, const ms_kv4_attn a, int row_tiles, int ranges) {
  constexpr int TT = 4096 / HD, ROWS = 8 * NT, COLS = HD / 4, GROUPS = kThreads / COLS;
  __shared__ float4 acc[kThreads];
  __shared__ float ls[GROUPS], ms[GROUPS];
  const int jobs = c.kv_heads * row_tiles, seq = blockIdx.x / jobs, job = blockIdx.x % jobs, r = blockIdx.y;
  const int rep = a.heads / c.kv_heads, rr = (job % row_tiles) * ROWS + r;
  int base;
  const Plan plan = make_plan<TT>(c, a, row_tiles, ranges, seq, &base);
  const SeqTiles st = seq_tiles<TT>(c, a, seq);
  const int j0 = base + job * st.units(), c0 = j0 / plan.chunk, c1 = (j0 + st.n - 1) / plan.chunk;
  pdl_wait_prior();                        // every block waits: this grid must not end before the first one
  pdl_launch_dependents();
  if (c0 == c1 || rr >= a.n_query * rep) return;   // finished by its block, or no such row
  const int h = (job / row_tiles) * rep + rr % rep;
  auto part = [&](int b) { return (const float*)a.work + ((int64_t)b * 2 + (b == c0 ? 1 : 0)) * partial_floats<HD, ROWS>(); };
  // a group of threads joins every GROUPS-th part on its own running maximum, FLIGHT loads under way at a time (8 where
  // no more are left)
  const int col = threadIdx.x % COLS, grp = threadIdx.x / COLS;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = kNone, l = 0.f;
  auto take = [&](int b0, auto flight) {
    constexpr int N = decltype(flight)::value;
    float4 x[N];
    float pm[N], pl[N], top = m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int b = b0 + i * GROUPS;
      pm[i] = kNone;
      pl[i] = 0.f;
      x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (b <= c1) {
        const float* p = part(b);
        pm[i] = p[ROWS * HD + r];
        pl[i] = p[ROWS * HD + ROWS + r];
        x[i] = *reinterpret_cast<const float4*>(p + r * HD + 4 * col);
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, pm[i]);
    float f = exp2_fast(m - top);
    v.x *= f; v.y *= f; v.z *= f; v.w *= f;
    l *= f;
    m = top;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      f = exp2_fast(pm[i] - top);
      v.x += f * x[i].x; v.y += f * x[i].y; v.z += f * x[i].z; v.w += f * x[i].w;
      l += f * pl[i];
    }
  };
  int b0 = c0 + grp;
  if (FLIGHT > 8)
    for (; b0 + 8 * GROUPS <= c1; b0 += FLIGHT * GROUPS) take(b0, std::integral_constant<int, FLIGHT>());
  for (; b0 <= c1; b0 += 8 * GROUPS) take(b0, std::integral_constant<int, 8>());
  acc[threadIdx.x] = v;
  if (col == 0) { ls[grp] = l; ms[grp] = m; }
  __syncthreads();
  if (grp) return;
  const float sink = a.sinks ? a.sinks[h] * kLog2e : kNone;
  float top = sink;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) top = fmaxf(top, ms[i]);
  l = a.sinks ? sink_share(sink, top) : 0.f;
  float keys = 0.f;                        // 0: the row has none
  v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const float4 x = acc[i * COLS + col];
    const float f = exp2_fast(ms[i] - top);
    v.x += f * x.x; v.y += f * x.y; v.z += f * x.z; v.w += f * x.w;
    l += f * ls[i];
    keys += ls[i];
  }
  const float inv = keys == 0.f ? 0.f : 1.f / l;
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
  // both kernels start while their predecessor ends and wait for it on the device
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = s;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(kThreads);
  cfg.gridDim = dim3(ranges_of(d, HD, NT));
  cfg.dynamicSmemBytes = smem;
  e = cudaLaunchKernelEx(&cfg, kv4_attn_kernel<T, HD, NT>, c, a, row_tiles, d.err);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(c.n_seqs * c.kv_heads * row_tiles, min(rows, 8 * NT));
  cfg.dynamicSmemBytes = 0;
  // Few jobs have many parts each, and one round of loads costs about a microsecond: 16 loads at a time then.  One
  // sequence, 4 heads of 128 dims, 8 against 16: 7.6 / 7.6 us (200 tokens), 9.1 / 8.7 (4,097), 12.8 / 11.1 (9,000).  With
  // many jobs the blocks' registers count: 32 sequences of 7,845 tokens on average 43.5 against 45.2 us.
  if (ranges_of(d, HD, NT) >= 32 * (int)cfg.gridDim.x)
    return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, HD, NT, 16>, c, a, row_tiles, ranges_of(d, HD, NT));
  return cudaLaunchKernelEx(&cfg, kv4_join_kernel<T, HD, NT, 8>, c, a, row_tiles, ranges_of(d, HD, NT));
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
