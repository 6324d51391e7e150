// kernels_prompt_attn.cu — causal attention of packed sequences of different lengths (grouped heads, sliding
// window, sinks, keys of a cached prefix in front of the queries), on the 5th-generation tensor cores.
//
//   out = sum_j p_j v_j / (sum_j p_j + exp(sink - m)),  p_j = exp(scale q . k_j - m)
//
// A query tile is 128 rows: all heads of one kv head's group for 128 / group tokens, so that K and V are read
// once for the group and short sequences still fill a tile.  A block holds NQ query tiles of one sequence (2; 1
// with 256 dims, whose output takes half of the tensor memory) and walks over the keys in tiles of BN.
//
// Warps: NQ groups of 4 for the softmax, one that issues the MMAs, two that issue the TMA copies (K and V).  Steps
// s = 0, 1, ... alternate between two score buffers in tensor memory: with NQ = 2 step s is query tile s & 1 and
// key tile s / 2, with NQ = 1 it is key tile s.  The MMA warp issues scores(s + 2) right after values(s), so the
// tensor core works on one buffer while the softmax works on the other.  A softmax thread owns a row: it reads
// the scores, writes the probabilities as 16-bit pairs, and the value product takes them from tensor memory.  With
// 128 and 256 dims they lie over the scores they came from, which the MMA warp overwrites next: the MMAs of
// one thread execute in the order of issue.  The running maximum is that of the row's first tile until the
// probabilities of a later one add up to too much (Range): only then the tile's maximum is looked for and the output
// rescaled, and no probability comes beyond the largest f16.  In f16 the probabilities are taken against the maximum less
// 7, so the largest is 2^7 and those that f16 rounds to a multiple of 2^-24 are off by 2^-32 of it at most (against the maximum
// itself, keys below 2^-25 of it would have counted in the sum and not in the output).  Sums are in f32 over the unrounded
// probabilities.
//
// Values of keys behind the sequence's end (other rows of the packed buffer, perhaps not finite) are zeroed in
// shared memory before the last product; their scores are masked.
//
// CL = 2 (256 dims): two blocks of a cluster share each MMA (M = 256), each with its own 128 rows and half of every K
// and V tile.  With one query tile a block, 256 dims read K and V from L2 for 128 rows only, 28 bytes a cycle and
// SM, and waited for them: a chunk of 2,048 queries behind 9,001 keys (336 GFLOP) took 352 us, with pairs 238 us on the same
// card, in a graph.  Now 241 us in a graph (1,394 TFLOP/s, 83 % of the cuBLAS rate in a burst) and 284 us call after call, under the
// power cap (1,186 TFLOP/s, 84 % of cuBLAS's sustained rate); its 128 pairs take two rounds of 74.  128 dims have two query
// tiles a block and lose by pairs, whose two blocks wait for each other: 463 us became 526 us for 8,192 tokens of 32 heads
// (550 GFLOP; now 462 to 519 us in a graph by the card's clock, 538 us call after call: 1,023 TFLOP/s, 73 % of the sustained
// rate).  There a key tile takes 3,900 cycles: the chain of scores (512), softmax (1,890, of which
// 1,024 are the special-function unit's for 128 exponentials a thread), values (512) and four hand-overs of a
// slot, two slots in turn.  What did not help there: a quarter of the exponentials as polynomials, probabilities
// handed over in halves, two threads a row (515 us), an MMA warp for each slot (interleaving their MMAs costs 40 %),
// blocks of half the tensor memory, two to an SM (64 dims: 235 us became 285, an MMA of 64 columns takes as long as one of 128).
#include <cuda.h>

#include <type_traits>

#include "../../include/moestream_cuda.h"
#include "attn_types.cuh"
#include "common.cuh"
#include "kernels.h"
#include "phases.h"
#include "umma.cuh"

namespace ms {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -1e30f;   // the running maximum before any key
// powers of two that the probabilities' base lies below the running maximum, and the sum of a row's probabilities of a
// tile that raises it (f16: its largest number; bf16 has the range of f32)
template <class T>
struct Range {
  static constexpr float below = 0.f, raise = 4096.f;
};
template <>
struct Range<__half> {
  static constexpr float below = 7.f, raise = 65504.f;
};

// CL: blocks that share an MMA (a pair reads each K and V tile once for twice the rows, half of it each)
template <int HD, int CL>
struct Shape {
  static_assert(CL == (HD == 256 ? 2 : 1));             // pairs of blocks have one query tile each
  static constexpr int NQ = CL == 2 ? 1 : 2;            // query tiles of a block
  static constexpr int BN = 128;                        // keys of a tile
  static constexpr int STAGES = HD == 64 ? 4 : 2;       // of K and of V
  static constexpr int Q_BYTES = 128 * HD * 2, KV_BYTES = BN * HD * 2 / CL;
  static constexpr int K_ROWS = BN / CL, V_BLOCKS = HD / 64 / CL;   // a block's share: rows of K, blocks of 64 dims of V
  static constexpr int SOFTMAX_WARPS = 4 * NQ, THREADS = 32 * (SOFTMAX_WARPS + 4);
  static constexpr int SMEM = 1024 + NQ * Q_BYTES + 2 * STAGES * KV_BYTES;
  // columns of tensor memory: two score buffers, the outputs and, with 64 dims, the probabilities of the two buffers;
  // otherwise all 512 columns are full and the probabilities take the first half of the scores they came from
  static constexpr uint32_t O_COL = 2 * BN, P_COL = HD == 64 ? O_COL + NQ * HD : 0, P_STEP = HD == 64 ? BN / 2 : BN;
  static constexpr uint32_t COLS = 512;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

// where a block works
struct Place {
  int seq, q0, q1, k0, k1;   // rows of the sequence
  int t0;                    // first token of the block
  int tiles, first;          // key tiles, and the first one's index in the sequence
  bool ok;
};
template <int HD, int CL>
__device__ __forceinline__ Place find_place(const ms_prompt_attn& a, int n_tok, int index, uint32_t* err) {
  using S = Shape<HD, CL>;
  const int lane = threadIdx.x & 31, per = CL * S::NQ * n_tok;
  Place p;
  p.ok = false;
  // Blocks of all sequences, those with the most keys first, so that the last ones to start are short.  Up to 32
  // sequences (a lane for each) are put in that order: more(c) is how many blocks of the lane's sequence have more
  // than c key tiles in front of their last query, and the place is found by bisection over c.  More sequences are
  // taken from the last one's last block on.
  int nqs = 0, nks = 0;
  auto blocks_of = [&](int i) {
    nqs = i < a.n_seqs ? max(0, min(a.cu_q[i + 1], a.total_q) - max(0, a.cu_q[i])) : 0;
    return (nqs + per - 1) / per;
  };
  const int n0 = blocks_of(lane);          // of the first 32, kept
  int total = __reduce_add_sync(0xffffffffu, n0);
  for (int b = 32; b < a.n_seqs; b += 32) total += __reduce_add_sync(0xffffffffu, blocks_of(b + lane));
  if (index >= total) return p;
  // number `index` of the lanes' n candidates: its lane, and k, the how manieth of that lane's (-1: it is behind them)
  int k = 0;
  auto pick = [&](int n) {
    int inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, index < inc);
    const int l = hit ? __ffs(hit) - 1 : 31;
    k = index - __shfl_sync(0xffffffffu, hit ? inc - n : inc, l);
    return hit ? l : -1;
  };
  if (a.n_seqs > 1 && a.n_seqs <= 32) {
    nks = lane < a.n_seqs ? max(0, min(a.cu_k[lane + 1], a.total_k) - max(0, a.cu_k[lane])) : 0;
    auto more = [&](int c) {               // blocks whose last query stands at key c BN or later
      const int need = c * S::BN - (nks - nqs) + 1;          // tokens up to and with that query
      return c < 0 || need <= 0 ? n0 : need > nqs ? 0 : n0 - (need - 1) / per;
    };
    int lo = 0, hi = __reduce_max_sync(0xffffffffu, nks) / S::BN + 1;   // the least c with more(c) <= index in all
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if ((int)__reduce_add_sync(0xffffffffu, more(mid)) <= index) hi = mid;
      else lo = mid + 1;
    }
    const int above = more(lo);
    index -= __reduce_add_sync(0xffffffffu, above);
    p.seq = pick(more(lo - 1) - above);
    p.t0 = (__shfl_sync(0xffffffffu, n0 - above - 1, p.seq) - k) * per;
  } else {
    index = total - 1 - index;
    p.seq = -1;
    for (int b = 0; b < a.n_seqs; b += 32) {
      const int l = pick(b ? blocks_of(b + lane) : n0);
      if (l >= 0) {
        p.seq = b + l;
        p.t0 = k * per;
        break;
      }
      index = k;
    }
    if (p.seq < 0) return p;
  }
  p.q0 = a.cu_q[p.seq]; p.q1 = a.cu_q[p.seq + 1];
  p.k0 = a.cu_k[p.seq]; p.k1 = a.cu_k[p.seq + 1];
  if (p.q0 < 0 || p.q1 > a.total_q || p.k0 < 0 || p.k1 < p.k0 || p.k1 > a.total_k) {
    if (threadIdx.x == 0) atomicOr(err, EF_BAD_INDEX);
    return p;
  }
  const int nk = p.k1 - p.k0, nq = p.q1 - p.q0;
  const int hi = nk - nq + min(nq, p.t0 + per) - 1;      // last key of the block's last query
  const int lo = a.window > 0 ? max(0, nk - nq + p.t0 - a.window + 1) : 0;
  p.first = lo / S::BN;
  p.tiles = hi < lo ? 0 : hi / S::BN - p.first + 1;
  p.ok = true;
  return p;
}

// ---- between the blocks of a pair ----
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
// Arrive on the same mbarrier of the block with rank 0.  What the arrival stands for was done by TMA or is in tensor
// memory (ordered by tcgen05.fence), so it needs no release of ordinary memory at cluster scope, which costs about a
// thousand cycles; the one place where it stands for ordinary stores fences by itself.
__device__ __forceinline__ void arrive_at_first(uint64_t* bar) {
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }

template <class T, int HD, int CL>
__global__ void __launch_bounds__(Shape<HD, CL>::THREADS, 1)
    prompt_attn_kernel(const ms_prompt_attn a, const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                       const __grid_constant__ CUtensorMap v_map, int n_tok, uint32_t* err) {
  using S = Shape<HD, CL>;
  constexpr int NQ = S::NQ, BN = S::BN, ST = S::STAGES, BLK = HD / 64;   // BLK: blocks of 64 dims
  constexpr bool BF16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
  extern __shared__ uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *sq = sm, *sk = sq + NQ * S::Q_BYTES, *sv = sk + ST * S::KV_BYTES;
  // *_other (rank 0 of a pair): the other block's share has arrived, too
  __shared__ uint64_t q_full, q_other, k_full[ST], k_other[ST], k_empty[ST], v_full[ST], v_other[ST], v_empty[ST], s_full[2], p_full[2],
      o_full[NQ], ended;
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CL == 2 ? cluster_rank() : 0, index = blockIdx.x / CL;
  const int head = index % a.kv_heads, rep = a.heads / a.kv_heads;
  if (warp == S::SOFTMAX_WARPS + 1 && lane < 3) prefetch_map(lane == 0 ? &q_map : lane == 1 ? &k_map : &v_map);
  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_other, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1); mbar_init(&k_other[i], 1); mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1); mbar_init(&v_other[i], 1); mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4 * CL); }
    for (int i = 0; i < NQ; ++i) mbar_init(&o_full[i], 1);
    mbar_init(&ended, 1);
    fence_mbar_init();
  }
  pdl_wait_prior();
  pdl_launch_dependents();
  if (warp == S::SOFTMAX_WARPS) umma::alloc_cg<CL>(&tmem_base, S::COLS);   // after the wait: the predecessor may hold it
  const Place pl = find_place<HD, CL>(a, n_tok, index / a.kv_heads, err);
  umma::fence_before_sync();
  __syncthreads();
  if (CL == 2) cluster_sync();
  umma::fence_after_sync();
  // the first blocks' (of a pair) last warps, which copy and multiply nothing, look the offsets over together
  auto look_over = [&]() {
    const int at = index * 32, step = gridDim.x / CL * 32;
    if (!offsets_ok(a.cu_q, a.n_seqs, a.total_q, at, step) || !offsets_ok(a.cu_k, a.n_seqs, a.total_k, at, step)) atomicOr(err, EF_BAD_INDEX);
  };
  if (!pl.ok) {                            // all threads, in both blocks of a pair
    if (warp == S::SOFTMAX_WARPS + 3 && rank == 0) look_over();
    if (warp == S::SOFTMAX_WARPS) umma::dealloc_cg<CL>(tmem_base, S::COLS);
    return;
  }
  constexpr uint32_t tmem = 0;             // all 512 columns are this block's, so they start at 0
  if (threadIdx.x == 0 && tmem_base != tmem) atomicOr(err, EF_BAD_SHAPE);
  const int nq = pl.q1 - pl.q0, nk = pl.k1 - pl.k0;
  // query tile i of this block begins at token t0 + (i + rank) n_tok; slots: the block's tiles that have rows
  const int slots = NQ == 2 && pl.t0 + n_tok < nq ? 2 : 1;

  // the two softmax groups need more than the 168 registers of 384 threads: 208 x 256 + 80 x 128 of 168 x 384
  if (warp >= S::SOFTMAX_WARPS) {
    if (NQ == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // (a wait that runs out does so for the whole warp)
    auto wait = [&](uint64_t* bar, int parity) {
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity & 1, err, EF_TIMEOUT_FULL));
    };
    // rows of V behind the sequence's end are rows of others: zeroed (16-byte units of 128-byte rows)
    auto clear_tail = [&](int j) {
      const int keys = nk - (pl.first + j) * BN, bad = BN - keys;
      if (bad <= 0) return false;
      for (int i = lane; i < bad * 8 * S::V_BLOCKS; i += 32) {
        const int b = i / (bad * 8), u = i % (bad * 8);
        *reinterpret_cast<uint4*>(sv + j % ST * S::KV_BYTES + b * BN * 128 + keys * 128 + u * 16) = make_uint4(0, 0, 0, 0);
      }
      umma::fence_proxy_async_smem();
      __syncwarp();
      return true;
    };
    // the first of the four warps issues the MMAs, the next two the copies of K and of V; in the other block of a pair the
    // first and the last tell the first block what has arrived
    const int role = warp - S::SOFTMAX_WARPS;
    if (role == 1 || role == 2) {
      // ---- TMA: Q and K, or V ----
      if (lane == 0 && pl.tiles > 0) {
        uint64_t *full = role == 1 ? k_full : v_full, *empty = role == 1 ? k_empty : v_empty;
        if (role == 1) {
          const int rows = n_tok * rep;
          mbar_expect_tx(&q_full, slots * BLK * rows * 128);
          for (int i = 0; i < slots; ++i)
            for (int b = 0; b < BLK; ++b)
              tma_3d(sq + i * S::Q_BYTES + b * 128 * 128, &q_map, 64 * b, head * rep, pl.q0 + pl.t0 + (i + rank) * n_tok, &q_full);
        }
        int j = 0;
        for (; j < pl.tiles; ++j) {
          const int st = j % ST, z = pl.k0 + (pl.first + j) * BN;
          if (j >= ST && !mbar_wait(&empty[st], (j / ST - 1) & 1, err, EF_TIMEOUT_EMPTY)) break;
          mbar_expect_tx(&full[st], S::KV_BYTES);
          if (role == 1) {
            for (int b = 0; b < BLK; ++b)
              tma_3d(sk + st * S::KV_BYTES + b * S::K_ROWS * 128, &k_map, 64 * b, head, z + rank * S::K_ROWS, &full[st]);
          } else {
            for (int b = 0; b < S::V_BLOCKS; ++b)
              tma_3d(sv + st * S::KV_BYTES + b * BN * 128, &v_map, 64 * (rank * S::V_BLOCKS + b), head, z, &full[st]);
          }
        }
        // nothing of this block may still be on its way when it ends, also where another warp has given up
        if (role == 1) mbar_wait(&q_full, 0, err, EF_TIMEOUT_FULL);
        for (int k = first_under_way(j, ST); k < j; ++k) mbar_wait(&full[k % ST], fill_phase(k, ST) & 1, err, EF_TIMEOUT_FULL);
      }
    } else if (rank == 1) {
      // ---- the other block of a pair: Q and K, or V ----
      bool alive = pl.tiles > 0;
      if (alive && role == 0) {
        alive = wait(&q_full, 0);
        if (alive && lane == 0) arrive_at_first(&q_other);
      }
      for (int j = 0; j < pl.tiles && alive; ++j) {
        alive = wait(role == 0 ? &k_full[j % ST] : &v_full[j % ST], fill_phase(j, ST));
        if (!alive) break;
        if (role == 3 && clear_tail(j)) fence_cluster();
        if (lane == 0) arrive_at_first(role == 0 ? &k_other[j % ST] : &v_other[j % ST]);
      }
    } else if (role == 3) {
      look_over();
    } else if (role == 0) {
      // ---- MMA: the whole warp walks, one thread issues ----
      constexpr uint32_t id_s = umma::idesc_f16(128 * CL, BN, BF16, false), id_o = umma::idesc_f16(128 * CL, HD, BF16, true);
      // descriptors of the first tiles; others are that many 16-byte units further
      const uint64_t dq = umma::smem_desc_sw128(sq, 0), dk = umma::smem_desc_sw128(sk, 0), dv = umma::smem_desc_sw128(sv, BN * 128);
      const bool one = umma::elect();
      // A step is the value product of a query tile and the scores after it.  slot is a constant: its addresses are, too.
      bool alive = pl.tiles > 0;
      auto need = [&](uint64_t* bar, uint64_t* bar_other, int parity) {
        alive = alive && wait(bar, parity) && (CL == 1 || bar_other == nullptr || wait(bar_other, parity));
      };
      auto need_k = [&](int j) {
        if (j < pl.tiles) need(&k_full[j % ST], &k_other[j % ST], fill_phase(j, ST));
      };
      auto need_v = [&](int j) {
        need(&v_full[j % ST], &v_other[j % ST], fill_phase(j, ST));
        if (alive && clear_tail(j) && CL == 2) fence_cluster();
      };
      auto scores = [&](auto slot_c, int j) {                // one thread; K of tile j has arrived
        constexpr int slot = decltype(slot_c)::value;
        const int st = j % ST;
        if (NQ == 1 || slot < slots) {
          const uint64_t q = dq + (NQ == 2 ? slot : 0) * (S::Q_BYTES >> 4), k = dk + st * (S::KV_BYTES >> 4);
#pragma unroll
          for (int b = 0; b < BLK; ++b)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma::mma_ss<CL>(slot * BN, q + (b * 128 * 128 + kk * 32) / 16, k + (b * S::K_ROWS * 128 + kk * 32) / 16, id_s, b || kk);
          umma::commit_cg<CL>(&s_full[slot]);
        }
        // (a place is released only where a copy waits for it: no arrival is left open at the end)
        if ((NQ == 1 || slot == 1) && j + ST < pl.tiles) umma::commit_cg<CL>(&k_empty[st]);
      };
      auto values = [&](auto slot_c, int j) {                // one thread; V of tile j and the slot's probabilities are there
        constexpr int slot = decltype(slot_c)::value;
        const int st = j % ST;
        if (NQ == 1 || slot < slots) {
          const uint64_t v = dv + st * (S::KV_BYTES >> 4);
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma::mma_ts<CL>(S::O_COL + (NQ == 2 ? slot * HD : 0), S::P_COL + slot * S::P_STEP + kk * 8, v + kk * 2048 / 16, id_o,
                             j > 0 || kk > 0);
          umma::commit_cg<CL>(&o_full[NQ == 2 ? slot : 0]);
        }
        if ((NQ == 1 || slot == 1) && j + ST < pl.tiles) umma::commit_cg<CL>(&v_empty[st]);
      };
      constexpr std::integral_constant<int, 0> s0;
      constexpr std::integral_constant<int, 1> s1;
      constexpr int AHEAD = NQ == 2 ? 1 : 2;                 // key tiles that the scores are ahead of the values
      // A poll costs about 100 cycles even when it finds what it waits for.  The MMAs of 64 dims take little longer, so
      // their step waits for all that it needs and then issues both products in one go (64 heads over 4,096 tokens:
      // 215 us for 233); those of 128 dims start sooner with the keys waited for between the products (16,384 tokens:
      // 1,704 us for 1,742), and 256 dims have no third place for keys (2,048 behind 9,001: 237 us for 266).
      constexpr bool GO = HD == 64;
      auto step = [&](auto slot_c, int j) {
        constexpr int slot = decltype(slot_c)::value;
        if (!alive || j >= pl.tiles) return;
        if (GO && slot == 0) need_k(j + 1);
        if (NQ == 1 || slot == 0) need_v(j);
        if (NQ == 1 || slot < slots) need(&p_full[slot], nullptr, NQ == 2 ? j : j >> 1);   // how often it was filled before
        if (!alive) return;
        umma::fence_after_sync();
        if (one) {
          values(slot_c, j);
          if (GO && j + 1 < pl.tiles) scores(slot_c, j + 1);
        }
        __syncwarp();
        if (GO || j + AHEAD >= pl.tiles) return;
        if (NQ == 1 || slot == 0) need_k(j + AHEAD);
        if (!alive) return;
        umma::fence_after_sync();
        if (one) scores(slot_c, j + AHEAD);
        __syncwarp();
      };
      need(&q_full, &q_other, 0);
      need_k(0);
      if (alive) {
        umma::fence_after_sync();
        if (one) {
          scores(s0, 0);
          if (NQ == 2) scores(s1, 0);
        }
        __syncwarp();
      }
      if (NQ == 1 && pl.tiles > 1) {
        need_k(1);
        if (alive) {
          umma::fence_after_sync();
          if (one) scores(s1, 1);
          __syncwarp();
        }
      }
      for (int j = 0; j < pl.tiles && alive; j += AHEAD) {
        step(s0, j);
        step(s1, NQ == 2 ? j : j + 1);
      }
      if (pl.tiles > 0 && !alive) {                          // a wait ran out: the products under way end before the block does
        if (one) umma::commit_here<CL>(&ended);
        __syncwarp();
        wait(&ended, 0);
      }
    }
  } else {
    // ---- softmax: thread = row ----
    if (NQ == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int tile = warp >> 2, r = threadIdx.x & 127;       // query tile of the block, row of it
    const int tok = pl.t0 + (tile + rank) * n_tok + r / rep;   // token of the sequence
    const bool row_ok = r < n_tok * rep && tok < nq;
    const int h = head * rep + r % rep;
    const int last = row_ok ? nk - nq + tok : -1;            // the row's last key
    const int lo = a.window > 0 ? max(0, last - a.window + 1) : 0;
    const float c2 = fmaxf(a.scale * kLog2e, 1e-37f);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_col = tmem + lanes + S::O_COL + (NQ == 2 ? tile * HD : 0);
    float m = kNone, l = 0.f;
    bool alive = true;
    auto wait = [&](uint64_t* bar, int parity) {
      return (bool)__all_sync(0xffffffffu, mbar_wait(bar, parity & 1, err, EF_TIMEOUT_FULL));
    };
    if (tile < slots) {
      for (int j = 0; j < pl.tiles; ++j) {
        const int slot = NQ == 2 ? tile : j & 1, turn = NQ == 2 ? j : j >> 1;
        alive = wait(&s_full[slot], turn);
        if (!alive) break;
        umma::fence_after_sync();
        const uint32_t s_col = tmem + lanes + slot * BN, p_col = tmem + lanes + S::P_COL + slot * S::P_STEP;
        const int key0 = (pl.first + j) * BN;
        uint32_t u[BN];
        auto load = [&]() {                                  // the scores, masked
#pragma unroll
          for (int i = 0; i < BN / 32; ++i) umma::ld_32x32b_x32_async(s_col + 32 * i, u + 32 * i);
          umma::wait_ld();
#pragma unroll
          for (int i = 0; i < BN / 32; ++i) umma::loaded(u + 32 * i);
          if (!__all_sync(0xffffffffu, key0 >= lo && key0 + BN - 1 <= last)) {
#pragma unroll
            for (int i = 0; i < BN; ++i)
              if (key0 + i > last || key0 + i < lo) u[i] = 0xFF800000u;   // -inf
          }
        };
        auto raise_max = [&]() {                             // to the tile's, with the sum and the output so far
          float top4[4];                                     // four chains
#pragma unroll
          for (int i = 0; i < 4; ++i) top4[i] = fmaxf(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
#pragma unroll
          for (int i = 8; i < BN; i += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) top4[e] = max3(top4[e], __uint_as_float(u[i + 2 * e]), __uint_as_float(u[i + 2 * e + 1]));
          const float top = fmaxf(fmaf(fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3])), c2, -Range<T>::below), m), f = exp2_fast(m - top);
          m = top;
          l *= f;
          return f;
        };
        auto exps = [&]() {                                  // u becomes pairs of probabilities; their sum
          const uint64_t c22 = pair(c2, c2), m22 = pair(-m, -m);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < BN; i += 2) {
            float2 e = unpair(fma2(pair(__uint_as_float(u[i]), __uint_as_float(u[i + 1])), c22, m22));
            e.x = exp2_fast(e.x);
            e.y = exp2_fast(e.y);
            sum[i / 2 & 1] = add2(sum[i / 2 & 1], pair(e.x, e.y));
            u[i / 2] = pack2<T>(e.x, e.y);
          }
          const float2 both = unpair(add2(sum[0], sum[1]));
          return both.x + both.y;
        };
        load();
        if (j == 0) raise_max();
        float sum = exps();
        if (__any_sync(0xffffffffu, sum > Range<T>::raise)) {         // (not with the first tile, whose maximum was taken)
          load();
          const float f = raise_max();
          sum = exps();
          if (j > 0) {
            // all value products of this output so far have to be done: with NQ = 2 the scores' arrival says so
            if (NQ == 1) alive = wait(&o_full[0], j - 1);
            if (!alive) break;
            umma::fence_after_sync();
#pragma unroll
            for (int i = 0; i < HD / 32; ++i) {
              uint32_t o[32];
              umma::ld_32x32b_x32_async(o_col + 32 * i, o);
              umma::wait_ld();
              umma::loaded(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              umma::st_32x32b_x32(o_col + 32 * i, o);
            }
          }
        }
        l += sum;
#pragma unroll
        for (int i = 0; i < BN / 64; ++i) umma::st_32x32b_x32(p_col + 32 * i, u + 32 * i);
        umma::wait_st();
        if (NQ == 1 && waits_before_handover(j, pl.tiles)) alive = wait(&o_full[0], j - 1);
        if (!alive) break;
        umma::fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (CL == 1) mbar_arrive(&p_full[slot]);
          else arrive_at_first(&p_full[slot]);
        }
      }
      // ---- output ----
      // A wait on a phase's parity tells it from the one before only: the scores of tile j vouch for the value products
      // up to j - 1 (NQ = 2) or j - 2, so with NQ = 1 the last but one was waited for before the last hand-over.
      if (pl.tiles > 0 && alive) alive = wait(&o_full[NQ == 2 ? tile : 0], pl.tiles - 1);
      umma::fence_after_sync();
      float f = 0.f;
      if (l > 0.f) {
        float den = l;
        f = 1.f;
        if (a.sinks) {
          const float sink = a.sinks[h] * kLog2e, mm = fmaxf(m, sink);
          f = exp2_fast(m - mm);
          den = l * f + sink_share(sink, mm);
        }
        f /= den;
      }
      T* dst = (T*)a.out + (int64_t)(pl.q0 + tok) * a.out_stride + h * HD;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        uint32_t o[32];
        if (pl.tiles > 0 && alive) {
          umma::ld_32x32b_x32_async(o_col + 32 * i, o);
          umma::wait_ld();
          umma::loaded(o);
        }
        if (row_ok && alive) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = l > 0.f || l != l ? __uint_as_float(o[e + k]) * f : 0.f;
            store8(dst + 32 * i + e, x);
          }
        }
      }
    }
  }
  umma::fence_before_sync();
  __syncthreads();
  if (CL == 2) cluster_sync();             // no arrival may find a block that has ended
  umma::fence_after_sync();
  if (warp == S::SOFTMAX_WARPS) umma::dealloc_cg<CL>(tmem, S::COLS);
}

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeFn)p;
  }();
  return fn;
}

// [tokens][heads][hd] with `stride` elements between tokens; boxes of 64 dims, `heads_box` heads, `tokens_box` tokens
bool make_map(CUtensorMap* map, bool bf16, const void* p, int hd, int heads, int tokens, int64_t stride, int heads_box,
              int tokens_box) {
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)heads_box, (cuuint32_t)tokens_box}, unit[3] = {1, 1, 1};
  return encoder()(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims,
                   strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int HD, int CL>
cudaError_t start(const DevCtx& d, const ms_prompt_attn& a, cudaStream_t s) {
  using S = Shape<HD, CL>;
  const int rep = a.heads / a.kv_heads, n_tok = 128 / rep;
  const bool bf16 = a.type == MS_Q_BF16;
  if (!encoder()) return cudaErrorNotSupported;
  CUtensorMap q, k, v;
  if (!make_map(&q, bf16, a.q, HD, a.heads, a.total_q, a.q_stride, rep, n_tok)) return cudaErrorInvalidValue;
  if (a.total_k == 0) k = v = q;   // no block has a key tile
  else if (!make_map(&k, bf16, a.k, HD, a.kv_heads, a.total_k, a.k_stride, 1, S::K_ROWS) ||
           !make_map(&v, bf16, a.v, HD, a.kv_heads, a.total_k, a.v_stride, 1, S::BN))
    return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(prompt_attn_kernel<T, HD, CL>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  if (e != cudaSuccess) return e;
  // blocks (pairs) of all sequences: at most one that is not full for each
  const int64_t places = ((int64_t)a.total_q / (CL * S::NQ * n_tok) + a.n_seqs) * a.kv_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(places * CL));
  cfg.blockDim = dim3(S::THREADS);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  if (CL == 2) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CL;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  } else {                                 // may start while its predecessor in the stream ends
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
  }
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, prompt_attn_kernel<T, HD, CL>, a, q, k, v, n_tok, d.err);
}

template <class T>
cudaError_t start_hd(const DevCtx& d, const ms_prompt_attn& a, cudaStream_t s) {
  if (a.head_dim == 64) return start<T, 64, 1>(d, a, s);
  if (a.head_dim == 128) return start<T, 128, 1>(d, a, s);
  return start<T, 256, 2>(d, a, s);
}

}  // namespace

cudaError_t launch_prompt_attention(const DevCtx& d, const ms_prompt_attn& a, cudaStream_t s) {
  if (a.total_q == 0 || a.n_seqs == 0) return cudaSuccess;
  return a.type == MS_Q_F16 ? start_hd<__half>(d, a, s) : start_hd<__nv_bfloat16>(d, a, s);
}

}  // namespace ms
