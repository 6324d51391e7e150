// phases.h — where the kernels wait on an mbarrier, and for which of its phases.  A wait names a phase by its parity, so
// it tells the phase that it means from the one in front of it only: when the barrier is already one phase further, the
// wait does not pass.  These are plain functions of counters, which the host can walk through, too.
#pragma once

#ifdef __CUDACC__
#define MS_PHASES_FN __host__ __device__ constexpr
#else
#define MS_PHASES_FN constexpr
#endif

namespace ms {

// Prompt attention, one query tile to a block: o_full completes a phase with each key tile's value product, and the product of tile j
// starts when all softmax warps have handed over tile j's probabilities.  Behind the last tile a warp waits for the
// last product; for the one before it it has to wait while its own last probabilities still hold the last one
// back.  True at the tile in front of whose hand-over that wait stands.
MS_PHASES_FN bool waits_before_handover(int tile, int tiles) { return tile > 0 && tile + 1 == tiles; }

// A ring of stages, filled and emptied in turn: fill k goes to stage k % stages and completes this phase of its barrier.
MS_PHASES_FN int fill_phase(int k, int stages) { return k / stages; }
// The first of so many fills that may be under way still: a stage is filled again when its last fill has been used.
MS_PHASES_FN int first_under_way(int fills, int stages) { return fills > stages ? fills - stages : 0; }

}  // namespace ms
