// What a warp keeps of its ring of asynchronous loads, apart from the instructions that load and wait, so that it can be
// followed without a GPU.  Load i goes to stage i % STAGES and completes phase i / STAGES of that stage's barrier; a wait
// is bounded and says whether the phase completed.
//
// A wait that ran out ends the ring: its stage may still be written to, so nothing more is loaded (a barrier whose phase is
// under way must not be armed again) and nothing more is taken, and before the block leaves, drain() waits, bounded
// again, for every load still under way: none should land in shared memory that already belongs to another block.
#pragma once

#ifdef __CUDACC__
#define SIAR_RING_FN __device__ __forceinline__
#else
#define SIAR_RING_FN inline
#endif

namespace siar {

template <int STAGES>
struct LoadRing {
  int issued = 0, taken = 0;
  bool expired = false;

  SIAR_RING_FN bool room() const { return !expired && issued - taken < STAGES; }
  SIAR_RING_FN int next() { return issued++ % STAGES; }             // the stage of the next load (where there is room)
  SIAR_RING_FN int stage() const { return taken % STAGES; }         // the stage of the oldest one
  SIAR_RING_FN void release() { ++taken; }                          // its data has been read
  // wait(stage, parity): true when that phase has completed.  False from the first wait on that ran out.
  template <typename Wait>
  SIAR_RING_FN bool take(Wait wait) {
    if (!expired && !wait(taken % STAGES, (taken / STAGES) & 1)) expired = true;
    return !expired;
  }
  template <typename Wait>
  SIAR_RING_FN void drain(Wait wait) {
    for (; taken < issued; ++taken) wait(taken % STAGES, (taken / STAGES) & 1);
  }
};

}  // namespace siar
