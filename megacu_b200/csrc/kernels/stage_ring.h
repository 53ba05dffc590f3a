// What is left to wait for when a producer stops in the middle of its ring of
// shared-memory stages. Load i (a producer counts its loads from 0) goes into
// stage i % stages and completes that stage's `full` barrier for the
// (i / stages)-th time.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define MEGACU_RING_FN __device__ __forceinline__
#else
#define MEGACU_RING_FN inline
#endif

namespace megacu_b200 {

// Waits for the last load of every stage: ops.wait(stage, parity). Every
// earlier load of a stage had landed before the stage was loaded again.
template <class Ops>
MEGACU_RING_FN void drain_ring(std::uint32_t issued, std::uint32_t stages, Ops &&ops) {
  for (std::uint32_t i = issued > stages ? issued - stages : 0; i < issued; ++i) {
    ops.wait(i % stages, i / stages & 1u);
  }
}

// The same for two CTAs whose loads count on the leader's barriers. Each load
// of the leader announces both CTAs' bytes, so that where one producer stopped
// before the other, the barriers first lose the follower's announced bytes
// that never come (ops.complete) or learn of those that were not announced
// (ops.announce). Neither CTA is more than one ring ahead, hence one such
// load per stage.
template <class Ops>
MEGACU_RING_FN void drain_pair_ring(std::uint32_t leader, std::uint32_t follower,
                                           std::uint32_t stages, Ops &&ops) {
  for (std::uint32_t i = leader; i < follower; ++i) ops.announce(i % stages);
  for (std::uint32_t i = follower; i < leader; ++i) ops.complete(i % stages);
  drain_ring(leader > follower ? leader : follower, stages, ops);
}

}  // namespace megacu_b200

#undef MEGACU_RING_FN
