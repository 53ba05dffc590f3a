// What the kernel's drains do (test infrastructure): the operations of
// drain_ring / drain_pair_ring in order, as (kind, stage, parity) triples with
// kind 0 = wait, 1 = announce, 2 = complete. Returns how many there are, at
// most `room` are stored.
#include <cstdint>

#include "kernels/stage_ring.h"

namespace {

struct recorder {
  std::uint32_t *out;
  std::uint32_t room, count;
  void add(std::uint32_t kind, std::uint32_t stage, std::uint32_t parity) {
    if (count < room) {
      out[3 * count] = kind;
      out[3 * count + 1] = stage;
      out[3 * count + 2] = parity;
    }
    ++count;
  }
  void wait(std::uint32_t stage, std::uint32_t parity) { add(0, stage, parity); }
  void announce(std::uint32_t stage) { add(1, stage, 0); }
  void complete(std::uint32_t stage) { add(2, stage, 0); }
};

}  // namespace

extern "C" std::uint32_t ring_drain_ops(std::uint32_t pair, std::uint32_t leader,
                                        std::uint32_t follower, std::uint32_t stages,
                                        std::uint32_t *out, std::uint32_t room) {
  recorder r{out, room, 0};
  if (pair != 0) {
    megacu_b200::drain_pair_ring(leader, follower, stages, r);
  } else {
    megacu_b200::drain_ring(leader, stages, r);
  }
  return r.count;
}
