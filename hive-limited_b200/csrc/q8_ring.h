// One warp's walk over blocks whose copies pass through a ring of its own: kStages are under way
// before it starts, and a block's place is filled again once the block has been used.
//
// A wait can run out. Then nothing more is used or copied, and every copy that is under way is
// waited for (again with a limit), so that none writes to the ring after the walk has ended.
// Apart from the kernel that has it, so that the order of waits and copies is tested on the CPU.
#pragma once

#ifdef __CUDACC__
#define HV_RING __device__ __forceinline__
#else
#define HV_RING inline
#endif

namespace hv {

// Blocks b, b + step, ... below end, the first kStages of them copied already (those there are), to
// places 0, 1, ... wait(place, parity): false when it ran out; fetch(block, place) is called for
// blocks past the end as well, and copies nothing then. False when a wait ran out.
template <int kStages, class Wait, class Fetch, class Use>
HV_RING bool ring_walk(int b, int end, int step, const Wait& wait, const Fetch& fetch, const Use& use) {
  int stage = 0, parity = 0;
  auto next = [&] {
    stage = stage + 1 == kStages ? 0 : stage + 1;
    parity ^= stage == 0;
  };
  for (; b < end; b += step) {
    if (!wait(stage, parity)) {
      for (int i = 0; i < kStages && b + i * step < end; ++i) {
        wait(stage, parity);
        next();
      }
      return false;
    }
    use(b, stage);
    fetch(b + kStages * step, stage);
    next();
  }
  return true;
}

}  // namespace hv
