// A warp's ring of bulk copies (w4_linear.cu): which place is asked for next and which is read next.  Plain C++, so that its
// order can be run on the CPU.
//
// Where a wait gives up, nothing more is asked for: so a place whose copy is still to come is never asked for again, and what is
// under way are the copies from the lost place on, up to the place that would have been asked for next.  Each of them is waited
// for before the block ends.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define W4_RING_FN __host__ __device__ __forceinline__
#else
#define W4_RING_FN inline
#endif

namespace mvb {

struct W4Ring {
  int pair;            // next pair of tiles to ask for, kStopped behind a wait that gave up
  int fill = 0;        // place of the next copy
  int read = 0;        // place of the next item
  uint32_t phase = 0;  // the parity of its barrier to wait for
  static constexpr int kStopped = 0x7fffffff;
  W4_RING_FN explicit W4Ring(int first) : pair(first) {}
  W4_RING_FN void asked(int stages) { fill = fill + 1 == stages ? 0 : fill + 1; }
  W4_RING_FN void next(int stages) {
    if (++read == stages) read = 0, phase ^= 1u;
  }
  // A wait gave up: the first one's place goes to `lost`.
  W4_RING_FN void stop(int& lost) {
    if (pair != kStopped) lost = read | static_cast<int>(phase << 8);
    pair = kStopped;
  }
  W4_RING_FN bool stopped() const { return pair == kStopped; }
  W4_RING_FN void back(int lost) { read = lost & 255, phase = static_cast<uint32_t>(lost >> 8); }
  // Whether another copy is under way after the one at `read`, which has been waited for.
  W4_RING_FN bool more(int stages) {
    next(stages);
    return read != fill;
  }
};

}  // namespace mvb
