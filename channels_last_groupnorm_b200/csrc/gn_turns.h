// How the two CTAs of a pair (gn_linear4.cu) end when a bounded wait has run out: plain C++, for the kernel and for tests on the host.
#pragma once

#if defined(__CUDACC__)
#define GNB200_BOTH __host__ __device__ __forceinline__
#else
#define GNB200_BOTH inline
#endif

namespace gnb200 {

// A warp's turns at the sums of one tile after the other.  After the first that did not come there is none: the barrier still stands in that
// turn's phase, so that a look for the next turn's parity would find the phase before it, complete, with sums that are old or half done.  Nor does such
// a warp say that it has taken anything, which would let the next products overwrite what other warps have not read.
struct Turns {
  bool gone = false;
  GNB200_BOTH bool take(bool there) {
    gone = gone || !there;
    return !gone;
  }
};

// What both CTAs know of each other at their end where a wait ran out
struct PairEnd {
  int loads[2];               // K tiles that the leader and its peer asked for
  int multiplied, announced;  // K tiles whose products have an arrival at `empty`, tiles with one at `sums`
};

// K tile k's copies as the leader's barrier has them, which counts those of both CTAs: which of its steps are missing where one CTA stopped in front of the other.
enum Missing { kNothing, kAnnouncement, kPeersBytes };  // ... nobody announced the peer's bytes; they were announced and the peer never asked for them
GNB200_BOTH Missing missing_of(int k, int leaders_loads, int peers_loads) { return k >= leaders_loads ? kAnnouncement : k >= peers_loads ? kPeersBytes : kNothing; }
// The first K tile whose copies, or arrival, may be under way when that many were begun (the stage of one before was taken again), and the end of the pair's copies
GNB200_BOTH int drain_begin(int count, int stages) { return count > stages ? count - stages : 0; }
GNB200_BOTH int drain_end(int leaders_loads, int peers_loads) { return leaders_loads > peers_loads ? leaders_loads : peers_loads; }

}  // namespace gnb200
