// A word between two blocks of a launch: one leaves sums in memory and sets the word to the call's tag, the other waits for it, for a limited time.
//
// A captured call has the same tag in every replay, so whatever happens the word is back to zero when both blocks have ended: the one that waits takes
// the tag back, or leaves its complement where it has given up; the one that sets the tag finds that in its place and takes its own tag back.  Each word has
// one of either in a launch.  `Word` has wait (false: in vain), exchange and store; the test has one of its own.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define HG_WORD __device__ __forceinline__
#else
#define HG_WORD inline
#endif

namespace hg {

template <typename Word>
HG_WORD bool take_tag(Word& word, uint64_t tag) {
  if (word.wait(tag)) {
    word.store(0);
    return true;
  }
  if (word.exchange(~tag) == tag) word.store(0);   // it was set after all; too late
  return false;
}

// What stood there before, which goes to `settle_tag` some time before the block ends.
template <typename Word>
HG_WORD uint64_t leave_tag(Word& word, uint64_t tag) { return word.exchange(tag); }
template <typename Word>
HG_WORD void settle_tag(Word& word, uint64_t tag, uint64_t before) {
  if (before == ~tag) word.store(0);
}

}  // namespace hg
