"""The words by which a unit's blocks meet (csrc/hg_tags.cuh), in every order that one block's accesses can come in between the other's.

The header is compiled for the host with a word that lets the block that sets the tag take its two steps before a chosen access of the one that waits."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "comp2029-hybridgemm_b200" / "csrc"

HARNESS = r"""
#include <functional>
#include "hg_tags.cuh"

constexpr int kPolls = 3, kAccesses = kPolls + 2;
struct Slot {
  uint64_t value;
  std::function<void()> turn = [] {};   // ahead of every access
  bool wait(uint64_t tag) {
    for (int i = 0; i < kPolls; ++i) { turn(); if (value == tag) return true; }
    return false;
  }
  uint64_t exchange(uint64_t to) { turn(); const uint64_t before = value; value = to; return before; }
  void store(uint64_t to) { turn(); value = to; }
};

// One launch: the sums are left ahead of access `left` of the block that waits, the word is looked at again ahead of access `settled`; plain: a store sets the
// tag, another takes it back.
static bool launch(uint64_t& word, uint64_t tag, int left, int settled, bool plain, bool* was_left) {
  Slot waiting{word};
  Slot other{0};
  int access = 0;
  bool gave = false, looked = false;
  uint64_t before = 0;
  auto step = [&](int at) {
    if (!gave && left <= at) {
      gave = true;
      other.value = waiting.value;
      if (plain) other.store(tag);
      else before = hg::leave_tag(other, tag);
      waiting.value = other.value;
    }
    if (gave && !looked && settled <= at) {
      looked = true;
      other.value = waiting.value;
      if (!plain) hg::settle_tag(other, tag, before);
      waiting.value = other.value;
    }
  };
  waiting.turn = [&] { step(access++); };
  bool taken;
  if (plain) { taken = waiting.wait(tag); waiting.store(0); }
  else taken = hg::take_tag(waiting, tag);
  *was_left = gave;
  step(1 << 20);
  word = waiting.value;
  return taken;
}

// Orders after which the word is not back to zero, or a launch found sums that were not there yet: three launches of one tag.
extern "C" int failures(uint64_t tag, uint64_t garbage, int plain) {
  int bad = 0;
  for (int left = 0; left <= kAccesses; ++left)
    for (int settled = left; settled <= kAccesses; ++settled)
      for (int next = 0; next <= kAccesses; ++next) {
        uint64_t word = garbage;
        bool there, wrong = false;
        for (int i = 0; i < 3; ++i) {
          const bool taken = i == 1 ? launch(word, tag, next, next, plain, &there) : launch(word, tag, left, settled, plain, &there);
          wrong |= (taken && !there) || word != 0;
          if ((i == 1 ? next : left) < kPolls) wrong |= !taken;   // it came in time
        }
        bad += wrong;
      }
  return bad;
}
"""


@pytest.fixture(scope="module")
def failures(tmp_path_factory):
    folder = tmp_path_factory.mktemp("tags")
    (folder / "tags.cpp").write_text(HARNESS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), str(folder / "tags.cpp"), "-o", str(folder / "tags.so")], check=True)
    function = C.CDLL(str(folder / "tags.so")).failures
    function.argtypes, function.restype = [C.c_uint64, C.c_uint64, C.c_int], C.c_int
    return function


@pytest.mark.parametrize("garbage", [0, 1, 2 ** 64 - 1, 0x9D3F6AC1E57B2481 * 5 % 2 ** 64])
def test_no_order_leaves_a_tag_behind(failures, garbage):
    assert failures(0x9D3F6AC1E57B2481, garbage, 0) == 0


def test_a_store_and_a_store_would(failures):
    """A block that comes after the wait was given up sets a tag that the next replay takes for its own."""
    assert failures(0x9D3F6AC1E57B2481, 0, 1) > 0


def test_no_complement_is_a_tag():
    """Tags are odd multiples of one odd number, modulo 2^64; their complements are even ones, and so none of them."""
    inverse = pow(0x9D3F6AC1E57B2481, -1, 2 ** 64)
    for call in (0, 1, 2, 12345, 2 ** 40, 2 ** 63 - 1):
        tag = 0x9D3F6AC1E57B2481 * (2 * call + 1) % 2 ** 64
        assert (2 ** 64 - 1 - tag) * inverse % 2 ** 64 % 2 == 0
