"""The tags of a group-norm workspace's launches, and how its words and its list are read, from the header that the kernels use,
compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = r"""
#include <cstdio>
#include "gn_epoch.h"
int main() {
  unsigned epoch = 0;
  for (int i = 0; i < 5; ++i) { unsigned t = gn_epoch_tag(epoch); std::printf("%u %d\n", t, gn_last_tag(t)); epoch = gn_epoch_after(t); }
  epoch = 0xFFFFFFF0u;
  for (int i = 0; i < 40; ++i) { unsigned t = gn_epoch_tag(epoch); std::printf("%u %d\n", t, gn_last_tag(t)); epoch = gn_epoch_after(t); }
}
"""


def launches(program, tmp_path):
    src, exe = tmp_path / "tags.cpp", tmp_path / "tags"
    src.write_text(program)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "dnanet_amd", "csrc"), str(src), "-o", str(exe)], check=True, timeout=120)
    rows = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.split()
    return [(int(t), clear == "1") for t, clear in zip(rows[::2], rows[1::2])]


def mistaken(rows):
    """Launches that would take a word of an earlier one, or one that was never written, for their own.  Every launch writes a word
    of its own and leaves it; clearing zeroes all of them behind the launch."""
    words, wrong = {0}, []
    for k, (tag, clear) in enumerate(rows):
        if tag in words:
            wrong.append(k)
        words = {0} if clear else words | {tag}
    return wrong


def test_no_tag_comes_twice_while_its_words_are_there(tmp_path):
    rows = launches(PROGRAM, tmp_path)
    first, around = rows[:5], rows[5:]
    assert [t for t, _ in first] == [1, 2, 3, 4, 5]
    assert [t for t, _ in around[13:18]] == [(1 << 32) - 2, (1 << 32) - 1, 1, 2, 3]
    assert not mistaken(rows), "words of the first launches are still there when the last tag has come"
    assert mistaken([(e % ((1 << 32) - 1) + 1, False) for e in ((1 << 32) - 2, (1 << 32) - 1, 0, 1)]) == [2], \
        "a tag that epochs 2^32 - 1 and 0 share is found"


WORDS = r"""
#include <cstdio>
#include "gn_epoch.h"
using word = unsigned long long;
int main() {
  // a word that arrives after `late` looks; before that the word of an earlier launch is there
  const int late[] = {0, 1, 7, 8, 1000};
  for (int n : late) {
    int looks = 0;
    unsigned value = 0;
    const bool there = gn_take(5, 8, [&] { return looks++ < n ? (word)4 << 32 | 111 : (word)5 << 32 | 222; }, &value);
    std::printf("%d %u %d\n", there, value, looks);
  }
  // places 3, (another launch's) 9, (outside the grid) 70, 6; then nothing
  const word list[] = {(word)5 << 32 | 3, (word)4 << 32 | 9, (word)5 << 32 | 70, (word)5 << 32 | 6};
  unsigned at = 0;
  for (int i = 0; i < 3; ++i)
    std::printf("%u\n", gn_take_listed(5, 8, 4, &at, 64, [&](unsigned k) { return list[k]; }, [](unsigned place) { return place < 64; }));
  std::printf("%u\n", at);
}
"""


def test_words_of_other_launches_are_not_taken(tmp_path):
    src, exe = tmp_path / "words.cpp", tmp_path / "words"
    src.write_text(WORDS)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(ROOT, "dnanet_amd", "csrc"), str(src), "-o", str(exe)], check=True, timeout=120)
    got = [tuple(map(int, line.split())) for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=60).stdout.splitlines()]
    assert got[:3] == [(1, 222, 1), (1, 222, 2), (1, 222, 8)]
    assert [(there, looks) for there, _, looks in got[3:5]] == [(0, 8), (0, 8)], "bounded, and told apart"
    assert got[5:] == [(3,), (6,), (64,), (4,)]
