// Epochs of a workspace's launches and the tags of the words that they publish there (plain C++: the host can run it).
//
// A launch finds the epoch of its workspace (0 at first: the workspace is zero-filled) and publishes its words with the tag
// epoch + 1, so that no word of an earlier launch, and no word that was never written, has its tag.  The launch's last block
// leaves the next epoch.  After the last tag, 2^32 - 1, it first zeroes every word and starts again from epoch 0: no tag comes a
// second time while a word of its first time is there.
#pragma once

constexpr unsigned gn_epoch_tag(unsigned epoch) { return epoch + 1; }
constexpr bool gn_last_tag(unsigned tag) { return tag == 0xFFFFFFFFu; }
constexpr unsigned gn_epoch_after(unsigned tag) { return gn_last_tag(tag) ? 0u : tag; }

// The 32-bit value of a published word {tag, value}: looks at it until its tag is `tag`, `looks` times at most; false: it is not there.
template <typename Load> constexpr bool gn_take(unsigned tag, int looks, Load load, unsigned* value) {
  for (; looks > 0; --looks) {
    const unsigned long long word = load();
    *value = (unsigned)word;
    if ((unsigned)(word >> 32) == tag) return true;
  }
  return false;
}
// The next of the listed places from *at on that a block of this launch has put there; `none` if there is none.  Words without the
// launch's tag, and places that valid(place) refuses, come from a workspace that was not zeroed: they are passed over.
template <typename Load, typename Valid>
constexpr unsigned gn_take_listed(unsigned tag, int looks, unsigned listed, unsigned* at, unsigned none, Load load, Valid valid) {
  while (*at < listed) {
    const unsigned i = (*at)++;
    unsigned place = 0;
    if (gn_take(tag, looks, [&] { return load(i); }, &place) && valid(place)) return place;
  }
  return none;
}
