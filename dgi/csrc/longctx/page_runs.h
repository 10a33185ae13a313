// dgi/csrc/longctx/page_runs.h — which rows of a step write a page's bounds.
//
// Rows of a page lie side by side; rows without a slot may lie between them, and slots may be left out.  The first of them takes them
// all, so that a page has one writer.  Plain C++: `ballot(f)` is f of each of 64 lanes, a bit a lane; on the device they are a wave's.
#pragma once

namespace dgi {

constexpr bool has_slot(int slot, long long n_slots) { return slot >= 0 && slot < n_slots; }
// of the page whose first slot is `page0`
constexpr bool in_page(int slot, int page0, int block_size) { return slot >= page0 && slot - page0 < block_size; }

// Whether the row before t that has a slot is of another page than row t.
template <class Ballot>
constexpr bool begins_page(Ballot ballot, const int* slots, long long n_slots, int block_size, int t, int page0) {
  if (t > 0 && has_slot(slots[t - 1], n_slots)) return !in_page(slots[t - 1], page0, block_size);      // mostly; one load for all lanes
  for (int from = t - 2; from >= 0; from -= 64) {
    auto slot = [=](int lane) { return from >= lane ? slots[from - lane] : -1; };
    const unsigned long long there = ballot([=](int lane) { return has_slot(slot(lane), n_slots); });
    const unsigned long long here = ballot([=](int lane) { return in_page(slot(lane), page0, block_size); });
    if (there) return !(here & (there & -there));
  }
  return true;
}

// Rows from t, the first of its page, to the last of it; those among them that have a slot are the page's.  `plain`: all have, one after another.
struct PageRows {
  int rows;
  bool plain;
};
template <class Ballot>
constexpr PageRows page_rows(Ballot ballot, const int* slots, long long n_slots, int block_size, int T, int t, int page0) {
  int rows = 1, in_turn = 0;
  for (int from = t; from < T; from += 64) {
    auto slot = [=](int lane) { return T - from > lane ? slots[from + lane] : -1; };
    const unsigned long long there = ballot([=](int lane) { return has_slot(slot(lane), n_slots); });
    const unsigned long long here = ballot([=](int lane) { return in_page(slot(lane), page0, block_size); });
    const unsigned long long next = ballot([=](int lane) { return (unsigned)slot(lane) - (from - t + lane) == (unsigned)slots[t]; });
    const unsigned long long others = there & ~here, mine = others ? here & ((others & -others) - 1) : here;
    if (mine) rows = from - t + 64 - __builtin_clzll(mine);
    in_turn += __builtin_popcountll(mine & next);
    if (others) break;
  }
  return {rows, in_turn == rows};
}

}  // namespace dgi
