// dgi/csrc/longctx/page_runs.h — which rows of a step write a page's bounds.
//
// Rows of a page lie side by side; rows without a slot may lie between them, and slots may be left out.  The first of them takes them
// all, so that a page has one writer.  Plain C++: `ballot(f)` is f of each of 64 lanes, a bit a lane; on the device they are a wave's.
#pragma once

namespace dgi {

constexpr bool has_slot(int slot, long long n_slots) { return slot >= 0 && slot < n_slots; }
// of the page whose first slot is `page0`
constexpr bool in_page(int slot, int page0, int block_size) { return slot >= page0 && slot - page0 < block_size; }

// Times 64 rows that are looked at together: as many loads are under way where many rows have no slot (a row beside 511 of them: 4.8 us, one load
// at a time 6.7).
constexpr int kLook = 8;

// Whether the row before t that has a slot is of another page than row t.
template <class Ballot>
constexpr bool begins_page(Ballot ballot, const int* slots, long long n_slots, int block_size, int t, int page0) {
  if (t > 0 && has_slot(slots[t - 1], n_slots)) return !in_page(slots[t - 1], page0, block_size);      // mostly; one load for all lanes
  for (int from = t - 2; from >= 0; from -= 64 * kLook) {
    unsigned long long there[kLook] = {}, here[kLook] = {};
#pragma unroll
    for (int j = 0; j < kLook; ++j) {
      const int at = from - 64 * j;
      auto slot = [=](int lane) {
        const int s = slots[at >= lane ? at - lane : 0];      // all lanes read, without a branch
        return at >= lane ? s : -1;
      };
      there[j] = ballot([=](int lane) { return has_slot(slot(lane), n_slots); });
      here[j] = ballot([=](int lane) { return in_page(slot(lane), page0, block_size); });
    }
#pragma unroll
    for (int j = 0; j < kLook; ++j)
      if (there[j]) return !(here[j] & (there[j] & -there[j]));
  }
  return true;
}

// Rows from t, the first of its page, to the last of it; those among them that have a slot are the page's.  `plain`: all have, one after another.
struct PageRows {
  int rows;
  bool plain;
};

// The same for N times 64 rows: `rows` from t on, and how many of them have the slot that follows from row t's.  Whether a row of another page ends it.
template <int N, class Ballot>
constexpr bool look_ahead(Ballot ballot, const int* slots, long long n_slots, int block_size, int T, int t, int page0, int from, int& rows, int& in_turn) {
  unsigned long long there[N] = {}, here[N] = {}, next[N] = {};
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int at = from + 64 * j;
    auto slot = [=](int lane) {
      const int s = slots[T - at > lane ? at + lane : T - 1];
      return T - at > lane ? s : -1;
    };
    there[j] = ballot([=](int lane) { return has_slot(slot(lane), n_slots); });
    here[j] = ballot([=](int lane) { return in_page(slot(lane), page0, block_size); });
    next[j] = ballot([=](int lane) { return (unsigned)slot(lane) - (at - t + lane) == (unsigned)slots[t]; });
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const unsigned long long others = there[j] & ~here[j], mine = others ? here[j] & ((others & -others) - 1) : here[j];
    if (mine) rows = from + 64 * j - t + 64 - __builtin_clzll(mine);
    in_turn += __builtin_popcountll(mine & next[j]);
    if (others) return true;
  }
  return false;
}

template <class Ballot>
constexpr PageRows page_rows(Ballot ballot, const int* slots, long long n_slots, int block_size, int T, int t, int page0) {
  int rows = 1, in_turn = 0;
  if (!look_ahead<1>(ballot, slots, n_slots, block_size, T, t, page0, t, rows, in_turn))
    for (int from = t + 64; from < T; from += 64 * kLook)
      if (look_ahead<kLook>(ballot, slots, n_slots, block_size, T, t, page0, from, rows, in_turn)) break;
  return {rows, in_turn == rows};
}

}  // namespace dgi
