// Which product of a step is scaled and added when, beside the matrix unit (blocks8.hip).  Plain C++, checked at compile time.
//
// A wave starts PRODUCTS block products a step, one a slot, and adds each one BEHIND slots later: its result has left the matrix unit by
// then.  The first slots add nothing, the last BEHIND products are added behind the last slot.  A product keeps its registers' place until
// it has been added, so there are BEHIND + 1 places.
#pragma once

namespace dl {

template <int PRODUCTS>
struct ProductSchedule {
  static constexpr int BEHIND = 3, PLACES = BEHIND + 1, LEFT = PRODUCTS - BEHIND;      // LEFT: the first one behind the last slot
  static constexpr int NONE = -1;
  static constexpr int added_in(int slot) { return slot < BEHIND ? NONE : slot - BEHIND; }
  static constexpr int place(int product) { return product % PLACES; }
  // Every product is added once, in order, from a place that no later one has taken.
  static constexpr bool sound() {
    int holds[PLACES] = {}, next = 0;
    for (int slot = 0; slot < PRODUCTS; ++slot) {
      holds[place(slot)] = slot;
      const int q = added_in(slot);
      if (q != NONE && (q != next++ || holds[place(q)] != q)) return false;
    }
    if (LEFT != next || LEFT < 0) return false;
    for (int q = LEFT; q < PRODUCTS; ++q)
      if (holds[place(q)] != q) return false;
    return true;
  }
};

}  // namespace dl
