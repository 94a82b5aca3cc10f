// Index arithmetic of skm_logprob.hip that host code can check as well.
#pragma once
#include <cstdint>

// Where label y lies in the tile whose `rem` classes start at class `base` of a row (base >= 0): 0 .. rem - 1, or -1 where it
// lies in another tile, is none (-1) or no class at all.  The row's last tile ends with the row, so what this gives is inside it
// whatever the label; labels on the device have been looked at by nobody before.
constexpr int lp_entry_of(int64_t y, int64_t base, int rem) { return y >= base && y - base < rem ? (int)(y - base) : -1; }
