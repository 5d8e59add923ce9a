// Which log decay a pass of linear attention reads for which row.
#pragma once

#include <cstdint>

namespace hipcx {

// The row of the log decays that is read for row r of a pass over rows [first, end) of a sequence of `length`, end > first: forwards the row's own, backwards that of the row which follows.  It is a
// row of the sequence always: behind the pass's last row that row's again, and of the sequence's last row, which none follows, its own (AttendNoDecay, SumDecays: neither counts).
constexpr int64_t AttendDecayRow(int64_t first, int64_t end, int64_t length, bool back, int64_t r) {
    const int64_t row = r < end - first ? r : end - first - 1;
    if (!back) return first + row;
    return end - row < length ? end - row : length - 1;
}

// Rows at a pass's start that no decay takes the state to: backwards, the sequence's last.
constexpr int64_t AttendNoDecay(int64_t end, int64_t length, bool back) { return back && end == length ? 1 : 0; }

}  // namespace hipcx
