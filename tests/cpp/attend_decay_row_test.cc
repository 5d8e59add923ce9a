// Rows of log decays that the passes of linear attention read: all of them in the sequence, and those that count the right ones.
#include <cstdio>
#include <vector>

#include "attend_decay_row.h"

int main() {
    using namespace hipcx;
    long checks = 0;
    for (const int64_t length : {int64_t{1}, int64_t{2}, int64_t{63}, int64_t{64}, int64_t{65}, int64_t{128}, int64_t{129}, int64_t{385}, int64_t{1} << 33}) {
        for (const int64_t count : {int64_t{1}, int64_t{2}, int64_t{64}, int64_t{65}, int64_t{192}, int64_t{193}}) {
            if (count > length) continue;
            for (const int64_t first : {int64_t{0}, (length - count) / 2, length - count}) {
                const int64_t end = first + count;
                for (const bool back : {false, true}) {
                    const int64_t none = AttendNoDecay(end, length, back);
                    if (none != (back && end == length ? 1 : 0)) return std::printf("%lld rows of %lld: %lld without a decay\n", (long long)count, (long long)length, (long long)none), 1;
                    for (int64_t r = 0; r < count + 192; ++r, ++checks) {  // a tile and two tiles ahead
                        const int64_t row = AttendDecayRow(first, end, length, back, r), want = back ? end - r : first + r;
                        if (row < 0 || row >= length || (r >= none && r < count && row != want)) {
                            return std::printf("row %lld of [%lld, %lld) of %lld, %s: reads %lld\n", (long long)r, (long long)first, (long long)end, (long long)length, back ? "back" : "on", (long long)row), 1;
                        }
                    }
                }
            }
        }
    }
    std::printf("all checks passed: %ld\n", checks);
    return 0;
}
