// A launch's rules asked for no members: a list that ended with the launch before.
#include "launch_rules.hpp"

#include <cstdio>
#include <initializer_list>

int main() {
    int bad = 0;
    for (long each : {8L, 56L, 768L, 1664L})
        for (long columns : {1L, 2L, 128L, 65535L}) {
            const int chunk = hb::norm_chunk(0, each, columns);
            if (chunk != 1) { ++bad; std::printf("%ld %ld: %d\n", each, columns, chunk); }
        }
    for (long each : {1L, 148L, 1L << 30})
        for (int most : {0, 2, 3})
            if (hb::norm_log_splits(0, each, most) != 0) { ++bad; std::printf("parts: %ld %d\n", each, most); }
    return bad != 0;
}
