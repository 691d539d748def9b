// Masks of the tile transforms: shapes whose blocks reach past the slots are refused before anything is written there (built with the address sanitizer, which ends the
// program at the first write past a message), those that tile the slots are painted.  Nothing of the device library is called.  Prints what does not hold.
#include "schedules.cpp"

#include <cstdio>

using namespace HELLM;
using namespace HELLM::sched;

int main() {
    const Evaluator ev(nullptr);
    MaskCache cache;
    Env e{ev, 2048, cache};
    int bad = 0;
    struct Case { i64 rows, cols, width; bool fits; };
    const Case cases[] = {
        {32, 32, 64, true}, {32, 32, 32, true}, {8, 32, 32, true}, {32, 8, 64, true}, {16, 16, 32, true}, {1, 1, 1, true}, {64, 32, 32, true},
        {20, 32, 32, false}, {32, 20, 32, false}, {32, 20, 64, false}, {20, 20, 64, false}, {128, 32, 32, false}, {33, 8, 64, false}, {20, 20, 40, false},
    };
    for (const Case &c : cases)
        for (bool vertical : {false, true}) {
            const TileTensorShape s(c.rows, c.cols, c.width);
            const DiagFamily f = family(s, vertical, false);
            bool refused = false;
            for (i64 idx = -f.main + 1; idx < f.main; ++idx) {
                if (f.bs == 0 || (idx >= f.sub) || (idx < 0 && idx >= f.sub - f.main)) continue;
                try {
                    const Message m = diag_family_mask(e, s, f, idx);
                    if (m.size() != 2048) { std::printf("%ld x %ld in %ld: a mask of %zu slots\n", (long)c.rows, (long)c.cols, (long)c.width, m.size()); ++bad; }
                } catch (const std::invalid_argument &) { refused = true; }
            }
            if (refused == c.fits) { std::printf("%ld x %ld in %ld, %s: %s\n", (long)c.rows, (long)c.cols, (long)c.width, vertical ? "rows" : "columns", refused ? "refused" : "not refused"); ++bad; }
        }
    return bad != 0;
}
