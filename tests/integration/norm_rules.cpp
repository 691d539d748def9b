// The rules of dispatch of the normalisation: every member is taken once, grids stay within their limits, and where there are CTAs enough nothing is split.
#include "launch_rules.hpp"

#include <cstdio>
#include <initializer_list>

using namespace hb;
static int bad = 0;
static void need(bool ok, const char *what, long a, long b, long c) { if (!ok) { ++bad; std::printf("%s: %ld %ld %ld\n", what, a, b, c); } }

int main() {
    for (long each : {2L, 8L, 56L, 128L, 384L, 768L, 1664L})
        for (long columns : {1L, 2L, 3L, 16L, 128L, 1000L, 65535L})
            for (int members : {1, 2, 3, 7, 8, 9, 16, 255, 256, 1000, 65536, 300000, 2000000}) {
                const int chunk = norm_chunk(members, each, columns);
                const long chunks = (members + (long)chunk - 1) / chunk;
                need(chunk >= 1 && chunk <= members, "a chunk is one member to all", members, each, columns);
                need(chunk * chunks >= members && chunk * (chunks - 1) < members, "chunks hold every member once", members, each, columns);
                need(columns * chunks <= 65535 || chunk == members, "a grid that reaches them", members, each, columns);
                if (chunk > 1 && columns * ((members + chunk - 2L) / (chunk - 1)) <= 65535) need(each * columns * chunks >= 148 * 8, "longer chunks only where CTAs are left", members, each, columns);
                for (int most : {2, 3}) {
                    const int log = norm_log_splits(members, each * columns, most);
                    need(log >= 0 && log <= most && (log == 0 || members >= 4 << (log - 1)), "parts of two members at least", members, each, columns);
                    need(log == 0 || (each * columns << (log - 1)) < 148 * 4, "parts only where CTAs are missing", members, each, columns);
                }
            }
    for (int tiles = 1; tiles <= 300; ++tiles) {
        const int some = grad_tiles(tiles), launches = (tiles + some - 1) / some;
        need(some >= 1 && some <= 8 && launches == (tiles + 7) / 8, "as few launches as there can be", tiles, some, launches);
    }
    for (int tiles = 1; tiles <= 40; ++tiles)
        for (int batch : {1, 2, 8, 33, 1 << 30}) // a product beyond 32 bits
            for (bool same : {false, true}) {
                need(grad_together(tiles, batch, same, 8) == (tiles <= 8 && tiles * (long)batch <= 8), "few CTAs: one kernel only for little work", tiles, batch, same);
                need(!grad_together(tiles, batch, same, 1 << 20) == (tiles > 8 && !same), "many CTAs: one kernel as long as it takes one launch, or reads nothing twice", tiles, batch, same);
            }
    return bad != 0;
}
