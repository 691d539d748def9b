// Blocks of products grouped by expert: their sides, and the rule that picks them against calls that were timed with each.  Prints what does not hold.
#include "launch_rules.hpp"

#include <algorithm>
#include <cstdio>

using namespace hb;
static int bad = 0;
#define CHECK(ok, ...) do { if (!(ok)) { std::printf(__VA_ARGS__); ++bad; } } while (0)

struct Call { int positions, tiles; double us[3]; }; // one expert, 128 copies at level 5; blocks of one, two and three positions
static const Call calls[] = {
    {1, 12, {740.9, 718.6, 798.5}}, {2, 12, {1450, 1267.5, 1245.4}}, {3, 12, {2174.9, 2026.2, 1844}}, {4, 12, {2887.1, 2494.5, 2640.2}}, {5, 12, {3614.6, 3276.5, 3123.6}},
    {6, 12, {4322.1, 3765.5, 3644.6}}, {7, 6, {2658.7, 2398.5, 2601.7}}, {8, 6, {3062.8, 2674.1, 2885.1}}, {3, 8, {1379.7, 1430.8, 1271}}, {4, 4, {1164.4, 938.2, 999.7}},
    {3, 4, {881.7, 783.5, 689.7}}, {2, 4, {595.3, 484.9, 481.8}}, {2, 1, {354.3, 304.8, 304.4}}, {3, 1, {526.1, 490.8, 418.3}}, {4, 2, {847.2, 728.1, 737}},
    {1, 1, {181.5, 201.3, 202.3}}, {1, 2, {221.1, 241.8, 242}}, {1, 3, {265.4, 279.5, 279.2}}, {1, 4, {311.8, 305.6, 303.7}}, {1, 6, {400.3, 392.8, 511.2}},
    {1, 8, {481.6, 559.1, 547}}, {2, 2, {423, 370.6, 364.4}}, {2, 3, {519.7, 432.5, 436.5}}, {2, 6, {779.7, 693.1, 788.3}}, {2, 8, {926.8, 896.8, 869.6}},
    {3, 6, {1167.5, 1090.9, 1080.2}}, {5, 6, {1929.3, 1751.7, 1851.8}}, {6, 6, {2308.7, 2015.4, 2114.8}}, {9, 6, {3400.4, 3069, 3135.1}}, {5, 4, {1461.8, 1239.2, 1183.4}},
    {7, 4, {2011.1, 1689.4, 1654.4}}, {4, 5, {1541.8, 1369.6, 1571.2}}, {3, 10, {2176.1, 2011.9, 1839.9}}, {2, 7, {909.1, 873.9, 874.3}}, {4, 9, {2888.2, 2521.5, 2276.9}},
    {5, 2, {1041.2, 942.3, 836.1}}, {5, 1, {873.1, 775, 708}},
};

int main() {
    for (int M = 1; M <= 3; ++M)
        for (int tiles = 1; tiles <= 2000; ++tiles) {
            const int T = expert_tiles(M, tiles);
            CHECK(T >= 1 && T <= (M == 1 ? 8 : M == 2 ? 6 : 4) && T != 5 && T != 7, "%d positions, %d tiles: a block of %d tiles has no kernel\n", M, tiles, T);
            CHECK(tiles > T || T - tiles <= 1, "%d positions, %d tiles: a block of %d\n", M, tiles, T);
        }
    for (const Call &c : calls) {
        const double got = c.us[expert_positions(1, c.tiles, [&](int) { return c.positions; }) - 1], best = *std::min_element(c.us, c.us + 3);
        CHECK(got <= 1.04 * best, "%d positions of %d tiles: %g us, %g with the best\n", c.positions, c.tiles, got, best);
    }
    // experts without positions change nothing, and a list of experts is the sum of them
    const int sizes[] = {0, 4, 0, 1, 0};
    CHECK(expert_positions(5, 12, [&](int e) { return sizes[e]; }) >= 1, "no positions\n");
    for (int p = 1; p < 40; ++p)
        for (int tiles = 1; tiles < 40; ++tiles) {
            const int one = expert_positions(1, tiles, [&](int) { return p; }), many = expert_positions(7, tiles, [&](int e) { return e % 2 ? p : 0; });
            CHECK(one == many, "%d positions of %d tiles: %d alone, %d thrice\n", p, tiles, one, many);
        }
    for (int p = 1; p < 300; ++p)
        for (int tiles = 1; tiles < 40; ++tiles)
            for (long each : {8L, 16L, 64L, 512L}) {
                const int T = expert_tiles_few(p, tiles, each);
                CHECK(T >= 1 && T <= 4 && T <= tiles, "%d positions of %d tiles, %ld CTAs each: %d\n", p, tiles, each, T);
                CHECK(T == 1 || p * ((tiles + T - 1L) / T) * each >= 148 * 3, "%d positions of %d tiles, %ld CTAs each: %d do not fill the GPU\n", p, tiles, each, T);
            }
    return bad != 0;
}
