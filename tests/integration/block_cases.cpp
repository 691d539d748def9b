// The blocks that the rules of dispatch make of cases read from the input, one a line: "experts <CTAs of a block> <tiles> <sizes ...>" gives "M T",
// "pairs <ring degree> <limbs> <heads> <tiles of one side> <of the other>" the number of the block and its ranges, "kernels" all M and T that there are kernels for.
#include "launch_rules.hpp"

#include <algorithm>
#include <iostream>
#include <sstream>
#include <string>
#include <vector>

using namespace hb;

int main() {
    for (std::string line; std::getline(std::cin, line);) {
        std::istringstream in(line);
        std::string what;
        in >> what;
        if (what == "kernels") {
            for (int M = 1; M <= 16; ++M)
                for (int T = 1; T <= 16; ++T)
                    if (expert_kernel(M, T)) std::cout << M << ' ' << T << ' ';
        } else if (what == "experts") {
            long each = 0;
            int tiles = 0;
            in >> each >> tiles;
            std::vector<int> sizes;
            for (int s; in >> s;) sizes.push_back(s);
            const ExpertBlocks b = expert_blocks((int)sizes.size(), tiles, each, [&](int e) { return sizes[(size_t)e]; });
            std::cout << b.M << ' ' << b.T;
        } else {
            int N = 0, limbs = 0, heads = 0, a = 0, b = 0;
            in >> N >> limbs >> heads >> a >> b;
            const int nr = std::max(a, b), nc = std::min(a, b), v = pair_block(nr, nc);
            std::cout << v << ' ' << pair_ranges(kPairBlocks[v], N, nr, nc, heads, limbs);
        }
        std::cout << '\n';
    }
}
