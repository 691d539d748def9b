// Products grouped by expert in a separately compiled program: Evaluator::matmulGrouped gives position by position the residues of matmulGroups, and refuses orders and
// weights of another number.  Returns 0 when it does.
#include "HEMMer.hpp"

#include <cstdio>
#include <vector>

int main() {
    const int d = 16, inputs = 2, tiles = 2; // N = 2^10: two tiles fill the 512 slots
    hb_params prm = {10, 8, 3, 3, 60, 42, 60, 32, 3.2, {1, 2, 3, 4}};
    HELLM::HEMMer *hemmer = HELLM::HEMMer::genHEMMer(/*device*/ 0, prm);
    const HELLM::Evaluator &ev = hemmer->eval();
    auto residues = [&](const HELLM::Ciphertext &t) {
        int level = 0, polys = 0, batch = 0, sp = 0;
        hb_ct_meta(t.raw(), &level, &polys, &batch, &sp);
        std::vector<uint64_t> r((size_t)batch * polys * (level + 1) * 1024);
        HELLM::check(hemmer->context(), hb_ct_export(hemmer->context(), t.raw(), r.data()));
        return r;
    };
    std::vector<double> x(d * d, 0.25), y(d * d, -0.5);
    std::vector<HELLM::Ciphertext> each;
    for (int i = 0; i < inputs; ++i) each.push_back(hemmer->encrypt2((i ? y : x).data(), (i ? x : y).data(), d, d, /*nonce*/ i + 1).get());
    const HELLM::Ciphertext pre = hemmer->matMulPre(HELLM::CtxtTensor(HELLM::TileTensorShape(d, d, 2 * d), ev.concat(each)), 2);
    int level = 0, batch = 0;
    hb_ct_meta(pre.raw(), &level, nullptr, &batch, nullptr);
    const std::vector<int32_t> sizes = {1, 0, 2}, order = {1, 0, 1};
    std::vector<HELLM::Plaintext> weights;
    std::vector<const hb_pt *> pts;
    for (int k = 0; k < 3 * tiles; ++k) {
        HELLM::Message m((size_t)512);
        for (int s = 0; s < 512; ++s) m.re[(size_t)s] = 0.001 * ((s * (k + 3)) % 101 - 50);
        weights.push_back(ev.encode(m, level));
    }
    for (int e = 0; e < 3; ++e)
        for (int t = 0; t < tiles; ++t) pts.push_back(sizes[(size_t)e] ? weights[(size_t)(e * tiles + t)].raw() : nullptr); // those of an expert without positions are not looked at
    int bad = 0;
    const std::vector<int> expert = {0, 2, 2};
    auto same = [&](const HELLM::Ciphertext &got, int p, int t, int input, int e) {
        return residues(ev.view(got, p * tiles + t, 1)) == residues(ev.matmulGroups(pre, inputs, input, {pts[(size_t)(e * tiles + t)]}, 2 * d));
    };
    const HELLM::Ciphertext got = ev.matmulGrouped(pre, inputs, order, sizes, pts, 1, tiles, 2 * d);
    if (got.getBatch() != 3 * tiles) ++bad;
    for (int p = 0; p < 3; ++p)
        for (int t = 0; t < tiles; ++t)
            if (!same(got, p, t, order[(size_t)p], expert[(size_t)p])) ++bad;
    const std::vector<int32_t> one_each = {1, 0, 1}; // without an order position p has input p
    const HELLM::Ciphertext plain = ev.matmulGrouped(pre, inputs, {}, one_each, pts, 1, tiles, 2 * d);
    for (int p = 0; p < 2; ++p)
        if (!same(plain, p, 1, p, 2 * p)) ++bad;
    const auto refused = [&](const std::vector<int32_t> &o, const std::vector<int32_t> &s, const std::vector<const hb_pt *> &w, int b, int t) {
        try { ev.matmulGrouped(pre, inputs, o, s, w, b, t, 2 * d); } catch (const std::invalid_argument &) { return true; }
        return false;
    };
    const std::vector<const hb_pt *> fewer(pts.begin(), pts.end() - 1);
    if (!refused({1, 0}, sizes, pts, 1, tiles) || !refused({1, 0, 1, 1}, sizes, pts, 1, tiles) || !refused(order, sizes, fewer, 1, tiles) || !refused(order, sizes, pts, 2, tiles)) ++bad;
    if (!refused(order, sizes, pts, 1, tiles + 1) || !refused(order, sizes, {}, 1, 0) || !refused({}, sizes, pts, 1, tiles) || !refused({2, 0, 1}, sizes, pts, 1, tiles)) ++bad;
    if (!refused({}, {}, {}, 1, tiles) || !refused({1}, {2, -1, 0}, pts, 1, tiles)) ++bad;
    delete hemmer;
    std::printf("%d results differ\n", bad);
    return bad ? 1 : 0;
}
