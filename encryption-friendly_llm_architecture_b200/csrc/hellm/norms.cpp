// Layer norm, its gradients, and the clipping of gradients by their global norm, on ciphertexts.  The sums, products and gradients are hb_norm_*, hb_square_sum_many and
// hb_scale_many; what stands between them (relinearisation, sums over slots by rotations, polynomials of the inverse root) is put together here.
#include "HEMMer.hpp"
#include "schedules.hpp"

#include <cmath>
#include <cstring>
#include <functional>

namespace HELLM {

namespace {
constexpr double kPi = 3.14159265358979323846264338327950288;

// a column tile of `columns` values in every row, zeros behind them
Plaintext columns_plaintext(const HEMMer &h, const TileTensorShape &s, const double *v, i64 columns, int level) {
    const i64 w = s.getBlockWidth();
    Message m((size_t)h.slots());
    for (i64 r = 0; r < s.getNumRows(); ++r)
        for (i64 c = 0; c < columns; ++c) m.re[(size_t)(r * w + c)] = v ? v[c] : 1.0;
    return h.eval().encode(m, level);
}
// Masks that depend on a number: the number's bits are part of their key.  They stay, since recorded graphs hold their addresses, and so there are kNormMasks of a kind at most:
// a program with more (another range of variances at every step) makes the others at every call, on the device, so that it can be recorded too.
constexpr size_t kNormMasks = 64;
Plaintext norm_mask(HEMMer &h, int kind, const TileTensorShape &s, double value, int level) {
    i64 bits;
    std::memcpy(&bits, &value, 8);
    const MaskCache::Key k{kind, s, bits, level};
    if (const Plaintext *p = h.masks().find(k)) return *p;
    const bool columns = kind == sched::kNormColumns; // ones in as many columns; otherwise the value in the first column.  Rows fill the slots (norm_shape)
    const int step = (int)s.getBlockWidth();
    if (h.masks().count(kind) >= kNormMasks) return h.eval().encodeMask(columns ? 1.0 : value, step, columns ? (int)value : 1, level);
    if (columns) return h.masks().put(k, columns_plaintext(h, s, nullptr, (i64)value, level));
    Message m((size_t)h.slots());
    for (i64 r = 0; r < s.getNumRows(); ++r) m.re[(size_t)(r * step)] = value;
    return h.masks().put(k, h.eval().encode(m, level)); // not while a graph records, when the mask would hold nothing until its replay
}
Ciphertext switched(const Evaluator &ev, const Ciphertext &x) { return ev.rescale(ev.relinearize(x)); }
// x at a lower level, or a view of x, which has to outlive it; a temporary is moved
Ciphertext down(const Evaluator &ev, const Ciphertext &x, int level) { return x.getLevel() == level ? ev.view(x, 0, x.getBatch()) : ev.levelDown(x, level); }
Ciphertext down(const Evaluator &ev, Ciphertext &&x, int level) { return x.getLevel() == level ? std::move(x) : ev.levelDown(x, level); }

// the sum of x rotated by 0, step, ... (count - 1) step, count a power of two: four terms at a time with one decomposition and one ModDown
Ciphertext sum_rotations(const Evaluator &ev, Ciphertext x, i64 step, i64 count) {
    while (count > 1) {
        const i64 some = count >= 4 ? 4 : 2;
        std::vector<i64> steps;
        for (i64 k = 0; k < some; ++k) steps.push_back(k * step);
        x = ev.rotateSumHoisted(x, ev.decompose(x), steps);
        step *= some; count /= some;
    }
    return x;
}
// `scale` times the sum over a row (and `other` times the first column of y), in all its columns; one level
Ciphertext row_mean(HEMMer &h, Ciphertext x, const TileTensorShape &s, double scale, const Ciphertext *y = nullptr, double other = 0.0) {
    const Evaluator &ev = h.eval();
    x = sum_rotations(ev, std::move(x), 1, s.getBlockWidth());
    const Plaintext mask = norm_mask(h, sched::kNormFirstCol, s, scale, x.getLevel());
    if (y) {
        const Plaintext second = norm_mask(h, sched::kNormFirstCol, s, other, x.getLevel());
        x = ev.multSumRescaledOnce({&x, y}, {&mask, &second});
    } else x = ev.mult(x, mask);
    return sum_rotations(ev, std::move(x), -1, s.getBlockWidth());
}
// the sum over all slots that are a multiple of `step` apart, in each of them
Ciphertext sum_slots(const HEMMer &h, Ciphertext x, i64 step) {
    return sum_rotations(h.eval(), std::move(x), step, h.slots() / step);
}

struct NormShape { TileTensorShape s; int groups, batch; i64 columns, pad; };
NormShape norm_shape(const HEMMer &h, const CtxtTensor &x, int groups, i64 columns, const char *what) {
    const std::string name = std::string("[") + what + "] ";
    const i64 w = x.getBlockWidth(), rows = x.getHeight();
    if (w < 1 || (w & (w - 1)) || rows < 1 || rows > h.slots() / w || rows * w != h.slots()) throw std::invalid_argument(name + "rows of a power of two that fill the slots");
    if (groups < 1 || x.get().getBatch() % groups) throw std::invalid_argument(name + "the batch does not split into that many column tiles");
    if (columns <= (groups - 1) * w || columns > groups * w) throw std::invalid_argument(name + "columns end in the last tile");
    return {x.getShape(), groups, x.get().getBatch() / groups, columns, groups * w - columns};
}
void need_level(int level, int least, const char *what) {
    if (level < least) throw std::invalid_argument(std::string("[") + what + "] level too low: " + std::to_string(level) + " of " + std::to_string(least));
}
// plaintexts of the column tiles: values (NULL: ones) of the first `columns`, zeros behind them
std::vector<Plaintext> column_plaintexts(HEMMer &h, const NormShape &n, const double *v, int level) {
    const i64 w = n.s.getBlockWidth();
    std::vector<Plaintext> p;
    for (i64 t = 0; t < n.groups; ++t) {
        const i64 here = std::min(w, n.columns - t * w);
        p.push_back(v ? columns_plaintext(h, n.s, v + t * w, here, level) : norm_mask(h, sched::kNormColumns, n.s, (double)here, level));
    }
    return p;
}
std::vector<const Plaintext *> pointers(const std::vector<Plaintext> &p) {
    std::vector<const Plaintext *> r;
    for (const Plaintext &x : p) r.push_back(&x);
    return r;
}

// ---- polynomials in Chebyshev form ----
// Coefficients of the interpolation of f over [lo, hi] at the n + 1 Chebyshev points: f(x) ~ sum_j c[j] T_j(u), u the place of x in [-1, 1].
template <class F> std::vector<double> chebyshev(F &&f, double lo, double hi, int n) {
    std::vector<double> y((size_t)n + 1), c((size_t)n + 1);
    for (int k = 0; k <= n; ++k) y[(size_t)k] = f(0.5 * (hi + lo) + 0.5 * (hi - lo) * std::cos(kPi * (k + 0.5) / (n + 1)));
    for (int j = 0; j <= n; ++j) {
        double s = 0.0;
        for (int k = 0; k <= n; ++k) s += y[(size_t)k] * std::cos(kPi * j * (k + 0.5) / (n + 1));
        c[(size_t)j] = s * (j ? 2.0 : 1.0) / (n + 1);
    }
    return c;
}
int log2_floor(int n) { int l = 0; while (n >> (l + 1)) ++l; return l; }
// levels of the evaluation below
int chebyshev_depth(int n) {
    if (n <= 3) return n;
    const int m = log2_floor(n), q = n - (1 << m);
    return std::max(std::max(m, q ? chebyshev_depth(q) : 0) + 1, chebyshev_depth((1 << m) - 1));
}
// T_m for m = 1, 2, 3 and the powers of two, from T_2a = 2 T_a^2 - 1 and T_3 = 2 T_1 T_2 - T_1; and sums of them: a polynomial of degree n is q T_m + r for the largest power of two m <= n, with
// q_j = 2 c_{m+j} (q_0 = c_m) and r_{m-j} = c_{m-j} - c_{m+j}, since T_m T_j = (T_{m+j} + T_{m-j}) / 2.  Constants are added last.
struct Chebyshev {
    const Evaluator &ev;
    std::vector<Ciphertext> t; // t[m]
    Chebyshev(const Evaluator &e, const Ciphertext &u, int n) : ev(e), t((size_t)std::max(n, 3) + 1) {
        t[1] = ev.view(u, 0, u.getBatch());
        for (int m = 2; m <= n; m <<= 1) {
            const Ciphertext s = ev.square(t[(size_t)m / 2]);
            t[(size_t)m] = ev.addConstant(ev.add(s, s), -1.0);
        }
        if (n >= 3) {
            const Ciphertext s = ev.mult(t[1], t[2]);
            t[3] = ev.sub(ev.add(s, s), t[1]);
        }
    }
    struct Sum { Ciphertext x; double c = 0.0; }; // x + c; no x: c alone
    Ciphertext whole(Sum &&s) const { return s.c == 0.0 ? std::move(s.x) : ev.addConstant(s.x, s.c); }
    Sum eval(std::vector<double> c) const {
        while (c.size() > 1 && c.back() == 0.0) c.pop_back();
        const int n = (int)c.size() - 1;
        Sum r;
        r.c = c[0];
        if (n == 0) return r;
        if (n <= 3) {
            const int level = t[(size_t)n].getLevel();
            std::vector<Ciphertext> x;
            std::vector<const Ciphertext *> px;
            std::vector<double> k;
            for (int j = 1; j <= n; ++j) {
                if (c[(size_t)j] == 0.0) continue;
                x.push_back(down(ev, t[(size_t)j], level));
                k.push_back(c[(size_t)j]);
            }
            for (const Ciphertext &y : x) px.push_back(&y);
            r.x = ev.rescale(ev.combine(px, k, r.c));
            r.c = 0.0;
            return r;
        }
        const int m = 1 << log2_floor(n);
        std::vector<double> q(c.begin() + m, c.end()), rest(c.begin(), c.begin() + m);
        for (int j = 1; j <= n - m; ++j) { rest[(size_t)(m - j)] -= q[(size_t)j]; q[(size_t)j] *= 2.0; }
        Sum high = eval(q), low = eval(rest);
        const Ciphertext &tm = t[(size_t)m];
        r.x = high.x.empty() ? ev.rescale(ev.combine({&tm}, {high.c})) : ev.mult(whole(std::move(high)), tm);
        if (!low.x.empty()) r.x = ev.add(r.x, low.x);
        r.c = low.c;
        return r;
    }
};
Ciphertext evaluate(const Evaluator &ev, const Ciphertext &u, const std::vector<double> &c) {
    const Chebyshev t(ev, u, (int)c.size() - 1);
    auto s = t.eval(c);
    if (s.x.empty()) throw std::invalid_argument("[chebyshev] a constant");
    return t.whole(std::move(s));
}
void need_degree(int degree, const char *what) { if (degree < 1 || degree > 63) throw std::invalid_argument(std::string("[") + what + "] polynomials have a degree from 1 to 63"); }
bool positive(double x) { return x > 0.0 && std::isfinite(x); }
} // namespace

std::vector<double> HEMMer::inverseRootPolynomial(double lo, double hi, int degree) {
    need_degree(degree, "layerNorm");
    if (!positive(lo) || !std::isfinite(hi) || !(hi > lo)) throw std::invalid_argument("[layerNorm] a range of positive variances");
    return chebyshev([](double x) { return 1.0 / std::sqrt(x); }, lo, hi, degree);
}
std::vector<double> HEMMer::clipPolynomial(double max_norm, double bound, int degree) {
    need_degree(degree, "clipGradNorm");
    if (!positive(max_norm) || !positive(bound) || !std::isfinite(bound * bound) || !(bound * bound > 0.0)) throw std::invalid_argument("[clipGradNorm] norms are positive");
    if (!(bound > max_norm)) throw std::invalid_argument("[clipGradNorm] nothing to clip: the bound is not above the norm");
    return chebyshev([&](double s) { return s > max_norm * max_norm ? max_norm / std::sqrt(s) : 1.0; }, 0.0, bound * bound, degree);
}
int HEMMer::polynomialDepth(int degree) { return chebyshev_depth(degree); }

HEMMer::LayerNorm HEMMer::layerNorm(const CtxtTensor &x, int groups, i64 columns, const double *gamma, const double *beta, double eps, double lo, double hi, int degree, const int32_t *tokens) {
    const NormShape n = norm_shape(*this, x, groups, columns, "layerNorm");
    bool padded = false;
    for (int b = 0; tokens && b < n.batch; ++b) {
        if (tokens[b] < 0 || tokens[b] > n.s.getNumRows()) throw std::invalid_argument("[layerNorm] a token tile has 0 to all of its rows");
        padded = padded || tokens[b] < n.s.getNumRows();
    }
    const std::vector<double> c = inverseRootPolynomial(lo, hi, degree);
    if (!(eps >= 0.0) || !std::isfinite(eps)) throw std::invalid_argument("[layerNorm] eps from 0");
    for (const double *v : {gamma, beta})
        for (i64 k = 0; v && k < columns; ++k) if (!std::isfinite(v[k])) throw std::invalid_argument("[layerNorm] a weight is not finite");
    const bool scaled = gamma || n.pad; // columns past the width come out as zeros
    need_level(x.getLevel(), 4 + polynomialDepth(degree) + (scaled ? 1 : 0), "layerNorm");
    const Evaluator &ev = eval_;
    // Masks hold 1 / columns and 2 / ((hi - lo) columns), and where a wide range leaves the second few units of the scale, its rounding is seen in the variance: 13 units in a sum of 32 columns, 100 in one of 256.
    // So mean and squares are those of x / 2^k, which the way down of x to the mean's level takes with it: the second factor grows by 4^k, until it has 2^24 units or as many as the first is left with.
    const double unit = ev.scale(x.getLevel() - 2);
    double shrink = 1.0, mean_scale = 1.0 / (double)columns, scale = 2.0 / ((hi - lo) * (double)columns);
    while (scale * unit < 0x1p24 && scale < mean_scale) { shrink *= 0.5; mean_scale *= 0.5; scale *= 4.0; }
    if (!(scale * unit >= 0x1p16)) throw std::invalid_argument("[layerNorm] the range is too wide for the scale");
    const Ciphertext mean = row_mean(*this, ev.sumGroups(x.get(), groups), n.s, mean_scale);
    auto resized = [&](const Ciphertext &y, double by) { return ev.rescale(ev.combine({&y}, {by})); }; // one level lower
    Ciphertext u;
    {
        Ciphertext squares = ev.normSquares(shrink == 1.0 ? down(ev, x.get(), mean.getLevel()) : resized(x.get(), shrink), &mean, groups, 0), row;
        if (n.pad) { // columns past the width hold zeros, whose differences are the mean: their squares are taken off the sum over the row
            std::vector<Ciphertext> both;
            both.push_back(std::move(squares)); both.push_back(ev.normSquares(mean, nullptr, 1, 0));
            const Ciphertext s = switched(ev, ev.concat(both)), of_mean = ev.group(s, 1, 2);
            row = row_mean(*this, ev.group(s, 0, 2), n.s, scale, &of_mean, -scale * (double)n.pad);
        } else row = row_mean(*this, switched(ev, squares), n.s, scale);
        const double zero = (2.0 * eps - hi - lo) / (hi - lo); // where a variance of nothing has its place
        u = ev.addConstant(row, zero); // the variance's place in [-1, 1]
        if (padded) { // rows of padding, all zeros, are moved to the middle of the range: where the polynomial is large, their noise would come out as values, or spoil all slots
            std::vector<Plaintext> p;
            for (int b = 0; b < n.batch; ++b) {
                Message m((size_t)slots_);
                std::fill(m.re.begin() + tokens[b] * n.s.getBlockWidth(), m.re.end(), -zero);
                p.push_back(eval_.encode(m, u.getLevel()));
            }
            u = ev.normAffine(u, {}, pointers(p));
        }
    }
    Ciphertext rstd = evaluate(eval_, u, c);
    const int level = rstd.getLevel();
    const Ciphertext low_mean = shrink == 1.0 ? down(ev, mean, level) : down(ev, resized(mean, 1.0 / shrink), level);
    Ciphertext xhat = switched(ev, ev.normScale(down(ev, x.get(), level), &low_mean, rstd, groups));
    Ciphertext y;
    if (scaled) {
        const std::vector<Plaintext> g = column_plaintexts(*this, n, gamma, level - 1), b = beta ? column_plaintexts(*this, n, beta, level - 1) : std::vector<Plaintext>();
        y = ev.rescale(ev.normAffine(xhat, pointers(g), pointers(b)));
    } else if (beta) {
        const std::vector<Plaintext> b = column_plaintexts(*this, n, beta, level - 1);
        y = ev.normAffine(xhat, {}, pointers(b));
    } else y = xhat;
    return {CtxtTensor(n.s, std::move(y)), CtxtTensor(n.s, std::move(xhat)), CtxtTensor(n.s, std::move(rstd))};
}

HEMMer::LayerNormGrads HEMMer::layerNormBackward(const CtxtTensor &dy, const CtxtTensor &xhat, const CtxtTensor &rstd, int groups, i64 columns, const double *gamma) {
    const NormShape n = norm_shape(*this, dy, groups, columns, "layerNormBackward");
    const Evaluator &ev = eval_;
    if (xhat.get().getBatch() != dy.get().getBatch() || rstd.get().getBatch() != n.batch) throw std::invalid_argument("[layerNormBackward] batches differ");
    for (i64 k = 0; gamma && k < columns; ++k) if (!std::isfinite(gamma[k])) throw std::invalid_argument("[layerNormBackward] a weight is not finite");
    const bool scaled = gamma || n.pad;
    const int level = std::min(dy.getLevel() - (scaled ? 1 : 0), xhat.getLevel());
    need_level(std::min(level - 3, rstd.getLevel()), n.pad ? 2 : 1, "layerNormBackward");
    Ciphertext g;
    if (scaled) {
        const std::vector<Plaintext> p = column_plaintexts(*this, n, gamma, dy.getLevel());
        g = down(ev, ev.rescale(ev.normAffine(dy.get(), pointers(p), {})), level);
    }
    const Ciphertext low_dy = down(ev, dy.get(), level), low_xhat = down(ev, xhat.get(), level);
    Evaluator::GradSums s = ev.normGradSums(low_dy, scaled ? &g : nullptr, low_xhat, groups);
    LayerNormGrads out;
    const i64 w = n.s.getBlockWidth();
    out.dgamma = CtxtTensor(n.s, sum_slots(*this, switched(ev, s.cols), w));
    out.dbeta = CtxtTensor(n.s, sum_slots(*this, s.colsum, w));
    const Ciphertext dot = row_mean(*this, switched(ev, s.rows), n.s, 1.0 / (double)columns);
    const Ciphertext mean = down(ev, row_mean(*this, std::move(s.rowsum), n.s, 1.0 / (double)columns), dot.getLevel());
    const Ciphertext &gl = scaled ? static_cast<const Ciphertext &>(g) : low_dy;
    const Ciphertext g2 = down(ev, gl, dot.getLevel()), x2 = down(ev, low_xhat, dot.getLevel());
    const Ciphertext inner = switched(ev, ev.normGradInput(g2, mean, x2, dot, groups));
    const int last = std::min(inner.getLevel(), rstd.getLevel());
    const Ciphertext factor = down(ev, rstd.get(), last);
    Ciphertext dx = switched(ev, ev.normScale(down(ev, inner, last), nullptr, factor, groups));
    if (n.pad) {
        const std::vector<Plaintext> ones = column_plaintexts(*this, n, nullptr, dx.getLevel());
        dx = ev.rescale(ev.normAffine(dx, pointers(ones), {}));
    }
    out.dx = CtxtTensor(n.s, std::move(dx));
    return out;
}

namespace {
int lowest_level(const std::vector<const Ciphertext *> &v) {
    int level = v[0]->getLevel();
    for (const Ciphertext *x : v) level = std::min(level, x->getLevel());
    return level;
}
void need_periods(const std::vector<i64> &periods, size_t count, i64 slots, const char *what) {
    if (periods.empty()) return;
    if (periods.size() != count) throw std::invalid_argument(std::string("[") + what + "] a period for every gradient");
    for (const i64 p : periods)
        if (p < 1 || p > slots || (p & (p - 1))) throw std::invalid_argument(std::string("[") + what + "] periods are powers of two up to the slots");
}
}

// A sum of squares with period p is the same after a sum over p slots as any other after one over all of them.  So the sums over the slots go from the longest period to the next, where the squares
// of that period come in, and so on: as many rotations as without periods.
Ciphertext HEMMer::gradNormSquared(const std::vector<const Ciphertext *> &grads, const std::vector<i64> &periods) {
    if (grads.empty()) throw std::invalid_argument("[gradNormSquared] no gradients");
    need_periods(periods, grads.size(), slots_, "gradNormSquared");
    const Evaluator &ev = eval_;
    const int level = lowest_level(grads);
    need_level(level, 1, "gradNormSquared");
    std::map<i64, std::vector<Ciphertext>, std::greater<i64>> by_period;
    for (size_t k = 0; k < grads.size(); ++k) by_period[periods.empty() ? slots_ : periods[k]].push_back(down(ev, *grads[k], level));
    std::vector<Ciphertext> sums;
    for (const auto &g : by_period) sums.push_back(ev.squareSumMany(g.second));
    const int kinds = (int)sums.size();
    Ciphertext squares = kinds == 1 ? switched(ev, sums[0]) : switched(ev, ev.concat(sums));
    Ciphertext sum;
    int k = 0;
    for (auto g = by_period.begin(); g != by_period.end(); ++k) {
        const i64 period = g->first, next = ++g == by_period.end() ? 1 : g->first;
        Ciphertext own = kinds == 1 ? std::move(squares) : ev.group(squares, k, kinds); // a view of several comes back from the sum as a ciphertext of its own, since another period follows
        sum = sum_rotations(ev, k ? ev.add(sum, own) : std::move(own), next, period / next);
    }
    return sum;
}

std::vector<Ciphertext> HEMMer::clipGradNorm(const std::vector<const Ciphertext *> &grads, double max_norm, double bound, int degree, Ciphertext *norm_squared, const std::vector<i64> &periods) {
    std::vector<double> c = clipPolynomial(max_norm, bound, degree);
    if (grads.empty()) throw std::invalid_argument("[clipGradNorm] no gradients");
    need_periods(periods, grads.size(), slots_, "clipGradNorm");
    const int level = lowest_level(grads);
    need_level(level, 3 + polynomialDepth(degree), "clipGradNorm");
    const Evaluator &ev = eval_;
    // 2 / bound^2 is a whole number of units of the scale.  Below 2^20 of them the rounding would be seen: the bound is widened to where they are whole, and the polynomial is that of the wider one.
    // With eight, the fewest, that is by up to 1/16 (at a scale of 2^42: bounds of 10^6), where the kink of a degree of 15 at bound = 4 max_norm comes out to 0.036 instead of 0.033.
    const double unit = ev.scale(level - 1);
    double factor_u = 2.0 / (bound * bound);
    if (factor_u * unit < 0x1p20) {
        const double whole = std::floor(factor_u * unit);
        if (whole < 8.0) throw std::invalid_argument("[clipGradNorm] the bound is too large for the scale: 2 / bound^2 has less than eight units of it");
        factor_u = whole / unit;
        c = clipPolynomial(max_norm, std::sqrt(2.0 / factor_u), degree);
    }
    Ciphertext square = gradNormSquared(grads, periods);
    const Ciphertext u = ev.rescale(ev.combine({&square}, {factor_u}, -1.0));
    const Ciphertext factor = evaluate(eval_, u, c);
    std::vector<Ciphertext> low;
    for (const Ciphertext *x : grads) low.push_back(down(ev, *x, factor.getLevel()));
    std::vector<Ciphertext> products = ev.scaleMany(low, factor), out;
    low.clear();
    // Small handles share the launches of their key switches, up to kTogether members: clipping 48 of one member, with 1, 8, 24, 64 members and all of them at once, 8.8, 7.1, 6.9, 6.8 and 6.8 ms; those
    // and three of 18 11.7, 10.0, 9.7, 9.7 and 9.5; twelve of four 6.3, 6.3, 6.1, 5.9 and 5.9.  More than 24 would give 2 % for temporaries that grow with the members.
    constexpr int kTogether = 24;
    for (size_t k = 0; k < products.size();) {
        size_t end = k;
        int members = 0;
        while (end < products.size() && (end == k || members + products[end].getBatch() <= kTogether)) members += products[end++].getBatch();
        if (end == k + 1) out.push_back(switched(ev, products[k]));
        else {
            std::vector<Ciphertext> part;
            for (size_t i = k; i < end; ++i) part.push_back(ev.view(products[i], 0, products[i].getBatch()));
            const Ciphertext all = switched(ev, ev.concat(part));
            int at = 0;
            for (size_t i = k; i < end; ++i) { out.push_back(ev.slice(all, at, products[i].getBatch())); at += products[i].getBatch(); }
        }
        k = end;
    }
    if (norm_squared) *norm_squared = std::move(square);
    return out;
}

} // namespace HELLM
