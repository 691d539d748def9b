// Sums of squares, products with one factor and gradients of a layer norm on ciphertexts (sm_100a).
//
// Members x[t][b] (t column tiles, outermost; b token tiles) are polynomial pairs (x0, x1); (x) is the tensor product (x0 y0, x0 y1 + x1 y0, x1 y1).  At every residue
//   squares      out[b]    = sum_t (x[t][b] - m[b])^2 - pad m[b]^2
//   scale        out[t][b] = (x[t][b] - m[b]) (x) r[b]
//   affine       out[t][b] = x[t][b] g[t] + K (beta[t], 0)
//   grad sums    rows[b] = sum_t g[t][b] (x) xhat[t][b], cols[t] = sum_b dy[t][b] (x) xhat[t][b], and the plain sums of g and dy over the same indices
//   grad input   out[t][b] = K (g[t][b] - m[b]) - xhat[t][b] (x) a[b]
// Sums are exact until one reduction at their end (FpAcc, PieceAcc).
//
// All of it is bound by HBM: a member's 18 to 58 FP64 instructions keep the pipes of an SM for 9 to 29 cycles a warp, its bytes take 22 to 77.  What it takes to be so bound, in the
// order of what it gave: words of the members ahead in flight while those before are multiplied (registers where every member has a result of its own, rings of asynchronous copies where they are
// summed, since a sum's registers leave no room), several members a CTA, no quotients by sizes, and addresses of a base that all threads share and a 32-bit offset.
#pragma once
#include "kernels.cuh"
#include <type_traits>

namespace hb {

// Residues as the sums of one kind of prime take them.
struct FpField { // primes below 2^44: whole numbers in doubles, differences with their sign
    using Value = double;
    using Sum = FpAcc;
    struct Plain { // of residues, as many between two reductions as a sum has room for products: below 2^49
        double v;
        __device__ __forceinline__ void zero() { v = 0.0; }
        __device__ __forceinline__ void add(double x) { v += x; }
        __device__ __forceinline__ u64 canonical(const PrimeConst &m) const { return canon_fp64(v, m.q_inv_f, (double)m.q); }
        __device__ __forceinline__ void relax(const PrimeConst &m) { v = u52_to_double(canonical(m)); }
    };
    struct Lean { // of products that are reduced one by one: half the registers of a Sum, seven instructions a product instead of four
        double v;
        __device__ __forceinline__ void zero() { v = 0.0; }
        __device__ __forceinline__ void add(const Lean &x, const PrimeConst &) { v += x.v; }
        __device__ __forceinline__ void set(double a, double b, const PrimeConst &m) { v = mul_fp64_lazy(a, b, m.q_inv_f, (double)m.q); }
        __device__ __forceinline__ void set(double a, double b, double c, double d, const PrimeConst &m) { v = mul_fp64_lazy(a, b, m.q_inv_f, (double)m.q) + mul_fp64_lazy(c, d, m.q_inv_f, (double)m.q); }
        __device__ __forceinline__ u64 canonical(const PrimeConst &m) const { return canon_fp64(v, m.q_inv_f, (double)m.q); } // 64 products below 2^44 in magnitude: below 2^50
        __device__ __forceinline__ void relax(const PrimeConst &m) { v = u52_to_double(canonical(m)); }
    };
    const PrimeConst &m;
    __device__ __forceinline__ explicit FpField(const PrimeConst &m_) : m(m_) {}
    __device__ __forceinline__ double value(u64 x) const { return u52_to_double(x); }
    __device__ __forceinline__ double minus(double a, double b) const { return a - b; }
    __device__ __forceinline__ double negative(double a) const { return -a; }
    static constexpr int kFewest = 8; // products of a sum before it is reduced, for the longest of these primes
    __device__ __forceinline__ int room() const { return m.q < (1ull << 42) ? 128 : kFewest; }
};
struct PieceField { // 45 to 60 bits
    using Value = u64;
    using Sum = PieceAcc;
    struct Plain { // of nine residues at most
        u64 v;
        __device__ __forceinline__ void zero() { v = 0; }
        __device__ __forceinline__ void add(u64 x) { v += x; }
        __device__ __forceinline__ u64 canonical(const PrimeConst &m) const { return canon_q(v, m.q, FoldQ{m.fold_shift, (1u << m.fold_shift) - 1u, m.fold_d}); }
        __device__ __forceinline__ void relax(const PrimeConst &m) { v = canonical(m); }
    };
    struct Lean {
        u64 v;
        __device__ __forceinline__ void zero() { v = 0; }
        __device__ __forceinline__ void add(const Lean &x, const PrimeConst &m) { v = add_mod(v, x.v, m.q); }
        __device__ __forceinline__ void set(u64 a, u64 b, const PrimeConst &m) { PieceAcc s; s.zero(); s.mac(a, b); v = s.finish(m); }
        __device__ __forceinline__ void set(u64 a, u64 b, u64 c, u64 d, const PrimeConst &m) { PieceAcc s; s.zero(); s.mac(a, b); s.mac(c, d); v = s.finish(m); }
        __device__ __forceinline__ u64 canonical(const PrimeConst &) const { return v; }
        __device__ __forceinline__ void relax(const PrimeConst &) {}
    };
    const PrimeConst &m;
    __device__ __forceinline__ explicit PieceField(const PrimeConst &m_) : m(m_) {}
    __device__ __forceinline__ u64 value(u64 x) const { return x; }
    __device__ __forceinline__ u64 minus(u64 a, u64 b) const { return sub_mod(a, b, m.q); }
    __device__ __forceinline__ u64 negative(u64 a) const { return m.q - a; } // up to q: products stay below 2^120
    static constexpr int kFewest = 8;
    __device__ __forceinline__ int room() const { return kFewest; }
};
template <class F> __device__ __forceinline__ void by_prime(const PrimeConst &m, F &&f) {
    if (m.fp) f(FpField(m)); else f(PieceField(m));
}

// Two residues side by side: 16 bytes a load, and two chains of arithmetic a thread.
struct Two { u64 v[2]; };
__device__ __forceinline__ Two load2(const u64 *p) { const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(p); return {{x.x, x.y}}; }
__device__ __forceinline__ void store2(u64 *p, const Two &x) { *reinterpret_cast<ulonglong2 *>(p) = make_ulonglong2(x.v[0], x.v[1]); }
// a polynomial pair at two residues
struct Pair {
    Two p[2];
    // at a short offset from an address that all threads share: whole pointers would take more registers than the words
    __device__ __forceinline__ void load(const u64 *from, size_t poly, u32 at) { p[0] = load2(from + at); p[1] = load2(from + poly + at); }
    template <class F, class V> __device__ __forceinline__ void values(const F &f, V (&v0)[2], V (&v1)[2]) const {
#pragma unroll
        for (int e = 0; e < 2; ++e) { v0[e] = f.value(p[0].v[e]); v1[e] = f.value(p[1].v[e]); }
    }
};
constexpr int kNormLanes = 512; // residues of a CTA: two a thread

// Members one after the other, or wherever a list says.
struct MemberRun {
    const u64 *p;
    size_t stride;
    __device__ __forceinline__ const u64 *at(int i) const { return p + i * stride; }
};
constexpr int kListMembers = 256; // of a launch
struct MemberList {
    const u64 *p[kListMembers];
    __device__ __forceinline__ const u64 *at(int i) const { return p[i]; }
};
struct OutRun {
    u64 *p;
    size_t stride;
    __device__ __forceinline__ u64 *at(int i) const { return p + i * stride; }
};
struct OutList {
    u64 *p[kListMembers];
    __device__ __forceinline__ u64 *at(int i) const { return p[i]; }
};

// out[b] (+)= the sum over t < groups, for `chunk` token tiles one after the other.  Threads of a CTA: `splits` parts (a power of two) of the members by 512 / splits residues; the
// parts, which have a chunk of one, are joined in shared memory, in order.  Words come through a ring of members, which every thread fills for itself: of a token tile the mean first, then the members.
// Level 5, us (floor: the bytes at the copy bandwidth): 3 tiles of 4 token tiles 24 (21), of 16 85 (85), 8 of 16 162 (162), 102 members of a list 97 (100).  Words straight to registers, four
// members ahead, two CTAs an SM: 31, 107, 188 and 103; rings of five and six stages and two CTAs, which let the sums of two members go without moves: 25.0 and 25.1, 88 and 86, 165 and 162, 99 and 97; four
// CTAs of 64 registers, which spill: 35, 111, 223 and 196.  The third CTA costs the sums with a mean 12 bytes of spills.
// grid = (N splits / 512, n, chunks): quotients by sizes would take a fifth of the instructions
struct SquareShape { int groups, batch, chunk, log_splits; u64 pad; };
constexpr int kSquareStages = 4;
constexpr size_t square_smem() { return (size_t)kSquareStages * 2 * kNormLanes * 8; }
template <class MEMBERS, bool MEAN>
__global__ void __launch_bounds__(256, 3) k_square_sums(u64 *out, const __grid_constant__ MEMBERS x, const u64 *mean, SquareShape w, int n, const PrimeConst *__restrict__ pc, int N, int accumulate) {
    constexpr int S = kSquareStages;
    extern __shared__ __align__(16) u64 words[]; // [S][2][512]; of parts, which have one token tile a CTA, [3][512] in the end
    const int splits = 1 << w.log_splits, wide = 256 >> w.log_splits, lane = threadIdx.x & (wide - 1), part = threadIdx.x >> (8 - w.log_splits);
    const int l = blockIdx.y, first = blockIdx.z * w.chunk, last = min(first + w.chunk, w.batch);
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N;
    const u32 at = (u32)(l * N) + (blockIdx.x * wide + lane) * 2;
    const int count = (w.groups - part + splits - 1) >> w.log_splits; // members of this part
    const u32 ring = smem_u32(words + 2 * threadIdx.x);
    int f_b = first, f_t = MEAN ? -1 : 0, f_stage = 0, stage = 0; // what is fetched next (-1: the mean), and what is read next
    auto fetch = [&] {
        if (f_b < last) {
            const u64 *p = MEAN && f_t < 0 ? mean + (size_t)f_b * 2 * poly : x.at((part + f_t * splits) * w.batch + f_b);
            const u32 to = ring + f_stage * (2 * kNormLanes * 8);
            cp_async16(to, p + at); cp_async16(to + kNormLanes * 8, p + poly + at);
            if (++f_t == count) { f_t = MEAN ? -1 : 0; ++f_b; }
            if (++f_stage == S) f_stage = 0;
        }
        cp_async_commit();
    };
    pdl_wait();
#pragma unroll
    for (int j = 0; j < S - 1; ++j) fetch();
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        using Sum = typename decltype(f)::Sum;
        auto next = [&](V (&v0)[2], V (&v1)[2]) {
            cp_async_wait<S - 2>();
            const u64 *y = words + stage * (2 * kNormLanes) + 2 * threadIdx.x;
            const Two a = load2(y), c = load2(y + kNormLanes);
#pragma unroll
            for (int e = 0; e < 2; ++e) { v0[e] = f.value(a.v[e]); v1[e] = f.value(c.v[e]); }
            if (++stage == S) stage = 0;
            fetch(); // into the stage that this thread read a member ago
        };
#pragma unroll 1
        for (int b = first; b < last; ++b) {
            Sum s[3][2];
            V m0[2], m1[2];
            if (MEAN) next(m0, m1);
#pragma unroll
            for (int e = 0; e < 2; ++e) { s[0][e].zero(); s[1][e].zero(); s[2][e].zero(); }
            auto member = [&] {
                V v0[2], v1[2];
                next(v0, v1);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (MEAN) { v0[e] = f.minus(v0[e], m0[e]); v1[e] = f.minus(v1[e], m1[e]); }
                    s[0][e].mac(v0[e], v0[e]); s[1][e].mac(v0[e], v1[e]); s[2][e].mac(v1[e], v1[e]);
                }
            };
#pragma unroll 1
            for (int t = 0; t < count; t += f.room()) {
                if (t) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) { s[k][0].relax(m); s[k][1].relax(m); }
                }
                const int some = min(f.room(), count - t);
#pragma unroll 1
                for (int i = 0; i < some; ++i) member(); // one by one: two a turn would save moves and cost the third CTA its registers
            }
            Two r[3];
#pragma unroll
            for (int k = 0; k < 3; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) r[k].v[e] = s[k][e].canonical(m);
            if (MEAN && w.pad && part == 0) { // less what members of padding have added
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[0][e].zero(); s[1][e].zero(); s[2][e].zero();
                    s[0][e].mac(m0[e], m0[e]); s[1][e].mac(m0[e], m1[e]); s[2][e].mac(m1[e], m1[e]);
#pragma unroll
                    for (int k = 0; k < 3; ++k) r[k].v[e] = sub_mod(r[k].v[e], mul_mod_any(s[k][e].canonical(m), w.pad, m), m.q);
                }
            }
            if (splits > 1) {
                u64 *const parts = words;
                __syncthreads(); // all members have been read
#pragma unroll
                for (int k = 0; k < 3; ++k) store2(parts + k * kNormLanes + 2 * threadIdx.x, r[k]);
                __syncthreads();
                if (part) continue;
                for (int j = 1; j < splits; ++j)
#pragma unroll
                    for (int k = 0; k < 3; ++k) {
                        const Two y = load2(parts + k * kNormLanes + 2 * (threadIdx.x + j * wide));
#pragma unroll
                        for (int e = 0; e < 2; ++e) r[k].v[e] = add_mod(r[k].v[e], y.v[e], m.q);
                    }
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) r[1].v[e] = add_mod(r[1].v[e], r[1].v[e], m.q);
            u64 *o = out + (size_t)b * 3 * poly + at;
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                if (accumulate) {
                    const Two y = load2(o + k * poly);
#pragma unroll
                    for (int e = 0; e < 2; ++e) r[k].v[e] = add_mod(r[k].v[e], y.v[e], m.q);
                }
                store2(o + k * poly, r[k]);
            }
        }
    });
}
// Members c, c + step, ... of a column c < step, `each` of them; a CTA takes a chunk of them one after the other.
struct Walk { int each, step, chunk; };
// out[i] = (x[i] - mean[c]) (x) r[c] for the members i = c, c + step, ... of column c < step: mean and factor are read once for a chunk of members.  EACH: a factor per member.
// Level 5, us (floor): 3 tiles of 4 token tiles 39 (37), of 16 142 (146), 8 of 16 335 (339); 102 members of a list 252 (246).
// grid = (N / 512, n, step * chunks)
template <class MEMBERS, class OUT, bool MEAN, bool EACH>
__global__ void __launch_bounds__(256, 4) k_scale_members(const __grid_constant__ OUT out, const __grid_constant__ MEMBERS x, const u64 *mean, const u64 *r, Walk w, int n, const PrimeConst *__restrict__ pc, int N) {
    const int l = blockIdx.y, c = (int)(blockIdx.z % (u32)w.step), first = (int)(blockIdx.z / (u32)w.step) * w.chunk, last = min(first + w.chunk, w.each);
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N;
    const u32 at = (u32)(l * N) + (blockIdx.x * 256 + threadIdx.x) * 2;
    Pair rr, mr{}, xr, er{};
    pdl_wait();
    // the first words do not wait for the constants of the prime, and those of the next member are in flight while this one is multiplied
    if (!EACH) rr.load(r + (size_t)c * 2 * poly, poly, at);
    if (MEAN) mr.load(mean + (size_t)c * 2 * poly, poly, at);
    auto fetch = [&](int t) {
        const int i = t * w.step + c;
        xr.load(x.at(i), poly, at);
        if (EACH) er.load(r + (size_t)i * 2 * poly, poly, at);
    };
    fetch(first);
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        V r0[2], r1[2], m0[2], m1[2];
        if (!EACH) rr.values(f, r0, r1);
        if (MEAN) mr.values(f, m0, m1);
#pragma unroll 1
        for (int t = first; t < last; ++t) {
            V v0[2], v1[2];
            xr.values(f, v0, v1);
            if (EACH) er.values(f, r0, r1);
            if (t + 1 < last) fetch(t + 1);
            Two d[3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (MEAN) { v0[e] = f.minus(v0[e], m0[e]); v1[e] = f.minus(v1[e], m1[e]); }
                typename decltype(f)::Sum s[3];
                s[0].zero(); s[1].zero(); s[2].zero();
                s[0].mac(v0[e], r0[e]); s[1].mac(v0[e], r1[e]); s[1].mac(v1[e], r0[e]); s[2].mac(v1[e], r1[e]);
#pragma unroll
                for (int k = 0; k < 3; ++k) d[k].v[e] = s[k].canonical(m);
            }
            u64 *o = out.at(t * w.step + c) + at;
#pragma unroll
            for (int k = 0; k < 3; ++k) store2(o + k * poly, d[k]);
        }
    });
}
// Plaintexts of the column tiles.
constexpr int kNormTiles = 128; // of a launch
struct AffineList { const u64 *gamma[kNormTiles], *beta[kNormTiles]; int tile0, tiles, batch, chunk; };
// members of the tiles tile0 ..: out = x gamma + K beta on the first polynomial, x gamma on the second; without gammas x + beta.  A CTA takes a chunk of one tile's members.
// Level 5, us (floor): 3 tiles of 4 token tiles 28.6 (26), of 16 100 (95), 8 of 16 264 (254).
// grid = (N / 512, n, tiles * chunks)
template <bool GAMMA>
__global__ void __launch_bounds__(256, 4) k_affine(u64 *out, const u64 *x, const __grid_constant__ AffineList a, const __grid_constant__ Scalars K, int n, const PrimeConst *__restrict__ pc, int N) {
    const int l = blockIdx.y, t = (int)(blockIdx.z % (u32)a.tiles), first = (int)(blockIdx.z / (u32)a.tiles) * a.chunk, last = min(first + a.chunk, a.batch);
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N;
    const u32 at = (u32)(l * N) + (blockIdx.x * 256 + threadIdx.x) * 2;
    const size_t from = ((size_t)a.tile0 + t) * a.batch * 2 * poly;
    Two be{}, ga{};
    Pair xr;
    auto fetch = [&](int b) { xr.load(x + from + (size_t)b * 2 * poly, poly, at); };
    pdl_wait();
    if (a.beta[t]) be = load2(a.beta[t] + at);
    if (GAMMA) ga = load2(a.gamma[t] + at);
    fetch(first);
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        V g[2] = {};
        if (GAMMA) {
            const V k = f.value(K.v[l]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                g[e] = f.value(ga.v[e]);
                typename decltype(f)::Sum s;
                s.zero();
                s.mac(f.value(be.v[e]), k);
                be.v[e] = s.canonical(m);
            }
        }
#pragma unroll 1
        for (int b = first; b < last; ++b) {
            Two v0 = xr.p[0], v1 = xr.p[1];
            if (b + 1 < last) fetch(b + 1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (GAMMA) {
                    typename decltype(f)::Sum s[2];
                    s[0].zero(); s[1].zero();
                    s[0].mac(f.value(v0.v[e]), g[e]); s[1].mac(f.value(v1.v[e]), g[e]);
                    v0.v[e] = s[0].canonical(m); v1.v[e] = s[1].canonical(m);
                }
                v0.v[e] = add_mod(v0.v[e], be.v[e], m.q);
            }
            u64 *o = out + from + (size_t)b * 2 * poly + at;
            store2(o, v0); store2(o + poly, v1);
        }
    });
}
// Both directions in one pass over dy, g and xhat.  A thread has one residue of TT column tiles: their sums over b stay in its registers, a word each, the sums over t of one b are written (+= for
// all but the first tiles of a call).  The words come through a ring of members in shared memory, which every thread fills for itself, several members ahead.  SAME: g is dy.
// Level 5, us (floor): 3 tiles of 4 token tiles 55 (51), of 16 195 (184), 8 of 16 478 to 498 (427), with g = dy 43 (40), 145 (138), 362 (304).  Sums over b as two words (h, l) a sum, registers for the words
// ahead: 61, 210 and 943 (spills); as one word, reduced at every product: 57, 201 and 561; with the ring 55, 195 and 480.  Tiles in teams of 128 threads that join their rows in shared memory
// behind a barrier a token tile: 579 for 8 of 16.  Stages and CTAs an SM by tiles: eight stages of 8 tiles 476, six 490, four 482; 6 tiles of 4 token tiles four stages and four CTAs 119, six and three 130.
// All tiles of 16 token tiles with four to eight stages and three to five CTAs: what is below is the best of them or within 2 %, but for 5 tiles (322; eight stages and three CTAs 313) and 6 (392; six and three 378, and
// with g = dy 277 and 264).  One tile wants four stages (91, six 108, and with g = dy eight 88 instead of 76); at five CTAs 4 tiles and more lose (6 tiles 426 to 480, 8 633 to 711), at four 8 tiles do (509).
// Without g = dy the 60-bit limb's sums spill 32, 108 and 156 bytes with 4, 5 and 6 tiles at four CTAs, which three CTAs do not make faster at 4 (249 against 253).
// grid = (N / 128, n)
struct GradShape { int batch, tile0; };
constexpr int grad_stages(int TT) { return TT == 1 || TT == 6 ? 4 : TT == 8 ? 8 : 6; }
constexpr size_t grad_smem(int TT, bool same) { return (size_t)grad_stages(TT) * (same ? 4 : 6) * 128 * 8; }
constexpr int grad_ctas(int TT) { return TT == 1 ? 7 : TT == 2 ? 5 : TT <= 6 ? 4 : 3; }
template <int TT, bool SAME, int S = grad_stages(TT)>
__global__ void __launch_bounds__(128, grad_ctas(TT)) k_grad_sums(u64 *rows, u64 *rowsum, u64 *cols, u64 *colsum, const u64 *dy, const u64 *g, const u64 *xhat, GradShape w, int n, const PrimeConst *__restrict__ pc, int N) {
    constexpr int P = SAME ? 4 : 6;
    extern __shared__ __align__(16) u64 words[]; // [S][P][128]
    const int l = blockIdx.y;
    const PrimeConst m = pc[l];
    // an address is one that all threads share, and a short offset: pointers of every tile and polynomial would take more registers than the sums
    const size_t poly = (size_t)n * N, per_tile = (size_t)w.batch * 2 * poly;
    const u32 at = (u32)(l * N) + blockIdx.x * 128 + threadIdx.x;
    const u32 ring = smem_u32(words + threadIdx.x);
    auto fetch = [&](int t, int b, u32 to) {
        const size_t i = (size_t)(w.tile0 + t) * per_tile + (size_t)b * 2 * poly;
        constexpr u32 line = 128 * 8;
        cp_async8(to, xhat + i + at); cp_async8(to + line, xhat + i + poly + at);
        cp_async8(to + 2 * line, dy + i + at); cp_async8(to + 3 * line, dy + i + poly + at);
        if (!SAME) { cp_async8(to + 4 * line, g + i + at); cp_async8(to + 5 * line, g + i + poly + at); }
    };
    pdl_wait();
#pragma unroll
    for (int j = 0; j < S - 1; ++j) {
        if (j / TT < w.batch) fetch(j % TT, j / TT, ring + j * (P * 1024));
        cp_async_commit();
    }
    by_prime(m, [&](auto f) {
        using F = decltype(f);
        using Rows = std::conditional_t<SAME, typename F::Lean, typename F::Sum>;
        typename F::Lean c[TT][3];
        typename F::Plain cs[TT][2];
#pragma unroll
        for (int t = 0; t < TT; ++t) {
#pragma unroll
            for (int k = 0; k < 3; ++k) c[t][k].zero();
            cs[t][0].zero(); cs[t][1].zero();
        }
        int held = 0, stage = 0;
#pragma unroll 1
        for (int b = 0; b < w.batch; ++b) {
            if (held == F::kFewest) { // members of a plain sum; a lean one has room for 32
#pragma unroll
                for (int t = 0; t < TT; ++t) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) c[t][k].relax(m);
                    cs[t][0].relax(m); cs[t][1].relax(m);
                }
                held = 0;
            }
            ++held;
            Rows r[3];
            typename F::Plain rs[2];
#pragma unroll
            for (int k = 0; k < 3; ++k) r[k].zero();
            rs[0].zero(); rs[1].zero();
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                cp_async_wait<S - 2>();
                const u64 *const y = words + stage * (P * 128) + threadIdx.x;
                const auto x0 = f.value(y[0]), x1 = f.value(y[128]), d0 = f.value(y[256]), d1 = f.value(y[384]), g0 = SAME ? d0 : f.value(y[512 % (P * 128)]), g1 = SAME ? d1 : f.value(y[640 % (P * 128)]);
                // into the stage that this thread has read a member ago
                if (b + (t + S - 1) / TT < w.batch) fetch((t + S - 1) % TT, b + (t + S - 1) / TT, ring + (stage ? stage - 1 : S - 1) * (P * 1024));
                cp_async_commit();
                if (++stage == S) stage = 0;
                typename F::Lean p[3];
                p[0].set(d0, x0, m); p[1].set(d0, x1, d1, x0, m); p[2].set(d1, x1, m);
#pragma unroll
                for (int k = 0; k < 3; ++k) c[t][k].add(p[k], m);
                cs[t][0].add(d0); cs[t][1].add(d1);
                if constexpr (SAME) {
#pragma unroll
                    for (int k = 0; k < 3; ++k) r[k].add(p[k], m);
                } else {
                    if (t && t % (F::kFewest / 2) == 0 && f.room() / 2 < TT) {
#pragma unroll
                        for (int k = 0; k < 3; ++k) r[k].relax(m);
                    }
                    r[0].mac(g0, x0); r[1].mac(g0, x1); r[1].mac(g1, x0); r[2].mac(g1, x1);
                }
                rs[0].add(g0); rs[1].add(g1);
            }
            const u64 res[5] = {r[0].canonical(m), r[1].canonical(m), r[2].canonical(m), rs[0].canonical(m), rs[1].canonical(m)};
            u64 *const o = rows + (size_t)b * 3 * poly, *const os = rowsum + (size_t)b * 2 * poly;
#pragma unroll
            for (int k = 0; k < 5; ++k) {
                u64 *p = (k < 3 ? o + k * poly : os + (k - 3) * poly) + at;
                *p = w.tile0 ? add_mod(res[k], *p, m.q) : res[k];
            }
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            u64 *const o = cols + (size_t)(w.tile0 + t) * 3 * poly + at, *const os = colsum + (size_t)(w.tile0 + t) * 2 * poly + at;
#pragma unroll
            for (int k = 0; k < 3; ++k) o[k * poly] = c[t][k].canonical(m);
            os[0] = cs[t][0].canonical(m); os[poly] = cs[t][1].canonical(m);
        }
    });
}
// One direction: out[j] = sum_i y(i, j) (x) xhat(i, j) and sum[j] = sum_i y(i, j), member (i, j) being i by_i + j by_j, for a chunk of results one after the other.  Parts and the ring as in
// k_square_sums.  Both directions, level 5, us (floor of one pass over dy, g and xhat): 12 tiles of 4 token tiles 228 (177), 24 of 2 at level 2 130 (101); six CTAs an SM 221 and 133, and 56 instead of 53
// for 40 tiles of 4 in a ring with 2^12 coefficients.  grid = (N splits / 256, n, chunks)
struct PairSumShape { int terms, results, by_i, by_j, chunk, log_splits; };
constexpr int kPairSumStages = 4, kPairSumLanes = 256;
constexpr size_t pair_sum_smem() { return (size_t)kPairSumStages * 4 * kPairSumLanes * 8; }
__global__ void __launch_bounds__(128, 5) k_pair_sums(u64 *out, u64 *sum, const u64 *y, const u64 *xhat, PairSumShape w, int n, const PrimeConst *__restrict__ pc, int N) {
    constexpr int S = kPairSumStages, L = kPairSumLanes;
    extern __shared__ __align__(16) u64 words[]; // [S][4][256]; of parts, which have one result a CTA, [5][256] in the end
    const int splits = 1 << w.log_splits, wide = 128 >> w.log_splits, lane = threadIdx.x & (wide - 1), part = threadIdx.x >> (7 - w.log_splits);
    const int l = blockIdx.y, first = blockIdx.z * w.chunk, last = min(first + w.chunk, w.results);
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N;
    const u32 at = (u32)(l * N) + (blockIdx.x * wide + lane) * 2;
    const int count = (w.terms - part + splits - 1) >> w.log_splits;
    const u32 ring = smem_u32(words + 2 * threadIdx.x);
    int f_j = first, f_i = 0, f_stage = 0, stage = 0;
    auto fetch = [&] {
        if (f_j < last) {
            const size_t from = ((size_t)(part + f_i * splits) * w.by_i + (size_t)f_j * w.by_j) * 2 * poly;
            const u32 to = ring + f_stage * (4 * L * 8);
            cp_async16(to, y + from + at); cp_async16(to + L * 8, y + from + poly + at);
            cp_async16(to + 2 * L * 8, xhat + from + at); cp_async16(to + 3 * L * 8, xhat + from + poly + at);
            if (++f_i == count) { f_i = 0; ++f_j; }
            if (++f_stage == S) f_stage = 0;
        }
        cp_async_commit();
    };
    pdl_wait();
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch();
    by_prime(m, [&](auto f) {
        using F = decltype(f);
        const int room = min(f.room() / 2, F::kFewest); // two products a member in the middle sums, and what a plain sum holds
#pragma unroll 1
        for (int j = first; j < last; ++j) {
            typename F::Sum s[3][2];
            typename F::Plain p[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) { s[0][e].zero(); s[1][e].zero(); s[2][e].zero(); p[0][e].zero(); p[1][e].zero(); }
#pragma unroll 1
            for (int t = 0; t < count; t += room) {
                if (t) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) { s[0][e].relax(m); s[1][e].relax(m); s[2][e].relax(m); p[0][e].relax(m); p[1][e].relax(m); }
                }
                const int some = min(room, count - t);
#pragma unroll 1
                for (int i = 0; i < some; ++i) {
                    cp_async_wait<S - 2>();
                    const u64 *v = words + stage * (4 * L) + 2 * threadIdx.x;
                    const Two a = load2(v), b = load2(v + L), c = load2(v + 2 * L), d = load2(v + 3 * L);
                    if (++stage == S) stage = 0;
                    fetch(); // into the stage that this thread read a member ago
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const auto y0 = f.value(a.v[e]), y1 = f.value(b.v[e]), x0 = f.value(c.v[e]), x1 = f.value(d.v[e]);
                        s[0][e].mac(y0, x0); s[1][e].mac(y0, x1); s[1][e].mac(y1, x0); s[2][e].mac(y1, x1);
                        p[0][e].add(y0); p[1][e].add(y1);
                    }
                }
            }
            Two r[5];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int k = 0; k < 3; ++k) r[k].v[e] = s[k][e].canonical(m);
                r[3].v[e] = p[0][e].canonical(m); r[4].v[e] = p[1][e].canonical(m);
            }
            if (splits > 1) {
                u64 *const parts = words;
                __syncthreads(); // all members have been read
#pragma unroll
                for (int k = 0; k < 5; ++k) store2(parts + k * L + 2 * threadIdx.x, r[k]);
                __syncthreads();
                if (part) continue;
                for (int q = 1; q < splits; ++q)
#pragma unroll
                    for (int k = 0; k < 5; ++k) {
                        const Two z = load2(parts + k * L + 2 * (threadIdx.x + q * wide));
#pragma unroll
                        for (int e = 0; e < 2; ++e) r[k].v[e] = add_mod(r[k].v[e], z.v[e], m.q);
                    }
            }
            u64 *const o = out + (size_t)j * 3 * poly + at, *const os = sum + (size_t)j * 2 * poly + at;
            store2(o, r[0]); store2(o + poly, r[1]); store2(o + 2 * poly, r[2]);
            store2(os, r[3]); store2(os + poly, r[4]);
        }
    });
}
// members c, c + step, ... of token tile c < step share mean and dot, which are read once for a chunk of them.  Level 5, us (floor): 3 tiles of 4 token tiles 51 (48), of 16 200 (192), 8 of 16
// 460 to 485 (462).  grid = (N / 512, n, step * chunks)
__global__ void __launch_bounds__(256, 3) k_grad_input(u64 *out, const u64 *g, const u64 *mean, const u64 *xhat, const u64 *dot, Walk w, const __grid_constant__ Scalars K, int n, const PrimeConst *__restrict__ pc,
                                                       int N) {
    const int l = blockIdx.y, c = (int)(blockIdx.z % (u32)w.step), first = (int)(blockIdx.z / (u32)w.step) * w.chunk, last = min(first + w.chunk, w.each);
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N;
    const u32 at = (u32)(l * N) + (blockIdx.x * 256 + threadIdx.x) * 2;
    pdl_wait();
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        V m0[2], m1[2], a0[2], a1[2];
        auto pair = [&](const u64 *p, V (&v0)[2], V (&v1)[2]) {
            Pair y;
            y.load(p, poly, at);
            y.values(f, v0, v1);
        };
        pair(mean + (size_t)c * 2 * poly, m0, m1);
        pair(dot + (size_t)c * 2 * poly, a0, a1);
        const V k = f.value(K.v[l]);
#pragma unroll 1
        for (int t = first; t < last; ++t) {
            const int i = t * w.step + c;
            V g0[2], g1[2], x0[2], x1[2];
            pair(g + (size_t)i * 2 * poly, g0, g1);
            pair(xhat + (size_t)i * 2 * poly, x0, x1);
            Two d[3];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const V n0 = f.negative(x0[e]), n1 = f.negative(x1[e]);
                typename decltype(f)::Sum s[3];
                s[0].zero(); s[1].zero(); s[2].zero();
                s[0].mac(f.minus(g0[e], m0[e]), k); s[0].mac(n0, a0[e]);
                s[1].mac(f.minus(g1[e], m1[e]), k); s[1].mac(n0, a1[e]); s[1].mac(n1, a0[e]);
                s[2].mac(n1, a1[e]);
#pragma unroll
                for (int j = 0; j < 3; ++j) d[j].v[e] = s[j].canonical(m);
            }
            u64 *o = out + (size_t)i * 3 * poly + at;
#pragma unroll
            for (int j = 0; j < 3; ++j) store2(o + j * poly, d[j]);
        }
    });
}

// ---- constants ----
// out = sum_j k[j] x_j + k0 on the first polynomial of every member, without the constant on the others; a plaintext of a constant would be N words of it.  32 members of two terms at level 5: 134 us, 4.3 TB/s;
// the sums of a polynomial have one member a token tile.
// grid = (N / 512, n, polynomials of all members)
constexpr int kCombineTerms = 16;
struct CombineList { const u64 *x[kCombineTerms]; u64 k[kCombineTerms][kMaxPrimes], k0[kMaxPrimes]; int count, np; };
__global__ void __launch_bounds__(256, 4) k_combine(u64 *out, const __grid_constant__ CombineList c, int n, const PrimeConst *__restrict__ pc, int N) {
    const int l = blockIdx.y;
    const PrimeConst m = pc[l];
    const size_t from = ((size_t)blockIdx.z * n + l) * N;
    const u32 at = (blockIdx.x * 256 + threadIdx.x) * 2;
    const u64 add = blockIdx.z % (u32)c.np ? 0 : c.k0[l];
    pdl_wait();
    by_prime(m, [&](auto f) {
        typename decltype(f)::Sum s[2];
        s[0].zero(); s[1].zero();
#pragma unroll 2
        for (int j = 0; j < c.count; ++j) {
            const Two x = load2(c.x[j] + from + at);
            if (j && j % f.kFewest == 0) { s[0].relax(m); s[1].relax(m); }
            const auto k = f.value(c.k[j][l]);
            s[0].mac(f.value(x.v[0]), k); s[1].mac(f.value(x.v[1]), k);
        }
        store2(out + from + at, Two{{add_mod(s[0].canonical(m), add, m.q), add_mod(s[1].canonical(m), add, m.q)}});
    });
}

} // namespace hb
