// Tensor products of all pairs of query and key tiles of a head (sm_100a).
//
// Tiles of one head are rows of two matrices over the residues, a [groups][nq] and b [groups][nk], each entry a polynomial pair (b, a), and
//     d[j][h][i] (+)= sum_g (b1 b2, a1 b2 + a2 b1, a1 a2),   (b1, a1) = a[g][h][i], (b2, a2) = b[g][h][j]
// is a matrix product at every residue.  Pair by pair (k_tensor) every product reads its own four words; here a warp takes up to 4 x 4 pairs of tiles, so that a
// word is read once for four products.  Its lanes are LR x LC blocks of TR x TC pairs, side by side for 32 / (LR LC) residues; the words of all its tiles come
// through a ring of stages in shared memory that belongs to the warp alone (16-byte asynchronous copies, several groups ahead), from which every lane reads the
// tiles of its block.  The ring runs on from one range of residues to the next.
// 8 groups, 6 heads, 4 query and 8 key tiles at level 5: 1.35 to 1.43 ms from box to box, with 5.4 GB (0.83 ms of HBM), 0.4 ms of FP64 and the 60-bit limb, a sixth of the products and a
// quarter of the time, which overlap in part: the grid has one limb after the other, so the CTAs of an SM have the same kind of work.  Into an accumulator, whose words are loaded only where they
// are added: 2.8 ms, with 1.8 GB more.  Words straight to registers: 2.2 ms.  Rings of 2, 3, 4, 6 and 8 stages, in one run: 1.95, 1.35, 1.30, 1.49 and 1.50 ms (the reads of the ring wait behind the copies in flight).  Twice
// as many pairs a warp (8 x 4, 168 registers): 1.5 ms; boxes of 64 residues by tensor-map copies and a ring of the CTA: 1.54 ms.  One query tile with four key tiles: 270 us, 98 % of the bandwidth.
// The middle sum comes from one product of the sums, (b1 + a1)(b2 + a2), from which the outer two are taken off at the end: three products a pair.
#pragma once
#include "kernels.cuh"
#include <type_traits>

namespace hb {

struct PairShape { int groups, heads, nq, nk; };
// Side R (rows of a block of pairs) has at least as many tiles as side C: queries or keys, whichever are more.
struct PairSides { const u64 *r, *c; int nr, nc, keys_r; };
template <int TR, int TC, int LR, int LC> struct PairTile {
    static constexpr int kRows = TR * LR, kCols = TC * LC, kBlocks = LR * LC, kX = 32 / kBlocks; // tiles of a warp's block; residues
    static constexpr int kLines = 2 * (kRows + kCols), kStage = kLines * kX;                      // polynomials; words of a stage
    static constexpr int kCopies = kLines * kX / 64;                                              // 16-byte copies of a lane for a stage
    static constexpr int kStages = 4;
    static constexpr size_t kSmem = (size_t)8 * kStages * kStage * 8;
    static __host__ __device__ constexpr bool on_side_c(int copy) { return copy * 32 / (kX / 2) >= 2 * kRows; }
    static_assert(kLines * kX % 64 == 0 && 4 * kRows * kX % 128 == 0, "a stage is a whole number of copies a lane, and so are its sides");
};
// grid = (N / (8 kX run) * blocks of pairs, heads * n): eight warps side by side, `run` ranges one after the other
template <int TR, int TC, int LR, int LC>
__global__ void __launch_bounds__(256, 2) k_tensor_pairs(u64 *d, PairSides sides, PairShape s, int run, int n, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, int N, int accumulate) {
    using T = PairTile<TR, TC, LR, LC>;
    constexpr int X = T::kX, S = T::kStages;
    extern __shared__ __align__(16) u64 words[];
    const int br = (sides.nr + T::kRows - 1) / T::kRows, blocks = br * ((sides.nc + T::kCols - 1) / T::kCols), blk = blockIdx.x % blocks, r0 = blk % br * T::kRows, c0 = blk / br * T::kCols;
    const int h = blockIdx.y / n, l = blockIdx.y % n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PrimeConst m = pc[map.prime[l]];
    const size_t poly = (size_t)n * N;
    const u32 x0 = blockIdx.x / blocks * (u32)(8 * X * run) + warp * X; // of the warp's first range
    u64 *const ring = words + warp * (S * T::kStage);
    // Lines of a stage: entry ((t * 2 + polynomial) * L + block) of a side has tile t of lane block `block`, so that the blocks of one instruction read neighbouring lines.
    // A lane's copies: two residues of the lines (lane + 32 i) / (X / 2)
    const u64 *from[T::kCopies];
#pragma unroll
    for (int i = 0; i < T::kCopies; ++i) {
        const bool col = T::on_side_c(i);
        const int q = lane + 32 * i, line = q / (X / 2), part = q % (X / 2), e = col ? line - 2 * T::kRows : line, L = col ? LC : LR, count = col ? sides.nc : sides.nr;
        const int tile = (col ? c0 : r0) + (e % L) * (col ? TC : TR) + e / (2 * L);
        from[i] = (col ? sides.c : sides.r) + (((size_t)h * count + min(tile, count - 1)) * 2 + e / L % 2) * poly + (size_t)l * N + x0 + 2 * part; // past the end: the last tile again, not stored
    }
    const i64 step_r = (i64)s.heads * sides.nr * 2 * poly, step_c = (i64)s.heads * sides.nc * 2 * poly, wrap_r = 8 * X - (s.groups - 1) * step_r, wrap_c = 8 * X - (s.groups - 1) * step_c;
    const u32 ring_at = smem_u32(ring) + lane * 16;
    int f_group = 0, f_stage = 0;
    auto fetch = [&] {
        const u32 to = ring_at + f_stage * (T::kStage * 8);
        const bool last = ++f_group == s.groups;
        const i64 by_r = last ? wrap_r : step_r, by_c = last ? wrap_c : step_c;
#pragma unroll
        for (int i = 0; i < T::kCopies; ++i) {
            cp_async16(to + i * 512, from[i]);
            from[i] += T::on_side_c(i) ? by_c : by_r;
        }
        if (last) f_group = 0;
        if (++f_stage == S) f_stage = 0;
    };
    const int total = s.groups * run;
    pdl_wait();
#pragma unroll 1
    for (int i = 0; i < S - 1; ++i) {
        if (i < total) fetch();
        cp_async_commit();
    }
    const int block = lane / X, lr = block % LR, lc = block / LR;
    const u64 *const mine_r = ring + lr * X + lane % X, *const mine_c = ring + (2 * T::kRows + lc) * X + lane % X;
    int stage = 0, left = total;
    auto next = [&](u64 (&vr)[TR][2], u64 (&vc)[TC][2]) {
        cp_async_wait<S - 2>();
        __syncwarp();
        const int at = stage * T::kStage;
#pragma unroll
        for (int t = 0; t < TR; ++t) { vr[t][0] = mine_r[at + (2 * t) * LR * X]; vr[t][1] = mine_r[at + (2 * t + 1) * LR * X]; }
#pragma unroll
        for (int t = 0; t < TC; ++t) { vc[t][0] = mine_c[at + (2 * t) * LC * X]; vc[t][1] = mine_c[at + (2 * t + 1) * LC * X]; }
        if (++stage == S) stage = 0;
        // the stage that the copies go to was read a step ago, by all lanes before the barrier above
        if (left > S - 1) fetch();
        cp_async_commit();
        --left;
    };
    const size_t to_row = (sides.keys_r ? (size_t)s.heads * s.nq : 1) * 3 * poly, to_col = (sides.keys_r ? 1 : (size_t)s.heads * s.nq) * 3 * poly; // from one pair to the next
    const int row = r0 + lr * TR, col = c0 + lc * TC;
    u64 *to = d + (size_t)h * s.nq * 3 * poly + row * to_row + col * to_col + (size_t)l * N + x0 + lane % X;
    auto store = [&](int i, int j, u64 v0, u64 v01, u64 v2) { // v01: the product of the sums
        if (row + i >= sides.nr || col + j >= sides.nc) return;
        const u64 v[3] = {v0, sub_mod(sub_mod(v01, v0, m.q), v2, m.q), v2};
        u64 *o = to + i * to_row + j * to_col;
#pragma unroll
        for (int k = 0; k < 3; ++k) o[k * poly] = accumulate ? add_mod(v[k], o[k * poly], m.q) : v[k];
    };
    // `run` ranges: the sums of all groups, `room` of them before the sums are reduced.  TWO at a time: FP64 sums change registers at every product.
    auto ranges = [&](auto two, auto &sums, int room, auto &&relax, auto &&step, auto &&finish) {
        constexpr bool TWO = decltype(two)::value;
#pragma unroll 1
        for (int item = 0; item < run; ++item) {
#pragma unroll
            for (int i = 0; i < TR * TC * 3; ++i) sums[i].zero();
#pragma unroll 1
            for (int g = 0; g < s.groups; g += room) {
                if (g) {
#pragma unroll
                    for (int i = 0; i < TR * TC * 3; ++i) relax(sums[i]);
                }
                const int some = min(room, s.groups - g);
                auto one = [&] {
                    u64 vr[TR][2], vc[TC][2];
                    next(vr, vc);
                    step(vr, vc);
                };
                int e = 0;
                if constexpr (TWO) {
#pragma unroll 1
                    for (; e + 1 < some; e += 2) { one(); one(); }
                }
#pragma unroll 1
                for (; e < some; ++e) one();
            }
#pragma unroll
            for (int i = 0; i < TR; ++i)
#pragma unroll
                for (int j = 0; j < TC; ++j) {
                    const int at = (i * TC + j) * 3;
                    store(i, j, finish(sums[at]), finish(sums[at + 1]), finish(sums[at + 2]));
                }
            to += 8 * X;
        }
    };
    if (m.fp) { // exact sums: the sums of two residues below 2^42 leave room for 32 products, below 2^44 for two
        const double qd = (double)m.q;
        FpAcc sums[TR * TC * 3];
        ranges(
            std::true_type{}, sums, m.q < (1ull << 42) ? 32 : 2, [&](FpAcc &a) { a.relax(m.q_inv_f, qd); },
            [&](const u64 (&vr)[TR][2], const u64 (&vc)[TC][2]) {
                double dr[TR][3], dc[TC][3];
#pragma unroll
                for (int i = 0; i < TR; ++i) { dr[i][0] = u52_to_double(vr[i][0]); dr[i][2] = u52_to_double(vr[i][1]); dr[i][1] = dr[i][0] + dr[i][2]; }
#pragma unroll
                for (int j = 0; j < TC; ++j) { dc[j][0] = u52_to_double(vc[j][0]); dc[j][2] = u52_to_double(vc[j][1]); dc[j][1] = dc[j][0] + dc[j][2]; }
#pragma unroll
                for (int i = 0; i < TR; ++i)
#pragma unroll
                    for (int j = 0; j < TC; ++j)
#pragma unroll
                        for (int k = 0; k < 3; ++k) sums[(i * TC + j) * 3 + k].mac(dr[i][k], dc[j][k]);
            },
            [&](const FpAcc &a) { return a.finish(m.q_inv_f, qd); });
    } else { // pieces of 30 bits, eight products at a time; the sums of two residues are reduced first
        PieceAcc sums[TR * TC * 3];
        ranges(
            std::false_type{}, sums, 8, [&](PieceAcc &a) { a.relax(m); },
            [&](const u64 (&vr)[TR][2], const u64 (&vc)[TC][2]) {
#pragma unroll
                for (int k = 0; k < 3; ++k) {
                    u64 wr[TR], wc[TC];
#pragma unroll
                    for (int i = 0; i < TR; ++i) wr[i] = k == 1 ? add_mod(vr[i][0], vr[i][1], m.q) : vr[i][k / 2];
#pragma unroll
                    for (int j = 0; j < TC; ++j) wc[j] = k == 1 ? add_mod(vc[j][0], vc[j][1], m.q) : vc[j][k / 2];
#pragma unroll
                    for (int i = 0; i < TR; ++i)
#pragma unroll
                        for (int j = 0; j < TC; ++j) sums[(i * TC + j) * 3 + k].mac(wr[i], wc[j]);
                }
            },
            [&](const PieceAcc &a) { return a.finish(m); });
    }
}

} // namespace hb
