// Tensor products of all pairs of query and key tiles of a head (sm_100a).
//
// Members of one head are rows of two matrices over the residues, a [groups][nq] and b [groups][nk], each entry a polynomial pair (b, a), and
//     d[j][h][i] (+)= sum_g (b1 b2, a1 b2 + a2 b1, a1 a2),   (b1, a1) = a[g][h][i], (b2, a2) = b[g][h][j]
// is a matrix product at every residue.  Tile by tile (k_tensor) every pair reads its own four words; here a thread keeps QI x KJ pairs of one residue in
// registers, so a word of a serves KJ pairs and a word of b QI.
// The middle sum comes from one product of the sums, (b1 + a1)(b2 + a2), from which the outer two are taken off at the end: three products a pair.
#pragma once
#include "kernels.cuh"

namespace hb {

struct PairShape { int groups, heads, nq, nk; };
// a [groups][heads][nq][2][n][N], b [groups][heads][nk][2][n][N], d [nk][heads][nq][3][n][N].  Blocks of pairs of one residue range run side by side and find
// its words in L2.  grid = (N / 256 * blocks of pairs, heads * n)
template <int QI, int KJ>
__global__ void __launch_bounds__(256, 2) k_tensor_pairs(u64 *d, const u64 *a, const u64 *b, PairShape s, int n, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, int N, int accumulate) {
    const int bq = (s.nq + QI - 1) / QI, blocks = bq * ((s.nk + KJ - 1) / KJ), blk = blockIdx.x % blocks, i0 = blk % bq * QI, j0 = blk / bq * KJ;
    const int h = blockIdx.y / n, l = blockIdx.y % n;
    const u32 x = blockIdx.x / blocks * 256 + threadIdx.x;
    const PrimeConst m = pc[map.prime[l]];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + x;
    const u64 *ap[QI], *bp[KJ];
#pragma unroll
    for (int i = 0; i < QI; ++i) ap[i] = a + ((size_t)h * s.nq + min(i0 + i, s.nq - 1)) * 2 * poly + at; // past the end: the last one again, not stored
#pragma unroll
    for (int j = 0; j < KJ; ++j) bp[j] = b + ((size_t)h * s.nk + min(j0 + j, s.nk - 1)) * 2 * poly + at;
    const size_t a_step = (size_t)s.heads * s.nq * 2 * poly, b_step = (size_t)s.heads * s.nk * 2 * poly;
    u64 r[QI][KJ][3];
    pdl_wait();
    auto terms = [&](auto &&product) {
        for (int g = 0; g < s.groups; ++g) {
            u64 va[QI][2], vb[KJ][2];
#pragma unroll
            for (int i = 0; i < QI; ++i) { va[i][0] = ap[i][0]; va[i][1] = ap[i][poly]; ap[i] += a_step; }
#pragma unroll
            for (int j = 0; j < KJ; ++j) { vb[j][0] = bp[j][0]; vb[j][1] = bp[j][poly]; bp[j] += b_step; }
            product(g, va, vb);
        }
    };
    if (m.fp) { // exact sums: the sums of two residues below 2^42 leave room for 32 products, below 2^44 for two
        const double qd = (double)m.q;
        const int room = m.q < (1ull << 42) ? 32 : 2;
        FpAcc acc[QI][KJ][3];
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int k = 0; k < 3; ++k) acc[i][j][k].zero();
        terms([&](int g, const u64 (&va)[QI][2], const u64 (&vb)[KJ][2]) {
            if (g && g % room == 0) {
#pragma unroll
                for (int i = 0; i < QI; ++i)
#pragma unroll
                    for (int j = 0; j < KJ; ++j)
#pragma unroll
                        for (int k = 0; k < 3; ++k) acc[i][j][k].relax(m.q_inv_f, qd);
            }
            double da[QI][3], db[KJ][3];
#pragma unroll
            for (int i = 0; i < QI; ++i) { da[i][0] = u52_to_double(va[i][0]); da[i][2] = u52_to_double(va[i][1]); da[i][1] = da[i][0] + da[i][2]; }
#pragma unroll
            for (int j = 0; j < KJ; ++j) { db[j][0] = u52_to_double(vb[j][0]); db[j][2] = u52_to_double(vb[j][1]); db[j][1] = db[j][0] + db[j][2]; }
#pragma unroll
            for (int i = 0; i < QI; ++i)
#pragma unroll
                for (int j = 0; j < KJ; ++j)
#pragma unroll
                    for (int k = 0; k < 3; ++k) acc[i][j][k].mac(da[i][k], db[j][k]);
        });
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
#pragma unroll
                for (int k = 0; k < 3; ++k) r[i][j][k] = acc[i][j][k].finish(m.q_inv_f, qd);
                r[i][j][1] = sub_mod(sub_mod(r[i][j][1], r[i][j][0], m.q), r[i][j][2], m.q);
            }
    } else { // the middle sum takes two products a group
        PieceAcc acc[QI][KJ][3];
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int k = 0; k < 3; ++k) acc[i][j][k].zero();
        terms([&](int g, const u64 (&va)[QI][2], const u64 (&vb)[KJ][2]) {
            if (g && g % 4 == 0) {
#pragma unroll
                for (int i = 0; i < QI; ++i)
#pragma unroll
                    for (int j = 0; j < KJ; ++j)
#pragma unroll
                        for (int k = 0; k < 3; ++k) acc[i][j][k].relax(m);
            }
#pragma unroll
            for (int i = 0; i < QI; ++i)
#pragma unroll
                for (int j = 0; j < KJ; ++j) {
                    acc[i][j][0].mac(va[i][0], vb[j][0]); acc[i][j][2].mac(va[i][1], vb[j][1]);
                    acc[i][j][1].mac(va[i][1], vb[j][0]); acc[i][j][1].mac(va[i][0], vb[j][1]);
                }
        });
#pragma unroll
        for (int i = 0; i < QI; ++i)
#pragma unroll
            for (int j = 0; j < KJ; ++j)
#pragma unroll
                for (int k = 0; k < 3; ++k) r[i][j][k] = acc[i][j][k].finish(m);
    }
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            if (i0 + i >= s.nq || j0 + j >= s.nk) continue;
            u64 *o = d + (((size_t)(j0 + j) * s.heads + h) * s.nq + i0 + i) * 3 * poly + at;
#pragma unroll
            for (int k = 0; k < 3; ++k) o[k * poly] = accumulate ? add_mod(r[i][j][k], o[k * poly], m.q) : r[i][j][k];
        }
}

} // namespace hb
