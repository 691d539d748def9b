// Ciphertext x plaintext products grouped by expert (sm_100a).
//
//     out[p][t] = sum_b sum_k pre[k][order[p]][b] (.) perm_{g_k}(w[e][t][b]),   e = the expert whose group position p lies in
// with groups of any size: k_matmul_acc for several inputs that share weights.  A thread works on one coefficient of both polynomials of M positions and T
// output tiles: a weight word is read (and converted) once for M positions, a copy word once for T tiles.  The blocks of one coefficient range, over
// all experts, run side by side, so that copies and weights come from L2 for all but the first of them.
#pragma once
#include "kernels.cuh"

namespace hb {

// What one launch works on: experts with their positions and weight words' addresses.  An argument, so that calls can be recorded and nothing is uploaded.
constexpr int kExpertPts = 384, kExpertGroups = 64, kExpertPositions = 256;
struct ExpertList {
    int experts, tiles, bcount;               // tiles: of this launch; w[(e * tiles + t) * bcount + b]
    int out_tiles, tile0;                     // member of position p and tile t: p * out_tiles + tile0 + t
    const u64 *w[kExpertPts];
    int first_block[kExpertGroups + 1];       // blocks of the experts before
    int first_pos[kExpertGroups + 1];         // positions of this launch before them
    int pos0;                                 // member positions before this launch's first
    int input[kExpertPositions];              // which input a position has
};
template <int T> constexpr int kExpertRing = T >= 3 ? 6 : 8;
template <int M, int T> constexpr size_t expert_smem() { return (size_t)kExpertRing<T> * (2 * M + T) * 256 * 8; }
// pre [copies][inputs][bcount][2][n][N].  grid = (N / 256 * blocks, n)
template <int M, int T>
__global__ void __launch_bounds__(256, 2) k_matmul_experts(u64 *out, const __grid_constant__ ExpertList el, const u64 *__restrict__ pre, int copies, int inputs, const u32 *__restrict__ gal, int n,
                                                           const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, int logn, int N) {
    extern __shared__ __align__(16) u64 words[];
    constexpr int kRing = kExpertRing<T>;
    const int blocks = el.first_block[el.experts], blk = blockIdx.x % blocks, l = blockIdx.y;
    int e = 0;
    while (blk >= el.first_block[e + 1]) ++e;
    const int tile_blocks = (el.tiles + T - 1) / T, in_e = blk - el.first_block[e];
    const int t0 = in_e % tile_blocks * T, p0 = el.first_pos[e] + in_e / tile_blocks * M, pn = min(M, el.first_pos[e + 1] - p0), tn = min(T, el.tiles - t0);
    const PrimeConst m = pc[map.prime[l]];
    const size_t poly = (size_t)n * N, limb = (size_t)l * N;
    const u32 x0 = blockIdx.x / blocks * 256 + threadIdx.x;
    const u64 *ring = words + threadIdx.x;
    const u32 ring_at = smem_u32(ring);
    const int bcount = el.bcount, total = copies * bcount;
    const u64 *const *w = el.w + (size_t)(e * el.tiles) * bcount;
    u64 *const o = out + ((size_t)(el.pos0 + p0) * el.out_tiles + el.tile0 + t0) * 2 * poly + limb + x0;

    // positions p .. p + MM - 1 of the block; past the end: the last one again, not stored
    auto body = [&](auto mm, int p, auto acc) {
        constexpr int MM = decltype(mm)::value, kStage = (2 * MM + T) * 256;
        using Acc = decltype(acc);
        const u64 *fa[MM];
#pragma unroll
        for (int i = 0; i < MM; ++i) fa[i] = pre + (size_t)el.input[p0 + min(p + i, pn - 1)] * bcount * 2 * poly + limb + x0;
        const size_t to_next_copy = (size_t)(inputs * bcount - bcount + 1) * 2 * poly;
        int fk = 0, fb = 0;
        u32 to = 0, g = __ldg(gal), src = g == 1 ? x0 : ntt_perm(x0, g, logn);
        auto fetch = [&] {
            const u32 r = ring_at + to;
#pragma unroll
            for (int i = 0; i < MM; ++i) { cp_async8(r + i * 4096, fa[i]); cp_async8(r + i * 4096 + 2048, fa[i] + poly); }
#pragma unroll
            for (int t = 0; t < T; ++t) cp_async8(r + (2 * MM + t) * 2048, w[min(t0 + t, el.tiles - 1) * bcount + fb] + limb + src);
            cp_async_commit();
            if (++fb < bcount) {
#pragma unroll
                for (int i = 0; i < MM; ++i) fa[i] += 2 * poly;
            } else if (fk + 1 < copies) {
                fb = 0; ++fk;
#pragma unroll
                for (int i = 0; i < MM; ++i) fa[i] += to_next_copy;
                g = __ldg(gal + fk);
                src = g == 1 ? x0 : ntt_perm(x0, g, logn);
            }
            to += kStage * 8;
            if (to == kRing * kStage * 8) to = 0;
        };
#pragma unroll 1
        for (int k = 0; k < kRing - 1; ++k) {
            if (k < total) fetch();
            else cp_async_commit();
        }
        Acc s[MM][T][2];
#pragma unroll
        for (int i = 0; i < MM; ++i)
#pragma unroll
            for (int t = 0; t < T; ++t) { s[i][t][0].zero(); s[i][t][1].zero(); }
        constexpr bool FP = std::is_same<Acc, FpAcc>::value;
        const double qd = (double)m.q;
        const int room = !FP ? 8 : m.q < (1ull << 42) ? 128 : 8;
        int held = 0, from = 0;
        auto term = [&](auto &&then) {
            cp_async_wait<kRing - 2>();
            const u64 *q = ring + from;
            u64 v[MM][2], wv[T];
#pragma unroll
            for (int i = 0; i < MM; ++i) { v[i][0] = q[i * 512]; v[i][1] = q[i * 512 + 256]; }
#pragma unroll
            for (int t = 0; t < T; ++t) wv[t] = q[(2 * MM + t) * 256];
            from += kStage;
            if (from == kRing * kStage) from = 0;
            then();
            if (++held > room) {
                held = 1;
#pragma unroll
                for (int i = 0; i < MM; ++i)
#pragma unroll
                    for (int t = 0; t < T; ++t)
#pragma unroll
                        for (int k = 0; k < 2; ++k) s[i][t][k].relax(m);
            }
            if constexpr (FP) {
                double vd[MM][2];
#pragma unroll
                for (int i = 0; i < MM; ++i) { vd[i][0] = u52_to_double(v[i][0]); vd[i][1] = u52_to_double(v[i][1]); }
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const double wd = u52_to_double(wv[t]);
#pragma unroll
                    for (int i = 0; i < MM; ++i) { s[i][t][0].mac(vd[i][0], wd); s[i][t][1].mac(vd[i][1], wd); }
                }
            } else {
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int i = 0; i < MM; ++i) { s[i][t][0].mac(v[i][0], wv[t]); s[i][t][1].mac(v[i][1], wv[t]); }
            }
        };
        const int fetching = max(0, total - (kRing - 1));
#pragma unroll 2
        for (int k = 0; k < fetching; ++k) term(fetch);
#pragma unroll 1
        for (int k = fetching; k < total; ++k) term([] { cp_async_commit(); });
#pragma unroll
        for (int i = 0; i < MM; ++i)
#pragma unroll
            for (int t = 0; t < T; ++t)
                if (p + i < pn && t < tn) {
                    u64 *z = o + ((size_t)(p + i) * el.out_tiles + t) * 2 * poly;
                    if constexpr (FP) { z[0] = s[i][t][0].finish(m.q_inv_f, qd); z[poly] = s[i][t][1].finish(m.q_inv_f, qd); }
                    else { z[0] = s[i][t][0].finish(m); z[poly] = s[i][t][1].finish(m); }
                }
    };
    if (m.fp) body(std::integral_constant<int, M>{}, 0, FpAcc{});
    else
        for (int p = 0; p < pn; ++p) { // the accumulators of one position fill the registers
            body(std::integral_constant<int, 1>{}, p, PieceAcc{});
        }
}

} // namespace hb
