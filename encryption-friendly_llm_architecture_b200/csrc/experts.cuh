// Ciphertext x plaintext products grouped by expert (sm_100a).
//
//     out[p][t] = sum_b sum_k pre[k][order[p]][b] (.) perm_{g_k}(w[e][t][b]),   e = the expert whose group position p lies in
// with groups of any size: what k_matmul_acc does, for several inputs that share weights.  A lane has one residue of both polynomials of M positions and of T
// output tiles: 2 M + T words a product step for 2 M T products.  The words come through a ring of stages in shared memory that belongs to the warp alone, by
// 16-byte asynchronous copies a few steps ahead: lines of 32 residues, of rotated weights the line that holds the residues wanted (a rotation permutes aligned
// runs of 32 as units, and within them), from which every lane reads its own.  The blocks of one range of residues, over all experts, run side by side, so that
// copies and weights come from L2 for all but the first of them.
// Two of three experts, twelve tiles, two K-groups of 128 copies, 8 positions at level 5: 9.9 ms (1.1 of HBM, 5.2 of FP64 at four instructions a product, nine modulo the 60-bit prime); five positions, one
// K-group, six tiles: 1.83 ms.  FP64 is 60 % active and 67 % of the issue slots are taken: a product costs 12.7 instructions, 5.7 of them FP64 (the 60-bit limb's nine
// and the conversions in it), 1.7 moves, the rest addresses and copies, and 168 registers leave three warps a scheduler.  Rings of 2, 3, 4 and 6 stages, in one run: 16.4, 10.4, 9.6 and 10.7 ms.  Sums that
// are kept as a double and modulo 2^64 (one FP64 instruction, three integer ones) for all, half or a third of the tiles: 13.2, 11.9 and 11.4 ms.
#pragma once
#include "pieces.cuh"

namespace hb {

// What one launch works on: experts with their positions and their weights' addresses.  An argument, so that calls can be recorded and nothing is uploaded.
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
// CTAs of four warps that an SM holds.  Blocks of nine to twelve sums a polynomial keep some words outside the registers with three CTAs; with two they do not and are slower (eight positions
// at two of three experts, twelve tiles 9.9 / 9.6 ms, five at four, six tiles 1.95 / 1.77).
template <int M, int T> constexpr int kExpertCtas = M * T > 3 ? 3 : 4;
constexpr int kExpertRing = 4;
template <int M, int T> constexpr size_t expert_smem() { return (size_t)4 * kExpertRing * (2 * M + T) * 256; }
// pre [copies][inputs][bcount][2][n][N].  Four warps side by side, 32 residues each.  grid = (N / 128 * blocks, n)
template <int M, int T>
__global__ void __launch_bounds__(128, kExpertCtas<M, T>) k_matmul_experts(u64 *out, const __grid_constant__ ExpertList el, const u64 *__restrict__ pre, int copies, int inputs, const u32 *__restrict__ gal,
                                                                           int n, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, int logn, int N) {
    extern __shared__ __align__(16) u64 words[];
    __shared__ const u64 *weights[T * 16];
    constexpr int S = kExpertRing;
    const int blocks = el.first_block[el.experts], blk = blockIdx.x % blocks, l = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int e = 0;
    while (blk >= el.first_block[e + 1]) ++e;
    const int tile_blocks = (el.tiles + T - 1) / T, in_e = blk - el.first_block[e];
    const int t0 = in_e % tile_blocks * T, p0 = el.first_pos[e] + in_e / tile_blocks * M, pn = min(M, el.first_pos[e + 1] - p0), tn = min(T, el.tiles - t0);
    const PrimeConst m = pc[map.prime[l]];
    const size_t poly = (size_t)n * N, limb = (size_t)l * N;
    const u32 x0 = blockIdx.x / blocks * 128 + warp * 32, x = x0 + lane;
    u64 *const ring = words + warp * (S * (2 * M + T) * 32);
    const int bcount = el.bcount, total = copies * bcount;
    u64 *const o = out + ((size_t)(el.pos0 + p0) * el.out_tiles + el.tile0 + t0) * 2 * poly + limb + x;
    const int half = lane >> 4, part = (lane & 15) * 2; // a lane copies two residues of one of two lines
    if (threadIdx.x < T * bcount) weights[threadIdx.x] = el.w[(e * el.tiles + min(t0 + (int)threadIdx.x / bcount, el.tiles - 1)) * bcount + threadIdx.x % bcount] + limb; // [tile][K-group]
    __syncthreads();

    // Positions p .. p + MM - 1 and tiles q .. q + TT - 1 of the block; tiles past the end: the last one again, not stored.  The products of a sum: all copies of one
    // K-group, then the next.
    auto body = [&](auto mm, auto tt, int p, int q, auto kind) {
        constexpr int MM = decltype(mm)::value, TT = decltype(tt)::value, kStage = (2 * MM + TT) * 32, kLoads = (TT + 1) / 2;
        using Sums = decltype(kind);
        const u64 *from[MM], *w[kLoads]; // both polynomials of a position and two tiles: one copy each
        auto weights_of = [&](int b) {
#pragma unroll
            for (int t = 0; t < kLoads; ++t) w[t] = weights[min(q + 2 * t + half, T - 1) * bcount + b] + part;
        };
#pragma unroll
        for (int i = 0; i < MM; ++i) from[i] = pre + ((size_t)el.input[p0 + p + i] * bcount * 2 + half) * poly + limb + x0 + part;
        weights_of(0);
        const i64 to_next = (i64)inputs * bcount * 2 * poly, to_group = (i64)2 * poly - (copies - 1) * to_next;
        const u32 ring_at = smem_u32(ring) + lane * 16, ex0 = 2 * (__brev(x0) >> (32 - logn)) + 1, ex = 2 * (__brev(x) >> (32 - logn)) + 1, mask = (2u << logn) - 1;
        auto turned = [&](u32 exponent, u32 g) { return __brev((g * exponent & mask) >> 1) >> (32 - logn); }; // ntt_perm of the residue with that exponent
        int fk = 0, fb = 0, rk = 0;
        u32 f_g = __ldg(gal), r_g = f_g; // of the copy that is fetched next, and of the one whose products come next
        auto fetch = [&](int stage) {
            const u32 to = ring_at + stage * (kStage * 8), line = turned(ex0, f_g) & ~31u;
            const bool last = ++fk == copies;
            if (last) fk = 0;
            f_g = __ldg(gal + fk);
#pragma unroll
            for (int i = 0; i < MM; ++i) { cp_async16(to + i * 512, from[i]); from[i] += last ? to_group : to_next; }
#pragma unroll
            for (int t = 0; t < kLoads; ++t)
                if (2 * t + 1 < TT || !half) cp_async16(to + MM * 512 + t * 512, w[t] + line);
            if (last && ++fb < bcount) weights_of(fb);
        };
        __syncwarp(); // the ring may still be read from a body before
#pragma unroll
        for (int k = 0; k < S - 1; ++k) {
            if (k < total) fetch(k);
            cp_async_commit();
        }
        Sums s[MM][TT][2];
        auto each = [&](auto &&f) { // every sum, with its position, tile and polynomial
#pragma unroll
            for (int i = 0; i < MM; ++i)
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int k = 0; k < 2; ++k) f(s[i][t][k], i, t, k);
        };
        each([](Sums &sum, int, int, int) { sum.zero(); });
        int left = total - (S - 1); // steps that are still to be fetched
        auto step = [&](int stage) { // always a constant
            cp_async_wait<S - 2>();
            __syncwarp();
            const u64 *at = ring + stage * kStage;
            const u32 place = turned(ex, r_g) & 31u; // of this lane's residue in a line of weights
            u64 v[MM][2], wv[TT];
#pragma unroll
            for (int t = 0; t < TT; ++t) wv[t] = at[MM * 64 + t * 32 + place];
#pragma unroll
            for (int i = 0; i < MM; ++i) { v[i][0] = at[i * 64 + lane]; v[i][1] = at[i * 64 + 32 + lane]; }
            if (left-- > 0) fetch((stage + S - 1) % S); // into the stage of a step ago
            cp_async_commit();
            if (++rk == copies) rk = 0;
            r_g = __ldg(gal + rk);
            typename Sums::Factor f[MM][2];
#pragma unroll
            for (int i = 0; i < MM; ++i) { f[i][0] = Sums::factor(v[i][0]); f[i][1] = Sums::factor(v[i][1]); }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                const typename Sums::Factor fw = Sums::factor(wv[t]);
#pragma unroll
                for (int i = 0; i < MM; ++i) { s[i][t][0].mac(f[i][0], fw); s[i][t][1].mac(f[i][1], fw); }
            }
        };
        const int room = Sums::room(m);
        auto relax = [&](int done) { if (done && done % room == 0) each([&](Sums &sum, int, int, int) { sum.relax(m); }); };
        int done = 0;
#pragma unroll 1
        for (; done + S <= total; done += S) { // as many steps as stages: the stages are constants, and FP64 sums may change registers
            relax(done);
#pragma unroll
            for (int k = 0; k < S; ++k) step(k);
        }
        if (done < total) relax(done);
#pragma unroll
        for (int k = 0; k < S - 1; ++k) if (done + k < total) step(k);
        each([&](Sums &sum, int i, int t, int k) {
            if (q + t < tn) o[((size_t)(p + i) * el.out_tiles + q + t) * 2 * poly + k * poly] = sum.finish(m);
        });
    };
    // as many positions as there are; modulo long primes, whose sums take more registers, one position and at most four tiles at a time
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, (M > 1 ? 2 : 1)> two{};
    if (m.fp) {
        constexpr std::integral_constant<int, T> all{};
        if (pn == M) body(std::integral_constant<int, M>{}, all, 0, 0, WholeSums{});
        else if (M > 2 && pn == 2) body(two, all, 0, 0, WholeSums{});
        else body(one, all, 0, 0, WholeSums{});
    } else {
        constexpr int TT = T > 4 ? T / 2 : T;
        constexpr std::integral_constant<int, TT> some{};
        for (int q = 0; q < T; q += TT)
            for (int p = 0; p < pn; ++p) body(one, some, p, q, PieceSums{});
    }
}

} // namespace hb
