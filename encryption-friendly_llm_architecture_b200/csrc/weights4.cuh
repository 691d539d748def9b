// Plaintext operands from 4-bit weights with group scales (sm_100a).
//
// A weight is (code - 8) * scale: a whole number below 16 times a 24-bit significand, exact in a double, and so is its half.  The slots of a plaintext hold
// four tiles of d rows of one column tile, 1/2 (W1 - i W3) | 1/2 (W2 - i W4); `diagonal`: column j rolled up by j, as the shifted copies meet it.
#pragma once
#include "embed.cuh"
#include "ntt.cuh"

namespace hb {

// codes [ceil(rows / 2)][cols], the even row in the low half of a byte; scales [ceil(rows / group)][cols]
struct Weights4 { const unsigned char *codes; const float *scales; int rows, cols, group; };
// block number first + y is K-group (.) % kb of column tile (.) / kb.  Quotients by 2 d and by the group come from products: by_row = ceil(2^32 / 2d) is exact for slots
// below 2^15, by_group = ceil(2^32 / group) for rows of a block, counted from the start of a group; 0 where a group is at least as long as a block, so that a block meets two
struct Blocks4 { int first, kb, d, diagonal; u32 by_row; u64 by_group; };
// Rows and columns of one block.
struct Block4 {
    const Weights4 &w;
    const Blocks4 &b;
    int row0, col0, group0, rest; // its first row and column; the group that row lies in, and its place there
    __device__ __forceinline__ Block4(const Weights4 &w_, const Blocks4 &b_, int block) : w(w_), b(b_) {
        row0 = block % b.kb * 4 * b.d; col0 = block / b.kb * b.d;
        group0 = row0 / w.group; rest = row0 - group0 * w.group;
    }
    // the weight at row r and column c of the block, halved; zero outside the matrix, of which the last row and column are read instead, so that no load waits for a branch
    __device__ __forceinline__ double half(int r, int c) const {
        const bool there = r < w.rows - row0 && c < w.cols - col0;
        const int rr = min(r, w.rows - 1 - row0), cc = min(col0 + c, w.cols - 1), row = row0 + rr; // the block's first row and column are there
        const int byte = __ldg(w.codes + (size_t)(row >> 1) * w.cols + cc), code = row & 1 ? byte >> 4 : byte & 15;
        const u32 t = (u32)(rest + rr), group = (u32)group0 + (b.by_group ? (u32)(t * b.by_group >> 32) : t >= (u32)w.group);
        const float scale = __ldg(w.scales + (size_t)group * w.cols + cc);
        return there ? (double)(code - 8) * (0.5 * (double)scale) : 0.0;
    }
    __device__ __forceinline__ double2 slot(int i) const { // the value of slot i
        const int d = b.d, r = (int)__umulhi((u32)i, b.by_row), c2 = i - r * 2 * d, right = c2 >= d, c = right ? c2 - d : c2;
        int from = r;
        if (b.diagonal) { from += c; if (from >= d) from -= d; }
        if (r >= d) from = 4 * d; // past the tiles
        else from += right * d;
        const double re = half(from, c), im = half(from + 2 * d, c);
        return r < d ? make_double2(re, 0.0 - im) : make_double2(0.0, 0.0);
    }
};
// Where the members of a batch of plaintexts lie: one buffer each.
constexpr int kBlocks4 = 64; // blocks of a launch
struct PtList {
    u64 *p[kBlocks4];
    __device__ __forceinline__ u64 *at(int member, int limb, int N) const { return p[member] + (size_t)limb * N; }
    __device__ __forceinline__ size_t off(int li, int period) const { return (size_t)(at(li / period, li % period, kN16) - (u64 *)nullptr); } // from a null base: the address of ntt16.cuh
};
// ---- slots -> coefficients: k_embed_inv_cols and k_embed_inv_small with the slots made on the way ----
// half-transformed slots v [count][2^15].  12 blocks of 768 x 768: 14.5 us, one wave of CTAs whose time is the latency of codes and scales and of two rounds of butterflies (10 us
// of it, the time of the row pass); 36 blocks 36 us.  The slots written first and read again by the column pass: 366 us for 36 plaintexts at level 5, 226 with them made here and
// the reduction in the column pass below.  grid = (16, count)
__global__ void __launch_bounds__(kEmbThreads) k_weight_cols(double2 *v, const __grid_constant__ Weights4 w, const __grid_constant__ Blocks4 b, EmbedTables tb) {
    __shared__ double2 sm[kEmbRows * 8];
    const int lane = threadIdx.x & 7, sub = threadIdx.x >> 3, col = blockIdx.x * 8 + lane;
    const Block4 block(w, b, b.first + (int)blockIdx.y);
    double2 x[16];
    pdl_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = block.slot((e * 16 + sub) * kEmbCols + col);
    inv_round<8>(x, tb.inv, 16 * kEmbCols, sub * kEmbCols + col);
#pragma unroll
    for (int e = 0; e < 16; ++e) sm[(e * 16 + sub) * 8 + lane] = x[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = sm[(sub * 16 + e) * 8 + lane];
    inv_round<8>(x, tb.inv, kEmbCols, col);
    double2 *o = v + (size_t)blockIdx.y * kSlots16 + col;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[(sub * 16 + e) * kEmbCols] = x[e];
}
// rounded coefficients at scale sc, coef [count][2 slots].  grid = count
__global__ void __launch_bounds__(256) k_weight_small(i64 *coef, const __grid_constant__ Weights4 w, const __grid_constant__ Blocks4 b, int log_slots, double sc, EmbedTables tb) {
    __shared__ double2 sm[kEmbSmallMax];
    const int slots = 1 << log_slots;
    const Block4 block(w, b, b.first + (int)blockIdx.x);
    pdl_wait();
    for (int i = threadIdx.x; i < slots; i += 256) sm[i] = block.slot(i);
    for (int h = slots >> 1; h >= 1; h >>= 1) {
        __syncthreads();
        for (int t = threadIdx.x; t < slots / 2; t += 256) {
            const int j = t & (h - 1), a = (t - j) * 2 + j;
            inv_bfly(sm[a], sm[a + h], __ldg(tb.inv + h + j));
        }
    }
    __syncthreads();
    const double inv = 1.0 / (double)slots;
    i64 *o = coef + (size_t)blockIdx.x * 2 * slots;
    for (int i = threadIdx.x; i < slots; i += 256) {
        const double2 x = sm[__brev((u32)i) >> (32 - log_slots)];
        o[i] = to_i64(rint(__dmul_rn(__dmul_rn(x.x, inv), sc)));
        o[i + slots] = to_i64(rint(__dmul_rn(__dmul_rn(x.y, inv), sc)));
    }
}
// ---- coefficients -> residues in transform order ----
// The column pass of ntt16v2_fwd_cols on coefficients coef [count][2^16], reduced on the way: a pass over the residues of every limb less (64 limbs: 19 us, the pass and the
// reduction apart 15 and 17; 216 limbs of 36 members 52 us).  Bound by the FP64 instructions of the butterflies and the wait between its two rounds.  One test of the
// magnitudes of all sixteen coefficients stands before the reductions, which would wait for a branch each.  map names the primes of the limbs of a member.
// grid = (16, count * map.n)
template <class LONG>
__global__ void __launch_bounds__(256, 4) k_coef_cols(const __grid_constant__ PtList to, const i64 *coef, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, Ntt16Tables tb) {
    __shared__ u64 sm[4096];
    const int member = blockIdx.y / map.n, li = blockIdx.y % map.n, pi = map.prime[li];
    const PrimeConst m = pc[pi];
    const ulonglong2 *tab = tb.fwd + (size_t)pi * Ntt16Layout::kEntries;
    const int tid = threadIdx.x, lane = tid & 15, sub = tid >> 4;
    const i64 *p = coef + (size_t)member * kN16 + blockIdx.x * 16 + lane;
    u64 *o = to.at(member, li, kN16) + blockIdx.x * 16 + lane;
    i64 a[16];
    u64 large = 0; // the magnitudes' bits: as a rule the coefficients are far below 2^44
    pdl_wait();
#pragma unroll
    for (int e = 0; e < 16; ++e) a[e] = p[(e * 16 + sub) * 256];
#pragma unroll
    for (int e = 0; e < 16; ++e) large |= (u64)(a[e] ^ (a[e] >> 63));
    if (m.small) {
        const DsConst c = ds_const(m);
        double v[16];
        if (large >> 50)
            for (int e = 0; e < 16; ++e) v[e] = ds_load(reduce_i64(a[e], m));
        else
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = ds_reduce(__longlong_as_double(a[e] + 0x4338000000000000ll) - kMagicS, c); // 2^52 + 2^51 + a
        fwd16_ds(v, TwiddlesA(tab + Ntt16Layout::colsA(0)), c);
        double *smd = reinterpret_cast<double *>(sm);
#pragma unroll
        for (int e = 0; e < 16; ++e) smd[(e * 16 + sub) * 16 + lane] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = smd[(sub * 16 + e) * 16 + lane];
        fwd16_ds(v, TwiddlesA(tab + Ntt16Layout::colsB(sub, 0)), c);
        double *od = reinterpret_cast<double *>(o);
#pragma unroll
        for (int e = 0; e < 16; ++e) od[(sub * 16 + e) * 256] = v[e];
    } else {
        u64 v[16];
        if (large >> 44)
            for (int e = 0; e < 16; ++e) v[e] = reduce_i64(a[e], m);
        else
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = a[e] < 0 ? (u64)a[e] + m.q : (u64)a[e];
        const typename LONG::Const c = LONG::make(m);
        LONG::template fwd16<0>(v, TwiddlesA(tab + Ntt16Layout::colsA(0)), c);
#pragma unroll
        for (int e = 0; e < 16; ++e) sm[(e * 16 + sub) * 16 + lane] = v[e];
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = sm[(sub * 16 + e) * 16 + lane];
        LONG::template fwd16<1>(v, TwiddlesA(tab + Ntt16Layout::colsB(sub, 0)), c);
#pragma unroll
        for (int e = 0; e < 16; ++e) o[(sub * 16 + e) * 256] = v[e];
    }
}
// the whole transform of a small ring's limb: ntt_small on coefficients.  grid = (map.n, count)
__global__ void __launch_bounds__(256) k_coef_small(const __grid_constant__ PtList to, const i64 *coef, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, NttTables tb, int logn) {
    extern __shared__ u64 sm_dyn[];
    const int N = 1 << logn, pi = map.prime[blockIdx.x];
    const PrimeConst m = pc[pi];
    const u64 q = m.q, q2 = q << 1;
    const i64 *p = coef + (size_t)blockIdx.y * N;
    u64 *o = to.at(blockIdx.y, blockIdx.x, N);
    const u64 *w = tb.psi + (size_t)pi * N, *ws = tb.psi_sh + (size_t)pi * N;
    pdl_wait();
    for (int i = threadIdx.x; i < N; i += 256) sm_dyn[i] = reduce_i64_any(p[i], m);
    __syncthreads();
    for (int h = 1, t = N >> 1; h < N; h <<= 1, t >>= 1) {
        for (int k = threadIdx.x; k < N / 2; k += 256) {
            const int i = k / t, i0 = 2 * i * t + (k - i * t);
            ct_bfly(sm_dyn[i0], sm_dyn[i0 + t], w[h + i], ws[h + i], q, q2);
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < N; i += 256) {
        u64 x = sm_dyn[i];
        x = x >= q2 ? x - q2 : x;
        o[i] = x >= q ? x - q : x;
    }
}
// ---- products ----
// out[v][j] = sum_b x[v][b] (.) p[j][b]: x [vectors][kb][2][n][N], operands p [columns][kb][limbs][N] of the limbs l0 .. and the columns j0 .., out [vectors][nb][2][n][N].  A thread has one
// coefficient of both polynomials of V vectors and of C columns: 2 V + C words for 2 V C products, as many in flight.  The blocks of one
// range of coefficients run side by side.  Four vectors, 2048 x 2048, 4 K-groups: 36 us a limb, 68 MB of results and 17 MB of x in it (13 us of HBM, 18 with the operands), the rest the wait for
// the words of a K-group (FP64 36 % active).  The whole call in CTAs of 128 threads and two K-groups a turn against 256 threads and one: four vectors 479 -> 463 us, one 325 -> 298,
// one of 32 K-groups 736 -> 620; with the words of the next K-group in flight as well 505, 321 and 708, since the registers cost warps.
// Three vectors take the block of four (2048 x 2048, level 5: 437 us for three, 458 for four), five that of eight (608 and 674).  grid = (N / 128 * blocks, limbs)
struct MatvecShape { int vectors, kb, columns, nb, j0, n, l0; };
template <int V, int C>
__global__ void __launch_bounds__(128, V == 1 ? 5 : 3) k_matvec(u64 *out, const u64 *x, const u64 *p, MatvecShape s, const PrimeConst *__restrict__ pc, int N) {
    const int bv = (s.vectors + V - 1) / V, blocks = bv * ((s.columns + C - 1) / C), blk = blockIdx.x % blocks, v0 = blk % bv * V, c0 = blk / bv * C, l = s.l0 + blockIdx.y, limbs = gridDim.y;
    const PrimeConst m = pc[l];
    const u32 at = blockIdx.x / blocks * 128 + threadIdx.x;
    const size_t poly = (size_t)s.n * N, limb = (size_t)limbs * N;
    const u64 *xp[V], *pp[C];
#pragma unroll
    for (int i = 0; i < V; ++i) xp[i] = x + (size_t)min(v0 + i, s.vectors - 1) * s.kb * 2 * poly + (size_t)l * N + at; // past the end: the last one again, not stored
#pragma unroll
    for (int j = 0; j < C; ++j) pp[j] = p + (size_t)min(c0 + j, s.columns - 1) * s.kb * limb + (size_t)blockIdx.y * N + at;
    pdl_wait();
    auto sum = [&](auto kind, int room) {
        decltype(kind) a[V][C][2];
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) { a[i][j][0].zero(); a[i][j][1].zero(); }
        auto group = [&](int b) {
            u64 xv[V][2], pv[C];
#pragma unroll
            for (int i = 0; i < V; ++i) { xv[i][0] = xp[i][0]; xv[i][1] = xp[i][poly]; xp[i] += 2 * poly; }
#pragma unroll
            for (int j = 0; j < C; ++j) { pv[j] = pp[j][0]; pp[j] += limb; }
            if (b && b % room == 0) {
#pragma unroll
                for (int i = 0; i < V; ++i)
#pragma unroll
                    for (int j = 0; j < C; ++j) { a[i][j][0].relax(m); a[i][j][1].relax(m); }
            }
#pragma unroll
            for (int i = 0; i < V; ++i)
#pragma unroll
                for (int j = 0; j < C; ++j) { a[i][j][0].product(xv[i][0], pv[j]); a[i][j][1].product(xv[i][1], pv[j]); }
        };
        int b = 0;
#pragma unroll 1
        for (; b + 1 < s.kb; b += 2) { group(b); group(b + 1); } // FP64 sums change registers at every product
        if (b < s.kb) group(b);
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < C; ++j) {
                if (v0 + i >= s.vectors || c0 + j >= s.columns) continue;
                u64 *o = out + ((size_t)(v0 + i) * s.nb + s.j0 + c0 + j) * 2 * poly + (size_t)l * N + at;
                o[0] = a[i][j][0].canonical(m); o[poly] = a[i][j][1].canonical(m);
            }
    };
    if (m.fp) sum(FpAcc{}, m.q < (1ull << 42) ? 128 : 8);
    else sum(PieceAcc{}, 8);
}

} // namespace hb
