// Plaintext operands from 4-bit weights with group scales (sm_100a).
//
// A weight is (code - 8) * scale: a whole number below 16 times a 24-bit significand, exact in a double, and so is its half.  The slots of a plaintext hold
// four tiles of d rows of one column tile, 1/2 (W1 - i W3) | 1/2 (W2 - i W4); `diagonal`: column j rolled up by j, as the shifted copies meet it.
#pragma once
#include "embed.cuh"

namespace hb {

// codes [ceil(rows / 2)][cols], the even row in the low half of a byte; scales [ceil(rows / group)][cols]
struct Weights4 { const unsigned char *codes; const float *scales; int rows, cols, group; };
// the weight at (r, c), halved; zero outside
__device__ __forceinline__ double half_weight(const Weights4 &w, int r, int c) {
    if (r >= w.rows || c >= w.cols) return 0.0;
    const int byte = __ldg(w.codes + (size_t)(r >> 1) * w.cols + c), code = r & 1 ? byte >> 4 : byte & 15;
    return (double)(code - 8) * (0.5 * (double)__ldg(w.scales + (size_t)(r / w.group) * w.cols + c));
}
struct Blocks4 { int first, kb, d, diagonal; }; // block number first + y is K-group (.) % kb of column tile (.) / kb
// the value of slot i of a block
__device__ __forceinline__ double2 slot_weight(const Weights4 &w, const Blocks4 &b, int block, int i) {
    const int d = b.d, r = i / (2 * d);
    if (r >= d) return make_double2(0.0, 0.0);
    const int c2 = i - r * 2 * d, half = c2 >= d, c = half ? c2 - d : c2;
    int from = r;
    if (b.diagonal) { from += c; if (from >= d) from -= d; }
    const int row = (block % b.kb * 4 + half) * d + from, col = block / b.kb * d + c;
    const double im = half_weight(w, row + 2 * d, col);
    return make_double2(half_weight(w, row, col), im == 0.0 ? 0.0 : -im);
}
// slots re, im [count][slots].  grid = (slots / 256, count)
__global__ void __launch_bounds__(256) k_weight_slots(double *re, double *im, Weights4 w, Blocks4 b, int slots) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    pdl_wait();
    if (i >= slots) return;
    const double2 v = slot_weight(w, b, b.first + (int)blockIdx.y, i);
    re[(size_t)blockIdx.y * slots + i] = v.x; im[(size_t)blockIdx.y * slots + i] = v.y;
}
// out[v][j] (+)= sum_b x[v][b] (.) p[j][b], one coefficient of both polynomials a thread: x [vectors][kb][2][n][N], p [columns][kb][n][N], out [vectors][nb][2][n][N] from column j0.
// grid = (N / 256, n, vectors * columns)
__global__ void __launch_bounds__(256) k_matvec(u64 *out, const u64 *x, const u64 *p, int kb, int columns, int nb, int j0, int n, const __grid_constant__ LimbMap map, const PrimeConst *__restrict__ pc, int N) {
    const int l = blockIdx.y, v = blockIdx.z / columns, j = blockIdx.z % columns;
    const PrimeConst m = pc[map.prime[l]];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + blockIdx.x * 256 + threadIdx.x;
    const u64 *xp = x + (size_t)v * kb * 2 * poly + at, *pp = p + (size_t)j * kb * poly + at;
    u64 *o = out + ((size_t)v * nb + j0 + j) * 2 * poly + at;
    pdl_wait();
    auto sum = [&](auto s0, int room) {
        auto s1 = s0;
        s0.zero(); s1.zero();
        for (int b = 0; b < kb; ++b, xp += 2 * poly, pp += poly) {
            if (b && b % room == 0) { s0.relax(m); s1.relax(m); }
            s0.product(xp[0], pp[0]); s1.product(xp[poly], pp[0]);
        }
        o[0] = s0.canonical(m); o[poly] = s1.canonical(m);
    };
    if (m.fp) sum(FpAcc{}, m.q < (1ull << 42) ? 128 : 8);
    else sum(PieceAcc{}, 8);
}

} // namespace hb
