// Sums of squares, products with one factor and gradients of a layer norm on ciphertexts (sm_100a).
//
// Members x[t][b] (t column tiles, outermost; b token tiles) are polynomial pairs (x0, x1); (x) is the tensor product (x0 y0, x0 y1 + x1 y0, x1 y1).  At every residue
//   squares      out[b]    = sum_t (x[t][b] - m[b])^2 - pad m[b]^2
//   scale        out[t][b] = (x[t][b] - m[b]) (x) r[b]
//   affine       out[t][b] = x[t][b] g[t] + K (beta[t], 0)
//   grad sums    rows[b] = sum_t g[t][b] (x) xhat[t][b], cols[t] = sum_b dy[t][b] (x) xhat[t][b], and the plain sums of g and dy over the same indices
//   grad input   out[t][b] = K (g[t][b] - m[b]) - xhat[t][b] (x) a[b]
// Sums are exact until one reduction at their end (FpAcc, PieceAcc).
#pragma once
#include "kernels.cuh"

namespace hb {

// Residues as the sums of one kind of prime take them.
struct FpField { // primes below 2^44: whole numbers in doubles, differences with their sign
    using Value = double;
    using Sum = FpAcc;
    const PrimeConst &m;
    __device__ __forceinline__ explicit FpField(const PrimeConst &m_) : m(m_) {}
    __device__ __forceinline__ double value(u64 x) const { return u52_to_double(x); }
    __device__ __forceinline__ double minus(double a, double b) const { return a - b; }
    __device__ __forceinline__ double negative(double a) const { return -a; }
    __device__ __forceinline__ int room() const { return m.q < (1ull << 42) ? 128 : 8; } // products of a sum before it is reduced
};
struct PieceField { // 45 to 60 bits
    using Value = u64;
    using Sum = PieceAcc;
    const PrimeConst &m;
    __device__ __forceinline__ explicit PieceField(const PrimeConst &m_) : m(m_) {}
    __device__ __forceinline__ u64 value(u64 x) const { return x; }
    __device__ __forceinline__ u64 minus(u64 a, u64 b) const { return sub_mod(a, b, m.q); }
    __device__ __forceinline__ u64 negative(u64 a) const { return m.q - a; } // up to q: products stay below 2^120
    __device__ __forceinline__ int room() const { return 8; }
};
template <class F> __device__ __forceinline__ void by_prime(const PrimeConst &m, F &&f) {
    if (m.fp) f(FpField(m)); else f(PieceField(m));
}
__device__ __forceinline__ u64 twice_mod(u64 a, u64 q) { return add_mod(a, a, q); }

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

// out[b] (+)= the sum over t < groups.  grid = N / 256 * batch * n, the residues of a limb side by side
template <class MEMBERS, bool MEAN>
__global__ void __launch_bounds__(256) k_square_sums(u64 *out, const __grid_constant__ MEMBERS x, const u64 *mean, int groups, int batch, u64 pad, int n, const PrimeConst *__restrict__ pc, int N, int accumulate) {
    const u32 px = N / 256, row = blockIdx.x / px;
    const int b = (int)row / n, l = (int)row % n;
    const u32 i = blockIdx.x % px * 256 + threadIdx.x;
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + i;
    pdl_wait();
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        typename decltype(f)::Sum s[3];
        for (auto &k : s) k.zero();
        V m0{}, m1{};
        if (MEAN) { m0 = f.value(mean[b * 2 * poly + at]); m1 = f.value(mean[(b * 2 + 1) * poly + at]); }
        for (int t = 0; t < groups; ++t) {
            if (t && t % f.room() == 0) for (auto &k : s) k.relax(m);
            const u64 *p = x.at(t * batch + b) + at;
            V v0 = f.value(p[0]), v1 = f.value(p[poly]);
            if (MEAN) { v0 = f.minus(v0, m0); v1 = f.minus(v1, m1); }
            s[0].mac(v0, v0); s[1].mac(v0, v1); s[2].mac(v1, v1);
        }
        u64 r[3] = {s[0].canonical(m), s[1].canonical(m), s[2].canonical(m)};
        if (MEAN && pad) {
            for (auto &k : s) k.zero();
            s[0].mac(m0, m0); s[1].mac(m0, m1); s[2].mac(m1, m1);
            for (int k = 0; k < 3; ++k) r[k] = sub_mod(r[k], mul_mod_any(s[k].canonical(m), pad, m), m.q);
        }
        r[1] = twice_mod(r[1], m.q);
        u64 *o = out + (size_t)b * 3 * poly + at;
        for (int k = 0; k < 3; ++k) o[k * poly] = accumulate ? add_mod(r[k], o[k * poly], m.q) : r[k];
    });
}
// out[i] = (x[i] - mean[i % batch]) (x) r[i % factors].  grid = N / 256 * members * n
template <class MEMBERS, class OUT, bool MEAN>
__global__ void __launch_bounds__(256) k_scale_members(const __grid_constant__ OUT out, const __grid_constant__ MEMBERS x, const u64 *mean, const u64 *r, int batch, int factors, int n, const PrimeConst *__restrict__ pc, int N) {
    const u32 px = N / 256, row = blockIdx.x / px;
    const int k = (int)row / n, l = (int)row % n;
    const u32 i = blockIdx.x % px * 256 + threadIdx.x;
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + i;
    pdl_wait();
    by_prime(m, [&](auto f) {
        using V = typename decltype(f)::Value;
        const u64 *p = x.at(k) + at, *rp = r + (size_t)(k % factors) * 2 * poly + at;
        V v0 = f.value(p[0]), v1 = f.value(p[poly]);
        const V r0 = f.value(rp[0]), r1 = f.value(rp[poly]);
        if (MEAN) {
            const u64 *mp = mean + (size_t)(k % batch) * 2 * poly + at;
            v0 = f.minus(v0, f.value(mp[0])); v1 = f.minus(v1, f.value(mp[poly]));
        }
        typename decltype(f)::Sum s[3];
        for (auto &e : s) e.zero();
        s[0].mac(v0, r0); s[1].mac(v0, r1); s[1].mac(v1, r0); s[2].mac(v1, r1);
        u64 *o = out.at(k) + at;
        for (int e = 0; e < 3; ++e) o[e * poly] = s[e].canonical(m);
    });
}
// Plaintexts of the column tiles.
constexpr int kNormTiles = 128; // of a launch
struct AffineList { const u64 *gamma[kNormTiles], *beta[kNormTiles]; int tile0, batch; };
// members of the tiles tile0 ..: out = x gamma + K beta on the first polynomial, x gamma on the second; without gammas x + beta.  grid = N / 256 * members * n
__global__ void __launch_bounds__(256) k_affine(u64 *out, const u64 *x, const __grid_constant__ AffineList a, const __grid_constant__ Scalars K, int n, const PrimeConst *__restrict__ pc, int N) {
    const u32 px = N / 256, row = blockIdx.x / px;
    const int k = (int)row / n, l = (int)row % n, t = k / a.batch;
    const u32 i = blockIdx.x % px * 256 + threadIdx.x;
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + i;
    pdl_wait();
    by_prime(m, [&](auto f) {
        const u64 *p = x + (size_t)(a.tile0 * a.batch + k) * 2 * poly + at;
        u64 *o = out + (size_t)(a.tile0 * a.batch + k) * 2 * poly + at;
        if (!a.gamma[t]) {
            o[0] = a.beta[t] ? add_mod(p[0], a.beta[t][at], m.q) : p[0];
            o[poly] = p[poly];
            return;
        }
        const auto g = f.value(a.gamma[t][at]);
        typename decltype(f)::Sum s[2];
        for (auto &e : s) e.zero();
        s[0].mac(f.value(p[0]), g); s[1].mac(f.value(p[poly]), g);
        if (a.beta[t]) s[0].mac(f.value(a.beta[t][at]), f.value(K.v[l]));
        o[0] = s[0].canonical(m); o[poly] = s[1].canonical(m);
    });
}
// Sums over one index: out[j] = sum_i y(i, j) (x) xhat(i, j) and sum[j] = sum_i y(i, j), member(i, j) = i * by_i + j * by_j.  grid = N / 256 * results * n
__global__ void __launch_bounds__(256) k_grad_sums_one(u64 *out, u64 *sum, const u64 *y, const u64 *xhat, int terms, int by_i, int by_j, int n, const PrimeConst *__restrict__ pc, int N) {
    const u32 px = N / 256, row = blockIdx.x / px;
    const int j = (int)row / n, l = (int)row % n;
    const u32 i = blockIdx.x % px * 256 + threadIdx.x;
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + i;
    pdl_wait();
    by_prime(m, [&](auto f) {
        typename decltype(f)::Sum s[3];
        for (auto &e : s) e.zero();
        u64 p0 = 0, p1 = 0;
        for (int e = 0; e < terms; ++e) {
            if (e && e % (f.room() / 2) == 0) for (auto &k : s) k.relax(m);
            const size_t from = ((size_t)e * by_i + (size_t)j * by_j) * 2 * poly + at;
            p0 = add_mod(p0, y[from], m.q); p1 = add_mod(p1, y[from + poly], m.q);
            const auto y0 = f.value(y[from]), y1 = f.value(y[from + poly]), x0 = f.value(xhat[from]), x1 = f.value(xhat[from + poly]);
            s[0].mac(y0, x0); s[1].mac(y0, x1); s[1].mac(y1, x0); s[2].mac(y1, x1);
        }
        u64 *o = out + (size_t)j * 3 * poly + at;
        for (int e = 0; e < 3; ++e) o[e * poly] = s[e].canonical(m);
        sum[(size_t)j * 2 * poly + at] = p0; sum[((size_t)j * 2 + 1) * poly + at] = p1;
    });
}
// grid = N / 256 * members * n
__global__ void __launch_bounds__(256) k_grad_input(u64 *out, const u64 *g, const u64 *mean, const u64 *xhat, const u64 *dot, int batch, const __grid_constant__ Scalars K, int n, const PrimeConst *__restrict__ pc, int N) {
    const u32 px = N / 256, row = blockIdx.x / px;
    const int k = (int)row / n, l = (int)row % n, b = k % batch;
    const u32 i = blockIdx.x % px * 256 + threadIdx.x;
    const PrimeConst m = pc[l];
    const size_t poly = (size_t)n * N, at = (size_t)l * N + i, from = (size_t)k * 2 * poly + at, of = (size_t)b * 2 * poly + at;
    pdl_wait();
    by_prime(m, [&](auto f) {
        const auto d0 = f.minus(f.value(g[from]), f.value(mean[of])), d1 = f.minus(f.value(g[from + poly]), f.value(mean[of + poly])), kl = f.value(K.v[l]);
        const auto x0 = f.negative(f.value(xhat[from])), x1 = f.negative(f.value(xhat[from + poly])), a0 = f.value(dot[of]), a1 = f.value(dot[of + poly]);
        typename decltype(f)::Sum s[3];
        for (auto &e : s) e.zero();
        s[0].mac(d0, kl); s[0].mac(x0, a0);
        s[1].mac(d1, kl); s[1].mac(x0, a1); s[1].mac(x1, a0);
        s[2].mac(x1, a1);
        u64 *o = out + (size_t)k * 3 * poly + at;
        for (int e = 0; e < 3; ++e) o[e * poly] = s[e].canonical(m);
    });
}

} // namespace hb
