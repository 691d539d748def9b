// Exact sums of products of residues on the FP64 pipe (sm_100a), in two forms with the same names: WholeSums for primes below 2^44, PieceSums for those up to
// 2^60.
#pragma once
#include "kernels.cuh"
#include <type_traits>

namespace hb {

// A residue below 2^60 is three pieces of 20 bits, whole numbers as doubles.  Products of pieces with the same weight are added up by multiply-adds that are
// exact (128 products of residues stay below 2^49 in every sum): nine in place for a product of residues, and the five sums are put together and
// reduced at the end.  A launch of grouped products modulo such a prime, two positions and eight tiles of 128 copies: 326 us with half of the tiles by PieceAcc
// (30-bit pieces and 32-bit multiplications, reduced every eight products), 318 with all by this.
struct PieceSums {
    static constexpr int kBits = 20;
    struct Factor { double p[3]; };
    double s[5];
    static __device__ __forceinline__ int room(const PrimeConst &) { return 128; } // products before relax() or finish()
    static __device__ __forceinline__ Factor factor(u64 v) {
        constexpr u64 mask = (1ull << kBits) - 1;
        return {{u52_to_double(v & mask), u52_to_double(v >> kBits & mask), u52_to_double(v >> 2 * kBits)}};
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 5; ++i) s[i] = 0.0;
    }
    __device__ __forceinline__ void mac(const Factor &a, const Factor &b) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int j = 0; j < 3; ++j) s[i + j] = __fma_rn(a.p[i], b.p[j], s[i + j]);
    }
    __device__ __forceinline__ u64 finish(const PrimeConst &m) const { // canonical
        unsigned __int128 v = 0; // 128 products: below 2^127
#pragma unroll
        for (int i = 0; i < 5; ++i) v += (unsigned __int128)mantissa52(__dadd_rn(s[i], kTwo52)) << (kBits * i);
        return barrett128((u64)(v >> 64), (u64)v, m);
    }
    __device__ __forceinline__ void relax(const PrimeConst &m) { // makes room for as many products again (the first three sums take the pieces of what there is: 2^20 more)
        const Factor f = factor(finish(m));
        zero();
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] = f.p[i];
    }
};
// FpAcc by the same names
struct WholeSums {
    using Factor = double;
    FpAcc a;
    static __device__ __forceinline__ int room(const PrimeConst &m) { return m.q < (1ull << 42) ? 128 : 8; }
    static __device__ __forceinline__ Factor factor(u64 v) { return u52_to_double(v); }
    __device__ __forceinline__ void zero() { a.zero(); }
    __device__ __forceinline__ void mac(Factor x, Factor y) { a.mac(x, y); }
    __device__ __forceinline__ u64 finish(const PrimeConst &m) const { return a.canonical(m); }
    __device__ __forceinline__ void relax(const PrimeConst &m) { a.relax(m); }
};

} // namespace hb
