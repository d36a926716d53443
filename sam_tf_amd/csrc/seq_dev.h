// What the sequence-policy kernels share (distill.hip, block_norm.hip, linattn.hip): element types, 16-byte pieces of a
// row at any alignment, sums over a row's threads.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include "samx_common.h"

namespace samx {
namespace seq {

// SAMX_F32 / SAMX_BF16 / SAMX_F16 of samx.h
enum Dtype { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct bf16 { uint16_t v; };
struct f16 { _Float16 v; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(bf16 x) { return __uint_as_float((uint32_t)x.v << 16); }
__device__ __forceinline__ float to_float(f16 x) { return (float)x.v; }

template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
// round to nearest, ties to even (the compiler's conversion instruction); a NaN stays one
template <> __device__ __forceinline__ bf16 from_float<bf16>(float x) {
    const __bf16 b = (__bf16)x;
    bf16 r;
    __builtin_memcpy(&r, &b, 2);
    return r;
}
template <> __device__ __forceinline__ f16 from_float<f16>(float x) { f16 r; r.v = (_Float16)x; return r; }

// 16 bytes of a row.  gfx950 loads and stores them at any address, so a piece starts at a multiple of kN elements of
// its row whatever the row's own alignment is.
template <typename T> struct Piece { static constexpr int kN = 16 / (int)sizeof(T); T e[kN]; };
struct Raw16 { uint32_t w[4]; } __attribute__((packed, aligned(2)));

// elements [at, at + kN) of a row of n, `fill` where there are none
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int64_t at, int64_t n, T fill) {
    Piece<T> p;
    if (at + Piece<T>::kN <= n) {
        const Raw16 r = *reinterpret_cast<const Raw16*>(row + at);
        __builtin_memcpy(&p, &r, 16);
    } else {
#pragma unroll
        for (int j = 0; j < Piece<T>::kN; ++j) p.e[j] = at + j < n ? row[at + j] : fill;
    }
    return p;
}

template <typename T>
__device__ __forceinline__ void store_piece(T* row, int64_t at, int64_t n, const Piece<T>& p) {
    if (at + Piece<T>::kN <= n) {
        Raw16 r;
        __builtin_memcpy(&r, &p, 16);
        *reinterpret_cast<Raw16*>(row + at) = r;
    } else {
#pragma unroll
        for (int j = 0; j < Piece<T>::kN; ++j)
            if (at + j < n) row[at + j] = p.e[j];
    }
}

struct OpSum { template <typename V> static __device__ __forceinline__ V f(V a, V b) { return a + b; } };
struct OpMax { template <typename V> static __device__ __forceinline__ V f(V a, V b) { return a > b ? a : b; } };

// All C values reduced over every group of L lanes (a power of two), the same result in each lane (a fixed tree).
template <typename Op, int L, int C, typename V>
__device__ __forceinline__ void lane_reduce(V (&v)[C]) {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1)
#pragma unroll
        for (int c = 0; c < C; ++c) v[c] = Op::f(v[c], __shfl_xor(v[c], o, 64));
}

// The same over the G threads of a row (G a power of two; the waves of a row lie side by side in the workgroup).
// sh: [2][waves of the workgroup][C], used by turns (`turn` alternates between calls), so that one barrier is enough: a
// wave writes a half again only behind the next call's barrier, when all have read it.  Where a row has several waves
// every thread of the workgroup has to come here.
template <typename Op, int G, int C, typename V>
__device__ __forceinline__ void row_reduce(V (&v)[C], V* sh, int waves, int& turn) {
    lane_reduce<Op, (G < 64 ? G : 64)>(v);
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6;
        V* mine = sh + (turn ? waves * C : 0);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int c = 0; c < C; ++c) mine[wave * C + c] = v[c];
        __syncthreads();
        const int first = wave / (G / 64) * (G / 64);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            V t = mine[first * C + c];
#pragma unroll
            for (int w = 1; w < G / 64; ++w) t = Op::f(t, mine[(first + w) * C + c]);
            v[c] = t;
        }
    }
}

inline int cu_count() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
        return 256;
    return n > 0 ? n : 256;
}

}  // namespace seq
}  // namespace samx
