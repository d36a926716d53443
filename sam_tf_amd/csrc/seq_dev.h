// What the sequence-policy kernels share (distill.hip, block_norm.hip, linattn.hip): element types, 16-byte pieces of a
// row at any alignment, sums over a row's threads.
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <math.h>
#include <atomic>
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

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// two values rounded to 16 bits each, the first in the low half
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<bf16>(float a, float b) {
    const bf16x2 v = __builtin_convertvector((f32x2){a, b}, bf16x2);
    uint32_t r;
    __builtin_memcpy(&r, &v, 4);
    return r;
}
template <> __device__ __forceinline__ uint32_t pack2<f16>(float a, float b) {
    const f16x2 v = __builtin_convertvector((f32x2){a, b}, f16x2);
    uint32_t r;
    __builtin_memcpy(&r, &v, 4);
    return r;
}

// 16 bytes of a row, packed as they lie there.  gfx950 loads and stores them at any address, so a piece starts at a
// multiple of kN elements of its row whatever the row's own alignment is.
template <typename T>
struct Piece {
    static constexpr int kN = 16 / (int)sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ uint32_t bits(int j) const {
        if constexpr (sizeof(T) == 4) return w[j];
        else return j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu;
    }
    __device__ __forceinline__ float f(int j) const;
};
template <> __device__ __forceinline__ float Piece<float>::f(int j) const { return __uint_as_float(w[j]); }
template <> __device__ __forceinline__ float Piece<bf16>::f(int j) const {
    return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
}
template <> __device__ __forceinline__ float Piece<f16>::f(int j) const {
    const uint16_t u = (uint16_t)bits(j);
    _Float16 h;
    __builtin_memcpy(&h, &u, 2);
    return (float)h;
}
struct Raw16 { uint32_t w[4]; } __attribute__((packed, aligned(2)));

// kN values, each rounded once (two of 16 bits by one instruction)
template <typename T>
__device__ __forceinline__ Piece<T> pack(const float* v) {
    Piece<T> p;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) p.w[j] = __float_as_uint(v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) p.w[j] = pack2<T>(v[2 * j], v[2 * j + 1]);
    }
    return p;
}

template <typename T> __device__ __forceinline__ uint32_t element_bits(const T* p) {
    if constexpr (sizeof(T) == 4) return *reinterpret_cast<const uint32_t*>(p);
    else return *reinterpret_cast<const uint16_t*>(p);
}

// elements [at, at + kN) of a row of n; where there are none the element whose bits are `fill`
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int64_t at, int64_t n, uint32_t fill) {
    Piece<T> p;
    if (at + Piece<T>::kN <= n) {
        const Raw16 r = *reinterpret_cast<const Raw16*>(row + at);
        __builtin_memcpy(&p, &r, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (sizeof(T) == 4) {
                p.w[j] = at + j < n ? element_bits(row + at + j) : fill;
            } else {
                const int64_t i = at + 2 * j;
                p.w[j] = (i < n ? element_bits(row + i) : fill) | (i + 1 < n ? element_bits(row + i + 1) : fill) << 16;
            }
        }
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
            if (at + j < n) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(row + at + j) = p.w[j];
                else *reinterpret_cast<uint16_t*>(row + at + j) = (uint16_t)p.bits(j);
            }
    }
}

// The compiler is not to keep what it has computed from the pieces so far: they are unpacked again where they are used
// next, which costs an instruction a value instead of a register.
template <typename T, int N>
__device__ __forceinline__ void forget(Piece<T> (&p)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(p[i].w[j]));
}

// minus infinity of a type
template <typename T> constexpr uint32_t kNegInf = sizeof(T) == 4 ? 0xff800000u : 0xff80u;
template <> inline constexpr uint32_t kNegInf<f16> = 0xfc00u;

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
// sh: two halves of `half` values (at least C for each wave of the workgroup; the same for all calls that share sh, whatever
// their C), used by turns (`turn` alternates between calls), so that one barrier is enough: a wave writes a half again only
// behind the next call's barrier, when all have read it.  Where a row has several waves
// every thread of the workgroup has to come here.
template <typename Op, int G, int C, typename V>
__device__ __forceinline__ void row_reduce(V (&v)[C], V* sh, int half, int& turn) {
    lane_reduce<Op, (G < 64 ? G : 64)>(v);
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6;
        V* mine = sh + (turn ? half : 0);
        turn ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int c = 0; c < C; ++c) mine[wave * C + c] = v[c];
        __syncthreads();
        constexpr int K = G / 64;
        const int first = wave / K * K;
        if constexpr (sizeof(V) == 4 && (C & (C - 1)) == 0 && K * C <= 64) {
            // one value a lane, reduced over the waves by lanes: the row's results come out of one register
            V t = mine[first * C + (threadIdx.x & (K * C - 1))];
#pragma unroll
            for (int o = C; o < K * C; o <<= 1) t = Op::f(t, __shfl_xor(t, o, 64));
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(t), c));
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                V t = mine[first * C + c];
#pragma unroll
                for (int w = 1; w < K; ++w) t = Op::f(t, mine[(first + w) * C + c]);
                v[c] = t;
            }
        }
    }
}

// units of the current device (asked once for each)
inline int cu_count() {
    static std::atomic<int> known[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

}  // namespace seq
}  // namespace samx
