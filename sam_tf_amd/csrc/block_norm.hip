// The norm behind a block, its gate, the scaled residual and the norm in front of the next block, in one pass over the
// rows, and the gradient of all of it.
//
//   n = N(y; w1, b1) ;  h = r x + g n ;  u = N(h; w2, b2)          g: nothing, one value a channel, or one an element
//   N(y; w, b) = w (y - m) s + b,  s = 1 / sqrt(mean (y - m)^2 + eps),  m = mean y (LayerNorm) or 0 without b (RMS norm)
//
// Backward, from the gradients dh (of h, by the residual path) and du (of u):
//   k = w2 du ;  dh' = dh + s_h (k - hh mean(k hh) [- mean k]),  hh = (h - m_h) s_h
//   dx = r dh' ;  dg = dh' n ;  k' = w1 g dh' ;  dy = s_y (k' - yh mean(k' yh) [- mean k'])
//   dw2 = sum du hh, db2 = sum du, dw1 = sum g dh' yh, db1 = sum g dh', over the rows
//
// Bound: HBM.  A row stays in the registers of its threads (E elements each); the channels' parameters, and in the
// gradient their sums, stay there over all the rows that a workgroup takes (row b, b + grid, ...), and the next row's
// loads are in flight while this one is reduced.  Statistics and sums are float32 (two passes over the registers for a
// variance), every output is rounded once.  The channel sums are added in a fixed order: the rows of a workgroup one
// after the other, then the workgroups in column_kernel.  Measured, bf16, 16384 x 4096 (a large copy reaches 4750 GB/s):
// forward 120 us, 4470 GB/s; gradient with the RMS norm 182 us, 4400 GB/s, with LayerNorm 225 us, 3600 GB/s (its four sums
// leave a few registers spilt), with a full gate beside it 257 us, 4200 GB/s.
#include "seq_dev.h"
#include "../../include/samx.h"

namespace {

using namespace samx::seq;

typedef float f32x4 __attribute__((ext_vector_type(4)));

enum Gate { kNone = 0, kChannel = 1, kFull = 2 };

struct Args {
    const void *x, *y, *h, *dh, *du, *gate;
    const float *w1, *b1, *w2, *b2;
    void *o1, *o2, *og;          // h, u  or  dx, dy, dgate (kFull)
    float* part;                 // gradient: [grid][sums][D]
    int64_t N; int D;
    float res, eps;
};

// This thread's elements of a row: P pieces, piece p the kN elements from at[p] on.  The row's last piece starts kN before
// its end, however few of its elements are not its neighbour's: those come as zeros (keep), so that every load is a whole
// one.  Rows of less than a piece are read by elements.
template <typename T, int G, int P>
struct Cols {
    static constexpr int N = Piece<T>::kN, E = P * N;
    static constexpr int R = (G < 256 ? 256 : G) / G;   // rows of the workgroup
    int D, at[P], first[P];               // first: elements that are the neighbour's (kN: all, no piece)
    uint32_t slot;                        // which of the workgroup's rows (the same in a whole wave where it can be)
    uint32_t keep[P][4];
    __device__ explicit Cols(int D_) : D(D_) {
        const int lane = threadIdx.x % G;
        slot = threadIdx.x / G;
        if constexpr (G >= 64) slot = __builtin_amdgcn_readfirstlane(slot);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int want = (p * G + lane) * N, last = D >= N ? D - N : 0;
            at[p] = want < last ? want : last;
            first[p] = want >= D ? N : want - at[p];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) keep[p][j] = j >= first[p] ? ~0u : 0u;
                else keep[p][j] = (2 * j >= first[p] ? 0xffffu : 0u) | (2 * j + 1 >= first[p] ? 0xffff0000u : 0u);
            }
        }
    }
    // whether element i of the thread is its own
    __device__ __forceinline__ bool own(int i) const {
        return i % N >= first[i / N] && at[i / N] + i % N < D;
    }
    __device__ __forceinline__ void channels(const float* w, int p, float* out) const {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = own(p * N + j) ? w[at[p] + j] : 0.f;
    }
    // the same of a row of at least a piece, the neighbour's elements with it
    __device__ __forceinline__ void channels_all(const float* w, int p, float* out) const {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const Raw16 v = *reinterpret_cast<const Raw16*>((const char*)w + (uint32_t)(at[p] + j) * 4u);
#pragma unroll
            for (int u = 0; u < 4; ++u) out[j + u] = __uint_as_float(v.w[u]);
        }
    }
    __device__ __forceinline__ void channels(const float* w, float (&out)[E]) const {
#pragma unroll
        for (int p = 0; p < P; ++p) channels(w, p, out + p * N);
    }
    // The pieces of row first + slot as they stand in memory (some row's where there is none): nothing waits for them
    // here.  The address is the workgroup's first row, and a 32-bit distance from it for each thread.
    __device__ __forceinline__ void load(const void* base, int64_t first_row, int64_t rows, Piece<T> (&r)[P]) const {
        const char* x = (const char*)base + (first_row < rows ? first_row : 0) * (int64_t)D * (int)sizeof(T);
        const uint32_t mine = first_row + slot < rows ? slot * (uint32_t)D : 0u;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (D >= N) {
                const Raw16 v = *reinterpret_cast<const Raw16*>(x + (mine + (uint32_t)at[p]) * (uint32_t)sizeof(T));
                __builtin_memcpy(&r[p], &v, 16);
            } else {
                r[p] = load_piece((const T*)x + mine, 0, first[p] == 0 ? D : 0, 0u);
            }
        }
    }
    // what of them is the thread's own, the rest zeros
    __device__ __forceinline__ void take(const Piece<T> (&r)[P], bool live, Piece<T> (&c)[P]) const {
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < 4; ++j) c[p].w[j] = r[p].w[j] & (live ? keep[p][j] : 0u);
    }
    // piece p of a row from kN values
    __device__ __forceinline__ void store(void* base, int64_t first_row, int p, const float* v) const {
        char* b = (char*)base + first_row * (int64_t)D * (int)sizeof(T);
        T* x = (T*)(b + (slot * (uint32_t)D + (uint32_t)at[p]) * (uint32_t)sizeof(T));
        const Piece<T> o = pack<T>(v);
        if (first[p] == 0 && D >= N) {
            Raw16 r;
            __builtin_memcpy(&r, &o, 16);
            *reinterpret_cast<Raw16*>(x) = r;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (own(p * N + j)) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(x + j) = o.w[j];
                    else *reinterpret_cast<uint16_t*>(x + j) = (uint16_t)o.bits(j);
                }
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t first_row, const float (&v)[E]) const {
#pragma unroll
        for (int p = 0; p < P; ++p) store(base, first_row, p, v + p * N);
    }
};

template <typename T, int G, int P, bool LAYER, int GATE>
__global__ __launch_bounds__(G < 256 ? 256 : G) void forward_kernel(Args a) {
    constexpr int B = G < 256 ? 256 : G, W = B / 64, N = Piece<T>::kN, E = P * N, R = B / G;
    __shared__ float sh[2 * W];
    int turn = 0;
    const int D = a.D;
    const Cols<T, G, P> cols(D);
    const float inv = 1.f / (float)D;
    float w1[E], w2[E], b1[E], b2[E];
    cols.channels(a.w1, w1);
    cols.channels(a.w2, w2);
    if constexpr (LAYER) {
        cols.channels(a.b1, b1);
        cols.channels(a.b2, b2);
    }
    if constexpr (GATE == kChannel) {   // a channel's gate is a factor of its weight and its bias
        float gc[E];
        cols.channels((const float*)a.gate, gc);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            w1[i] *= gc[i];
            if constexpr (LAYER) b1[i] *= gc[i];
        }
    }
    const int64_t step = (int64_t)gridDim.x * R;
    const int64_t start = (int64_t)blockIdx.x * R;
    Piece<T> ry[P], rx[P], rg[P];
    cols.load(a.y, start, a.N, ry);
    cols.load(a.x, start, a.N, rx);
    if constexpr (GATE == kFull) cols.load(a.gate, start, a.N, rg);
    for (int64_t base = start; base < a.N; base += step) {
        Piece<T> cy[P], cx[P], cg[P];
        const bool live = base + cols.slot < a.N;
        cols.take(ry, live, cy);
        cols.take(rx, live, cx);
        if constexpr (GATE == kFull) cols.take(rg, live, cg);
        cols.load(a.y, base + step, a.N, ry);
        cols.load(a.x, base + step, a.N, rx);
        if constexpr (GATE == kFull) cols.load(a.gate, base + step, a.N, rg);
        float h[E];
        float v[1] = {0.f};
        if constexpr (LAYER) {
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = cy[i / N].f(i % N); v[0] += h[i]; }
            row_reduce<OpSum, G>(v, sh, W, turn);
            const float m = v[0] * inv;
            v[0] = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = cols.own(i) ? h[i] - m : 0.f; v[0] += h[i] * h[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = cy[i / N].f(i % N); v[0] += h[i] * h[i]; }
        }
        row_reduce<OpSum, G>(v, sh, W, turn);
        const float sy = 1.f / sqrtf(v[0] * inv + a.eps);
        v[0] = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float n = h[i] * sy * w1[i];
            if constexpr (LAYER) n += b1[i];
            if constexpr (GATE == kFull) n *= cg[i / N].f(i % N);
            h[i] = a.res * cx[i / N].f(i % N) + n;
            v[0] += LAYER ? h[i] : h[i] * h[i];
        }
        if (live) cols.store(a.o1, base, h);
        row_reduce<OpSum, G>(v, sh, W, turn);
        if constexpr (LAYER) {
            const float m = v[0] * inv;
            v[0] = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = cols.own(i) ? h[i] - m : 0.f; v[0] += h[i] * h[i]; }
            row_reduce<OpSum, G>(v, sh, W, turn);
        }
        const float su = 1.f / sqrtf(v[0] * inv + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            h[i] = h[i] * su * w2[i];
            if constexpr (LAYER) h[i] += b2[i];
        }
        if (live) cols.store(a.o2, base, h);
    }
}

// sums over the rows: A = sum g dh' yh (g: kFull, else without it), dw2, and for LayerNorm B = sum g dh', db2.  A channel's
// gate is a factor of its sums: dw1 = g A, db1 = g B, dgate = w1 A + b1 B.
template <bool LAYER> constexpr int kSums = LAYER ? 4 : 2;

// Waves a SIMD that the gradient's registers leave room for.  Four are better than fewer as long as little is spilt
// (16384 x 4096 bf16 LayerNorm: 225 us with 16 registers spilt, 273 us with two waves and none); with a full gate 40 are,
// and fewer waves win (377 us against 291; 16384 x 1024: 124 against 94 with three).
template <typename T, int G, bool LAYER, int GATE>
constexpr int kWaves = LAYER && GATE == kFull && sizeof(T) == 2 && G <= 512 ? G == 512 ? 2 : 3 : 4;

template <typename T, int G, int P, bool LAYER, int GATE>
__global__ __launch_bounds__(G < 256 ? 256 : G, (kWaves<T, G, LAYER, GATE>)) void backward_kernel(Args a) {
    constexpr int B = G < 256 ? 256 : G, W = B / 64, N = Piece<T>::kN, E = P * N, R = B / G;
    __shared__ float sh[2 * W * 4];
    int turn = 0;
    const int D = a.D;
    const Cols<T, G, P> cols(D);
    const float inv = 1.f / (float)D;
    // The channels' parameters stand in LDS, each thread's own (so nothing waits for another's), and leave the registers
    // to the sums: in registers the LayerNorm of 16-bit rows spilt 30 to 60 of them and took 403 us for 16384 x 4096.
    // Where a thread holds two pieces of a row (kTwo) two of the sums stand there instead, and the parameters are read
    // from the cache for each row: either alone leaves 100 registers and more spilt (4096 x 16384 RMS: 460 us).
    constexpr bool kTwo = P > 1;
    constexpr int kB1 = LAYER && GATE == kFull && !kTwo;
    __shared__ f32x4 mine[2 + kB1][E / 4][B];
    const auto put = [&](int which, const float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += 4) mine[which][i / 4][threadIdx.x] = (f32x4){v[i], v[i + 1], v[i + 2], v[i + 3]};
    };
    const auto get = [&](int which, int p, float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 x = mine[which][(p * N + i) / 4][threadIdx.x];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i + j] = x[j];
        }
    };
    const auto add = [&](int which, int p, const float (&v)[N]) {
#pragma unroll
        for (int i = 0; i < N; i += 4) mine[which][(p * N + i) / 4][threadIdx.x] += (f32x4){v[i], v[i + 1], v[i + 2], v[i + 3]};
    };
    const auto w1_of = [&](int p, float (&v)[N]) {   // a channel's gate is a factor of its weight
        if constexpr (!kTwo) get(0, p, v);
        else {
            cols.channels_all(a.w1, p, v);
            if constexpr (GATE == kChannel) {
                float gc[N];
                cols.channels_all((const float*)a.gate, p, gc);
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] *= gc[j];
            }
        }
    };
    const auto w2_of = [&](int p, float (&v)[N]) {
        if constexpr (!kTwo) get(1, p, v);
        else cols.channels_all(a.w2, p, v);
    };
    float sa[E], sw[E], sb[E], sv[E];
#pragma unroll
    for (int i = 0; i < E; ++i) sa[i] = sw[i] = sb[i] = sv[i] = 0.f;
    if constexpr (kTwo) {
        put(0, sa);
        put(1, sw);
    } else {
        float w[E];
        cols.channels(a.w2, w);
        put(1, w);
        cols.channels(a.w1, w);
        if constexpr (GATE == kChannel) {
            float gc[E];
            cols.channels((const float*)a.gate, gc);
#pragma unroll
            for (int i = 0; i < E; ++i) w[i] *= gc[i];
        }
        put(0, w);
        if constexpr (kB1) {
            cols.channels(a.b1, w);
            put(2, w);
        }
    }
    const int64_t step = (int64_t)gridDim.x * R;
    const int64_t start = (int64_t)blockIdx.x * R;
    // The next row's pieces are fetched ahead where a thread holds one piece of a row; where it holds two the registers
    // are needed for the sums.  The current row's stay packed (unpacked again at each use).
    constexpr bool kAhead = !kTwo;
    Piece<T> ry[P], rh[P], rdu[P], rdh[P], rg[P];
    auto load = [&](int64_t r) {
        cols.load(a.y, r, a.N, ry);
        cols.load(a.h, r, a.N, rh);
        cols.load(a.du, r, a.N, rdu);
        cols.load(a.dh, r, a.N, rdh);
        if constexpr (GATE == kFull) cols.load(a.gate, r, a.N, rg);
    };
    if constexpr (kAhead) load(start);
    for (int64_t base = start; base < a.N; base += step) {
        if constexpr (!kAhead) load(base);
        const bool live = base + cols.slot < a.N;
        Piece<T> y[P], h[P], du[P], dh[P], g[P];
        cols.take(ry, live, y);
        cols.take(rh, live, h);
        cols.take(rdu, live, du);
        cols.take(rdh, live, dh);
        if constexpr (GATE == kFull) cols.take(rg, live, g);
        forget(y);
        forget(h);
        forget(du);
        forget(dh);
        if constexpr (GATE == kFull) forget(g);
        if constexpr (kAhead) load(base + step);
        float my = 0.f, mh = 0.f;
        if constexpr (LAYER) {
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < E; ++i) { v[0] += y[i / N].f(i % N); v[1] += h[i / N].f(i % N); }
            row_reduce<OpSum, G>(v, sh, 4 * W, turn);
            my = v[0] * inv;
            mh = v[1] * inv;
            forget(y);
            forget(h);
        }
        // {sum y^2, sum h^2, sum k h, sum k}, k = w2 du (zero where an element is not the thread's own)
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        asm volatile("" ::: "memory");   // (the parameters are read again for each row, not kept)
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float w2[N];
            w2_of(p, w2);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float k = du[p].f(j) * w2[j], yc = y[p].f(j) - my, hc = h[p].f(j) - mh;
                const bool in = !LAYER || cols.own(p * N + j);
                v[0] += in ? yc * yc : 0.f;
                v[1] += in ? hc * hc : 0.f;
                v[2] += k * hc;
                if constexpr (LAYER) v[3] += k;
            }
        }
        row_reduce<OpSum, G>(v, sh, 4 * W, turn);
        forget(y);
        forget(h);
        forget(du);
        // (a group without a row adds nothing: its spread is not one over a zero)
        const float sy = live ? 1.f / sqrtf(v[0] * inv + a.eps) : 0.f;
        const float s = live ? 1.f / sqrtf(v[1] * inv + a.eps) : 0.f;
        const float kh = v[2] * s * inv, km = LAYER ? v[3] * inv : 0.f;
        float kp[E], t[2] = {0.f, 0.f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float dx[N], dg[N], w1[N], w2[N], b1[N], ta[N], tw[N];
            w1_of(p, w1);
            w2_of(p, w2);
            if constexpr (kB1) get(2, p, b1);
            else if constexpr (LAYER && GATE == kFull) cols.channels_all(a.b1, p, b1);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int i = p * N + j;
                const float hh = (h[p].f(j) - mh) * s, yh = (y[p].f(j) - my) * sy, d = du[p].f(j);
                const float all = dh[p].f(j) + s * (d * w2[j] - hh * kh - km);
                float dn = all;
                if constexpr (GATE == kFull) dn *= g[p].f(j);
                if constexpr (kTwo) { tw[j] = d * hh; ta[j] = dn * yh; }
                else { sw[i] += d * hh; sa[i] += dn * yh; }
                if constexpr (LAYER) { sv[i] += d; sb[i] += dn; }
                kp[i] = LAYER && kTwo && !cols.own(i) ? 0.f : dn * w1[j];
                t[0] += kp[i] * yh;
                if constexpr (LAYER) t[1] += kp[i];
                if constexpr (GATE == kFull) dg[j] = all * (LAYER ? yh * w1[j] + b1[j] : yh * w1[j]);
                dx[j] = a.res * all;
            }
            if constexpr (kTwo) {
                add(0, p, ta);
                add(1, p, tw);
            }
            if (live) {
                cols.store(a.o1, base, p, dx);
                if constexpr (GATE == kFull) cols.store(a.og, base, p, dg);
            }
        }
        row_reduce<OpSum, G>(t, sh, 4 * W, turn);
        forget(y);
        const float ky = t[0] * inv, kn = LAYER ? t[1] * inv : 0.f;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float o[N];
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] = sy * (kp[p * N + j] - (y[p].f(j) - my) * sy * ky - kn);
            if (live) cols.store(a.o2, base, p, o);
        }
    }
    // the workgroup's sums: groups of a wave first, then its waves one after the other
    constexpr int S = kSums<LAYER>, GW = G < 64 ? 64 : G;
    float* part = a.part + (int64_t)blockIdx.x * S * D;
    if constexpr (kTwo)
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float t[N];
            get(0, p, t);
#pragma unroll
            for (int j = 0; j < N; ++j) sa[p * N + j] = t[j];
            get(1, p, t);
#pragma unroll
            for (int j = 0; j < N; ++j) sw[p * N + j] = t[j];
        }
    float all[4][E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float v[4] = {sa[i], sw[i], sb[i], sv[i]};
#pragma unroll
        for (int o = G; o < 64; o <<= 1)
#pragma unroll
            for (int c = 0; c < S; ++c) v[c] += __shfl_xor(v[c], o, 64);
#pragma unroll
        for (int c = 0; c < S; ++c) all[c][i] = v[c];
    }
    if constexpr (GW < B) {
        __shared__ float red[E][B];
#pragma unroll
        for (int c = 0; c < S; ++c) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i) red[i][threadIdx.x] = all[c][i];
            __syncthreads();
            if (threadIdx.x < G)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    for (int w = GW; w < B; w += GW) all[c][i] += red[i][threadIdx.x + w];
        }
    }
    if (threadIdx.x < G)
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (cols.own(i))
#pragma unroll
                for (int c = 0; c < S; ++c) part[c * D + cols.at[i / N] + i % N] = all[c][i];
}

struct Columns { const float *w1, *b1, *gate; float *dw1, *dw2, *db1, *db2, *dgate; };

// the sums of all parts and what follows from them: 16 columns a workgroup, 64 threads a column that take every 64th part
template <bool LAYER>
__global__ __launch_bounds__(1024) void column_kernel(const float* __restrict__ part, int parts, int D, Columns c) {
    constexpr int S = kSums<LAYER>;
    __shared__ float sh[16][S][16];
    const int d = blockIdx.x * 16 + (threadIdx.x & 15), g = threadIdx.x >> 4;
    float v[S];
#pragma unroll
    for (int k = 0; k < S; ++k) v[k] = 0.f;
    if (d < D)
        for (int p = g; p < parts; p += 64)
#pragma unroll
            for (int k = 0; k < S; ++k) v[k] += part[((int64_t)p * S + k) * D + d];
#pragma unroll
    for (int o = 16; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < S; ++k) v[k] += __shfl_xor(v[k], o, 64);
    if ((threadIdx.x & 63) < 16)
#pragma unroll
        for (int k = 0; k < S; ++k) sh[threadIdx.x >> 6][k][threadIdx.x & 15] = v[k];
    __syncthreads();
    if (threadIdx.x >= 16 || d >= D) return;
    for (int w = 1; w < 16; ++w)
#pragma unroll
        for (int k = 0; k < S; ++k) v[k] += sh[w][k][threadIdx.x];
    const float gate = c.gate ? c.gate[d] : 1.f;
    c.dw1[d] = gate * v[0];
    c.dw2[d] = v[1];
    if constexpr (LAYER) { c.db1[d] = gate * v[2]; c.db2[d] = v[3]; }
    if (c.dgate) c.dgate[d] = LAYER ? c.w1[d] * v[0] + c.b1[d] * v[2] : c.w1[d] * v[0];
}

// rows of a workgroup, pieces of a thread: a thread holds 8 elements (bf16, f16) or 4 of float32 until a row needs more
// than 1024 threads
template <typename T> int row_threads(int D) {
    const int n = (D + Piece<T>::kN - 1) / Piece<T>::kN;
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : n <= 512 ? 512 : 1024;
}

// workgroups: as many as the device holds at once (`waves` a SIMD), each row group with a row at least
int grid_of(int64_t N, int threads_row, int waves = 4) {
    const int block = threads_row < 256 ? 256 : threads_row, R = block / threads_row;
    const int64_t most = (int64_t)cu_count() * (256 * waves / block), want = (N + R - 1) / R;
    return (int)(want < most ? want : most);
}

template <typename T, bool LAYER, int GATE, bool BACK>
int launch(const Args& a, int G, int grid, hipStream_t st) {
    const int n = (a.D + Piece<T>::kN - 1) / Piece<T>::kN;
#define SAMX_GO(G_, P_)                                                                                        \
    {                                                                                                          \
        constexpr int B = G_ < 256 ? 256 : G_;                                                                 \
        if constexpr (BACK) backward_kernel<T, G_, P_, LAYER, GATE><<<grid, B, 0, st>>>(a);                    \
        else forward_kernel<T, G_, P_, LAYER, GATE><<<grid, B, 0, st>>>(a);                                    \
    }
    if (G == 8) SAMX_GO(8, 1)
    else if (G == 16) SAMX_GO(16, 1)
    else if (G == 32) SAMX_GO(32, 1)
    else if (G == 64) SAMX_GO(64, 1)
    else if (G == 128) SAMX_GO(128, 1)
    else if (G == 256) SAMX_GO(256, 1)
    else if (G == 512) SAMX_GO(512, 1)
    else if (n <= 1024) SAMX_GO(1024, 1)
    else SAMX_GO(1024, 2)
#undef SAMX_GO
    SAMX_LAUNCH_CHECK();
    return SAMX_OK;
}

template <typename T, bool BACK>
int pick(const Args& a, int G, int grid, int kind, int gate, hipStream_t st) {
    if (kind == SAMX_NORM_LAYER) {
        if (gate == kNone) return launch<T, true, kNone, BACK>(a, G, grid, st);
        if (gate == kChannel) return launch<T, true, kChannel, BACK>(a, G, grid, st);
        return launch<T, true, kFull, BACK>(a, G, grid, st);
    }
    if (gate == kNone) return launch<T, false, kNone, BACK>(a, G, grid, st);
    if (gate == kChannel) return launch<T, false, kChannel, BACK>(a, G, grid, st);
    return launch<T, false, kFull, BACK>(a, G, grid, st);
}

int threads_of(int dtype, int D) { return dtype == kF32 ? row_threads<float>(D) : row_threads<bf16>(D); }
int most_dim(int dtype) { return dtype == kF32 ? 8192 : 16384; }

int check(const char* who, int64_t N, int64_t D, int dtype, int kind, int gate, float res, float eps) {
    SAMX_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown element type %d", who, dtype);
    SAMX_REQUIRE(N >= 0 && N < (int64_t(1) << 40), "%s: N %lld out of range", who, (long long)N);
    SAMX_REQUIRE(D > 0 && D <= most_dim(dtype), "%s: D %lld must be in [1, %d]", who, (long long)D, most_dim(dtype));
    SAMX_REQUIRE(kind == SAMX_NORM_RMS || kind == SAMX_NORM_LAYER, "%s: unknown norm %d", who, kind);
    SAMX_REQUIRE(gate >= kNone && gate <= kFull, "%s: unknown gate %d", who, gate);
    SAMX_REQUIRE(isfinite(res) && eps >= 0.f && isfinite(eps), "%s: res_scale must be finite, eps finite and not negative", who);
    return SAMX_OK;
}

}  // namespace

extern "C" {

int samx_block_norm(const void* x, const void* y, int dtype, int64_t N, int64_t D, const float* post_w, const float* post_b,
                    int gate_kind, const void* gate, const float* pre_w, const float* pre_b, float res_scale, int kind,
                    float eps, void* h, void* u, void* stream) {
    if (int rc = check("samx_block_norm", N, D, dtype, kind, gate_kind, res_scale, eps)) return rc;
    if (N == 0) return SAMX_OK;
    SAMX_REQUIRE(x && y && post_w && pre_w && h && u && (gate_kind == kNone || gate) &&
                     (kind == SAMX_NORM_RMS || (post_b && pre_b)), "samx_block_norm: null pointer");
    SAMX_REQUIRE(h != u, "samx_block_norm: h and u are two outputs");
    Args a{};
    a.x = x; a.y = y; a.gate = gate; a.w1 = post_w; a.b1 = post_b; a.w2 = pre_w; a.b2 = pre_b;
    a.o1 = h; a.o2 = u; a.N = N; a.D = (int)D; a.res = res_scale; a.eps = eps;
    const int G = threads_of(dtype, (int)D), grid = grid_of(N, G);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == kF32) return pick<float, false>(a, G, grid, kind, gate_kind, st);
    if (dtype == kBF16) return pick<bf16, false>(a, G, grid, kind, gate_kind, st);
    return pick<f16, false>(a, G, grid, kind, gate_kind, st);
}

size_t samx_block_norm_grad_ws_bytes(int dtype, int64_t N, int64_t D) {
    if (dtype < 0 || dtype > 2 || N < 0 || D <= 0 || D > most_dim(dtype)) return 0;
    const int G = threads_of(dtype, (int)D);
    return (size_t)grid_of(N, G) * 4 * D * sizeof(float) + 256;
}

int samx_block_norm_grad(const void* y, const void* h, const void* dh, const void* du, int dtype, int64_t N, int64_t D,
                         const float* post_w, const float* post_b, int gate_kind, const void* gate, const float* pre_w,
                         float res_scale, int kind, float eps, void* dx, void* dy, void* dgate,
                         float* dpost_w, float* dpost_b, float* dpre_w, float* dpre_b, void* ws, size_t ws_bytes,
                         void* stream) {
    if (int rc = check("samx_block_norm_grad", N, D, dtype, kind, gate_kind, res_scale, eps)) return rc;
    SAMX_REQUIRE(post_w && pre_w && dpost_w && dpre_w && ws && (N == 0 || (y && h && dh && du && dx && dy)),
                 "samx_block_norm_grad: null pointer");
    SAMX_REQUIRE(gate_kind == kNone || ((gate || (gate_kind == kFull && N == 0)) && (dgate || (gate_kind == kFull && N == 0))),
                 "samx_block_norm_grad: a gate needs its gradient's buffer");
    SAMX_REQUIRE(kind == SAMX_NORM_RMS || (post_b && dpost_b && dpre_b), "samx_block_norm_grad: LayerNorm needs its biases");
    SAMX_REQUIRE(((uintptr_t)ws & 15) == 0, "samx_block_norm_grad: the workspace has to be 16-byte aligned");
    if (ws_bytes < samx_block_norm_grad_ws_bytes(dtype, N, D))
        return samx::fail(SAMX_ERR_WORKSPACE, "samx_block_norm_grad: workspace %zu < %zu", ws_bytes,
                          samx_block_norm_grad_ws_bytes(dtype, N, D));
    Args a{};
    a.y = y; a.h = h; a.dh = dh; a.du = du; a.gate = gate; a.w1 = post_w; a.b1 = post_b; a.w2 = pre_w;
    a.o1 = dx; a.o2 = dy; a.og = dgate; a.part = (float*)ws; a.N = N; a.D = (int)D; a.res = res_scale; a.eps = eps;
    const int G = threads_of(dtype, (int)D);
    const bool fewer = kind == SAMX_NORM_LAYER && gate_kind == kFull && dtype != kF32 && G <= 512;   // (kWaves)
    const int grid = grid_of(N, G, fewer ? G == 512 ? 2 : 3 : 4);
    const hipStream_t st = (hipStream_t)stream;
    if (N > 0) {
        const int rc = dtype == kF32 ? pick<float, true>(a, G, grid, kind, gate_kind, st)
                     : dtype == kBF16 ? pick<bf16, true>(a, G, grid, kind, gate_kind, st)
                                      : pick<f16, true>(a, G, grid, kind, gate_kind, st);
        if (rc) return rc;
    }
    const bool channel = gate_kind == kChannel;
    const Columns c{post_w, post_b, channel ? (const float*)gate : nullptr, dpost_w, dpre_w, dpost_b, dpre_b,
                    channel ? (float*)dgate : nullptr};
    const unsigned blocks = (unsigned)((D + 15) / 16);
    if (kind == SAMX_NORM_LAYER) column_kernel<true><<<blocks, 1024, 0, st>>>((const float*)ws, grid, (int)D, c);
    else column_kernel<false><<<blocks, 1024, 0, st>>>((const float*)ws, grid, (int)D, c);
    SAMX_LAUNCH_CHECK();
    return SAMX_OK;
}

}  // extern "C"
