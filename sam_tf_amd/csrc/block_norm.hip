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
// after the other, then the workgroups in column_kernel.
#include "seq_dev.h"
#include "../../include/samx.h"

namespace {

using namespace samx::seq;

enum Gate { kNone = 0, kChannel = 1, kFull = 2 };

struct Args {
    const void *x, *y, *h, *dh, *du, *gate;
    const float *w1, *b1, *w2, *b2;
    void *o1, *o2, *og;          // h, u  or  dx, dy, dgate (kFull)
    float* part;                 // gradient: [grid][sums][D]
    int64_t N; int D;
    float res, eps;
};

// E float32 channel values of this thread; a lane's elements are P pieces of kN, piece p at (p * G + lane) * kN
template <typename T, int G, int P>
__device__ __forceinline__ void load_channels(const float* w, int D, int lane, float other, float (&out)[P * Piece<T>::kN]) {
    constexpr int N = Piece<T>::kN;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int at = (p * G + lane) * N + j;
            out[p * N + j] = w && at < D ? w[at] : other;
        }
}

template <typename T, int G, int P>
__device__ __forceinline__ void load_row(const void* base, int64_t row, int64_t rows, int D, int lane, Piece<T> (&r)[P]) {
    const T* at = (const T*)base + (row < rows ? row : 0) * (int64_t)D;
#pragma unroll
    for (int p = 0; p < P; ++p) r[p] = load_piece(at, (int64_t)(p * G + lane) * Piece<T>::kN, row < rows ? D : 0, from_float<T>(0.f));
}

template <typename T, int G, int P>
__device__ __forceinline__ void store_row(void* base, int64_t row, int D, int lane, const float (&v)[P * Piece<T>::kN]) {
    constexpr int N = Piece<T>::kN;
    T* at = (T*)base + row * (int64_t)D;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        Piece<T> o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.e[j] = from_float<T>(v[p * N + j]);
        store_piece(at, (int64_t)(p * G + lane) * N, (int64_t)D, o);
    }
}

// the lanes' elements that are channels at all (the others hold zeros and stay out of a variance)
template <typename T, int G, int P>
__device__ __forceinline__ bool in_row(int D, int lane, int i) {
    constexpr int N = Piece<T>::kN;
    return (i / N * G + lane) * N + i % N < D;
}

template <typename T, int G, int P, bool LAYER, int GATE>
__global__ __launch_bounds__(G < 256 ? 256 : G) void forward_kernel(Args a) {
    constexpr int B = G < 256 ? 256 : G, W = B / 64, N = Piece<T>::kN, E = P * N, R = B / G;
    __shared__ float sh[2 * W];
    int turn = 0;
    const int lane = threadIdx.x % G, D = a.D;
    const float inv = 1.f / (float)D;
    float w1[E], w2[E], b1[E], b2[E], gc[E];
    load_channels<T, G, P>(a.w1, D, lane, 0.f, w1);
    load_channels<T, G, P>(a.w2, D, lane, 0.f, w2);
    if constexpr (LAYER) {
        load_channels<T, G, P>(a.b1, D, lane, 0.f, b1);
        load_channels<T, G, P>(a.b2, D, lane, 0.f, b2);
    }
    if constexpr (GATE == kChannel) load_channels<T, G, P>((const float*)a.gate, D, lane, 0.f, gc);
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G;
    Piece<T> ry[P], rx[P], rg[P];
    load_row<T, G, P>(a.y, row, a.N, D, lane, ry);
    load_row<T, G, P>(a.x, row, a.N, D, lane, rx);
    if constexpr (GATE == kFull) load_row<T, G, P>(a.gate, row, a.N, D, lane, rg);
    for (int64_t base = (int64_t)blockIdx.x * R; base < a.N; base += step, row += step) {
        float h[E];
        float v[1] = {0.f};
        if constexpr (LAYER) {
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = to_float(ry[i / N].e[i % N]); v[0] += h[i]; }
            row_reduce<OpSum, G>(v, sh, W, turn);
            const float m = v[0] * inv;
            v[0] = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = in_row<T, G, P>(D, lane, i) ? h[i] - m : 0.f; v[0] += h[i] * h[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = to_float(ry[i / N].e[i % N]); v[0] += h[i] * h[i]; }
        }
        float x[E], g[E];
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = to_float(rx[i / N].e[i % N]);
        if constexpr (GATE == kFull)
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = to_float(rg[i / N].e[i % N]);
        load_row<T, G, P>(a.y, row + step, a.N, D, lane, ry);
        load_row<T, G, P>(a.x, row + step, a.N, D, lane, rx);
        if constexpr (GATE == kFull) load_row<T, G, P>(a.gate, row + step, a.N, D, lane, rg);
        row_reduce<OpSum, G>(v, sh, W, turn);
        const float sy = 1.f / sqrtf(v[0] * inv + a.eps);
        v[0] = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float n = h[i] * sy * w1[i];
            if constexpr (LAYER) n += b1[i];
            if constexpr (GATE == kChannel) n *= gc[i];
            if constexpr (GATE == kFull) n *= g[i];
            h[i] = a.res * x[i] + n;
            v[0] += LAYER ? h[i] : h[i] * h[i];
        }
        if (row < a.N) store_row<T, G, P>(a.o1, row, D, lane, h);
        row_reduce<OpSum, G>(v, sh, W, turn);
        if constexpr (LAYER) {
            const float m = v[0] * inv;
            v[0] = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) { h[i] = in_row<T, G, P>(D, lane, i) ? h[i] - m : 0.f; v[0] += h[i] * h[i]; }
            row_reduce<OpSum, G>(v, sh, W, turn);
        }
        const float su = 1.f / sqrtf(v[0] * inv + a.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            h[i] = h[i] * su * w2[i];
            if constexpr (LAYER) h[i] += b2[i];
        }
        if (row < a.N) store_row<T, G, P>(a.o2, row, D, lane, h);
    }
}

// sums over the rows, in this order: dw1, dw2, [db1, db2 (LAYER)], [dgate (kChannel)]
template <bool LAYER, int GATE> constexpr int kSums = 2 + (LAYER ? 2 : 0) + (GATE == kChannel ? 1 : 0);

template <typename T, int G, int P, bool LAYER, int GATE>
__global__ __launch_bounds__(G < 256 ? 256 : G) void backward_kernel(Args a) {
    constexpr int B = G < 256 ? 256 : G, W = B / 64, N = Piece<T>::kN, E = P * N, R = B / G;
    __shared__ float sh[2 * W * 4];
    int turn = 0;
    const int lane = threadIdx.x % G, D = a.D;
    const float inv = 1.f / (float)D;
    float w1[E], w2[E], b1[E], gc[E];
    load_channels<T, G, P>(a.w1, D, lane, 0.f, w1);
    load_channels<T, G, P>(a.w2, D, lane, 0.f, w2);
    if constexpr (LAYER && GATE != kNone) load_channels<T, G, P>(a.b1, D, lane, 0.f, b1);
    if constexpr (GATE == kChannel) load_channels<T, G, P>((const float*)a.gate, D, lane, 0.f, gc);
    float dw1[E], dw2[E], db1[E], db2[E], dgc[E];
#pragma unroll
    for (int i = 0; i < E; ++i) dw1[i] = dw2[i] = db1[i] = db2[i] = dgc[i] = 0.f;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G;
    Piece<T> ry[P], rh[P], rdu[P], rdh[P], rg[P];
    load_row<T, G, P>(a.y, row, a.N, D, lane, ry);
    load_row<T, G, P>(a.h, row, a.N, D, lane, rh);
    load_row<T, G, P>(a.du, row, a.N, D, lane, rdu);
    load_row<T, G, P>(a.dh, row, a.N, D, lane, rdh);
    if constexpr (GATE == kFull) load_row<T, G, P>(a.gate, row, a.N, D, lane, rg);
    for (int64_t base = (int64_t)blockIdx.x * R; base < a.N; base += step, row += step) {
        float y[E], h[E], du[E], dh[E], g[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
            y[i] = to_float(ry[i / N].e[i % N]);
            h[i] = to_float(rh[i / N].e[i % N]);
            du[i] = to_float(rdu[i / N].e[i % N]);
            dh[i] = to_float(rdh[i / N].e[i % N]);
            if constexpr (GATE == kFull) g[i] = to_float(rg[i / N].e[i % N]);
        }
        load_row<T, G, P>(a.y, row + step, a.N, D, lane, ry);
        load_row<T, G, P>(a.h, row + step, a.N, D, lane, rh);
        load_row<T, G, P>(a.du, row + step, a.N, D, lane, rdu);
        load_row<T, G, P>(a.dh, row + step, a.N, D, lane, rdh);
        if constexpr (GATE == kFull) load_row<T, G, P>(a.gate, row + step, a.N, D, lane, rg);
        if constexpr (LAYER) {
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < E; ++i) { v[0] += y[i]; v[1] += h[i]; }
            row_reduce<OpSum, G>(v, sh, W, turn);
            const float my = v[0] * inv, mh = v[1] * inv;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const bool in = in_row<T, G, P>(D, lane, i);
                y[i] = in ? y[i] - my : 0.f;
                h[i] = in ? h[i] - mh : 0.f;
            }
        }
        // {sum y^2, sum h^2, sum k h, sum k}, k = w2 du
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float k = du[i] * w2[i];
            v[0] += y[i] * y[i];
            v[1] += h[i] * h[i];
            v[2] += k * h[i];
            if constexpr (LAYER) v[3] += k;
        }
        row_reduce<OpSum, G>(v, sh, W, turn);
        // (a group without a row adds nothing: its spread is not one over a zero)
        const float sy = row < a.N ? 1.f / sqrtf(v[0] * inv + a.eps) : 0.f;
        const float s = row < a.N ? 1.f / sqrtf(v[1] * inv + a.eps) : 0.f;
        const float kh = v[2] * s * inv, km = LAYER ? v[3] * inv : 0.f;
        // dh becomes the whole gradient of h, y the normalised y
        float t[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float hh = h[i] * s;
            dh[i] += s * (du[i] * w2[i] - hh * kh - km);
            dw2[i] += du[i] * hh;
            if constexpr (LAYER) db2[i] += du[i];
            y[i] *= sy;
            float dn = dh[i];
            if constexpr (GATE == kChannel) dn *= gc[i];
            if constexpr (GATE == kFull) dn *= g[i];
            dw1[i] += dn * y[i];
            if constexpr (LAYER) db1[i] += dn;
            const float k = dn * w1[i];
            t[0] += k * y[i];
            if constexpr (LAYER) t[1] += k;
            // du: the gate's gradient, h: k'
            if constexpr (GATE != kNone) {
                const float n = LAYER ? y[i] * w1[i] + b1[i] : y[i] * w1[i];
                if constexpr (GATE == kChannel) dgc[i] += dh[i] * n;
                else du[i] = dh[i] * n;
            }
            h[i] = k;
            dh[i] *= a.res;
        }
        if (row < a.N) {
            store_row<T, G, P>(a.o1, row, D, lane, dh);
            if constexpr (GATE == kFull) store_row<T, G, P>(a.og, row, D, lane, du);
        }
        row_reduce<OpSum, G>(t, sh, W, turn);
        const float ky = t[0] * inv, kn = LAYER ? t[1] * inv : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) h[i] = sy * (h[i] - y[i] * ky - kn);
        if (row < a.N) store_row<T, G, P>(a.o2, row, D, lane, h);
    }
    // this row group's sums; the groups of a wave are added first
    constexpr int S = kSums<LAYER, GATE>, GW = G < 64 ? 64 : G;
    float* part = a.part + ((int64_t)blockIdx.x * (B / GW) + threadIdx.x / GW) * S * D;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        float v[5] = {dw1[i], dw2[i], db1[i], db2[i], dgc[i]};
#pragma unroll
        for (int o = G; o < 64; o <<= 1)
#pragma unroll
            for (int c = 0; c < 5; ++c) v[c] += __shfl_xor(v[c], o, 64);
        dw1[i] = v[0]; dw2[i] = v[1]; db1[i] = v[2]; db2[i] = v[3]; dgc[i] = v[4];
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int at = (i / N * G + lane) * N + i % N;
        if (at < D && threadIdx.x % GW < G) {
            part[at] = dw1[i];
            part[D + at] = dw2[i];
            if constexpr (LAYER) { part[2 * D + at] = db1[i]; part[3 * D + at] = db2[i]; }
            if constexpr (GATE == kChannel) part[(S - 1) * D + at] = dgc[i];
        }
    }
}

struct Columns { float* out[5]; };

// out[s][d] = sum over the parts: 64 columns a workgroup, 16 threads a column that take every 16th part
__global__ __launch_bounds__(1024) void column_kernel(const float* __restrict__ part, int parts, int D, int sums, Columns c) {
    __shared__ float sh[16][64];
    const int64_t col = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), all = (int64_t)sums * D;
    const int g = threadIdx.x >> 6;
    float v = 0.f;
    if (col < all)
        for (int p = g; p < parts; p += 16) v += part[p * all + col];
    sh[g][threadIdx.x & 63] = v;
    __syncthreads();
    if (g == 0 && col < all) {
        for (int i = 1; i < 16; ++i) v += sh[i][threadIdx.x & 63];
        c.out[col / D][col % D] = v;
    }
}

// rows of a workgroup, pieces of a thread: a thread holds 8 elements (bf16, f16) or 4 of float32 until a row needs more
// than 1024 threads
template <typename T> int row_threads(int D) {
    const int n = (D + Piece<T>::kN - 1) / Piece<T>::kN;
    return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : n <= 512 ? 512 : 1024;
}

// workgroups: as many as the device holds at once (two waves of work each a SIMD), each row group with a row at least
int grid_of(int64_t N, int threads_row) {
    const int block = threads_row < 256 ? 256 : threads_row, R = block / threads_row;
    const int64_t most = (int64_t)cu_count() * (1024 / block), want = (N + R - 1) / R;
    return (int)(want < most ? want : most);
}

// column sums that a workgroup leaves
int parts_of(int threads_row) { return threads_row <= 64 ? 4 : threads_row <= 256 ? 256 / threads_row : 1; }

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
    SAMX_REQUIRE(x && y && post_w && pre_w && h && u && (gate_kind == kNone || gate), "samx_block_norm: null pointer");
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
    return (size_t)grid_of(N, G) * parts_of(G) * 5 * D * sizeof(float) + 256;
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
    SAMX_REQUIRE(kind == SAMX_NORM_RMS || (dpost_b && dpre_b), "samx_block_norm_grad: LayerNorm needs dpost_b and dpre_b");
    if (ws_bytes < samx_block_norm_grad_ws_bytes(dtype, N, D))
        return samx::fail(SAMX_ERR_WORKSPACE, "samx_block_norm_grad: workspace %zu < %zu", ws_bytes,
                          samx_block_norm_grad_ws_bytes(dtype, N, D));
    Args a{};
    a.y = y; a.h = h; a.dh = dh; a.du = du; a.gate = gate; a.w1 = post_w; a.b1 = post_b; a.w2 = pre_w;
    a.o1 = dx; a.o2 = dy; a.og = dgate; a.part = (float*)ws; a.N = N; a.D = (int)D; a.res = res_scale; a.eps = eps;
    const int G = threads_of(dtype, (int)D), grid = grid_of(N, G);
    const hipStream_t st = (hipStream_t)stream;
    if (N > 0) {
        const int rc = dtype == kF32 ? pick<float, true>(a, G, grid, kind, gate_kind, st)
                     : dtype == kBF16 ? pick<bf16, true>(a, G, grid, kind, gate_kind, st)
                                      : pick<f16, true>(a, G, grid, kind, gate_kind, st);
        if (rc) return rc;
    }
    Columns c{};
    int sums = 0;
    c.out[sums++] = dpost_w;
    c.out[sums++] = dpre_w;
    if (kind == SAMX_NORM_LAYER) { c.out[sums++] = dpost_b; c.out[sums++] = dpre_b; }
    if (gate_kind == kChannel) c.out[sums++] = (float*)dgate;
    column_kernel<<<(unsigned)(((int64_t)sums * D + 63) / 64), 1024, 0, st>>>((const float*)ws, grid * parts_of(G), (int)D, sums, c);
    SAMX_LAUNCH_CHECK();
    return SAMX_OK;
}

}  // extern "C"
