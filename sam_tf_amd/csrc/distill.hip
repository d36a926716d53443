// Imitation of a teacher's top logits: the cross-entropy part of KL(teacher || student) on K entries of a row of V logits,
// and its gradient.
//
//   x_k = t_k / tau - lse ;  p_k = e^{x_k}                lse: the teacher's normaliser, or over the K entries themselves
//   lse_z = log sum_j e^{z_j / tau}
//   loss = w sum_k p_k (x_k - (z_{i_k} / tau - lse_z))
//   grad_j = (scale w / tau) (P q_j - sum_{k: i_k = j} p_k),   q = softmax(z / tau),  P = sum_k p_k
//
// Bound: HBM, the logits read once and the gradient written once (4096 x 32000 bf16: 126 us for 526 MB, 4180 GB/s, where a
// large copy reaches 4750; the loss alone 63 us, 4200 GB/s).  A row therefore stays packed in the registers of the threads
// that read it, up to 8 pieces of 16 bytes for each of 1024 threads (65536 values of 16 bits; twice that for the gradient of
// float32 rows); a wider row is read twice.  Sums and statistics are float32, the K terms of the loss float64 (they cancel
// where student and teacher agree); each gradient value is rounded once.
#include "seq_dev.h"
#include "../../include/samx.h"

namespace {

using namespace samx::seq;

struct Args {
    const void* z; int64_t ld; int64_t N, V;
    const int32_t* idx; const float* teacher; int K;
    double inv_tau;
    const float* lse; const float* weight;
    double scale;           // of the gradient: scale / tau
    float* loss; void* grad; int64_t ldg;
};

// dynamic LDS of a row: {index, p, z} of its K entries
__host__ __device__ __forceinline__ size_t row_lds(int K) { return (size_t)((K + 3) & ~3) * 12; }

struct RowStat { float m, rs; };   // the row's maximum (0 where there is none) and one over sum e^{(z - m) / tau}

// What a row's threads do with the teacher's K entries once the statistics of the student are known.  Entries outside
// [0, V) do not count.
template <typename T, int G>
struct Teacher {
    int32_t* si; float* sp; float* sz;
    int K;
    __device__ Teacher(char* lds, int K_) : K(K_) {
        const int n = (K_ + 3) & ~3;
        si = (int32_t*)lds; sp = (float*)lds + n; sz = (float*)lds + 2 * n;
    }
    // indices, the student's logits there (before anything of the row is overwritten) and the largest teacher logit
    __device__ __forceinline__ float load(const Args& a, int64_t row, int lane, bool on) {
        const T* z = (const T*)a.z + row * a.ld;
        float mt = -INFINITY;
        for (int k = lane; k < ((K + 3) & ~3); k += G) {
            int32_t i = -1;
            float t = -INFINITY;
            if (on && k < K) {
                i = a.idx[row * K + k];
                if (i < 0 || i >= a.V) i = -1;
                else t = a.teacher[row * K + k];
            }
            si[k] = i;
            sp[k] = t;
            sz[k] = i >= 0 ? to_float(z[i]) : 0.f;
            mt = OpMax::f(mt, t);
        }
        return mt;
    }
    // sum of e^{(t - mt) / tau} (this thread's part)
    __device__ __forceinline__ float sum(float mt, float c2, int lane) const {
        float s = 0.f;
        for (int k = lane; k < K; k += G) s += __builtin_amdgcn_exp2f((sp[k] - mt) * c2);
        return s;
    }
    // p of a teacher's logit: by the caller's normaliser, or by the K entries' own maximum and sum
    struct Prob { bool given; float lse, mt, rt, c2; double inv_tau; };
    static __device__ __forceinline__ float prob(const Prob& o, float t) {
        return o.given ? expf((float)((double)t * o.inv_tau - (double)o.lse)) : __builtin_amdgcn_exp2f((t - o.mt) * o.c2) * o.rt;
    }
    // this thread's part of P
    __device__ __forceinline__ float mass(const Prob& o, int lane) const {
        float v = 0.f;
        for (int k = lane; k < K; k += G) v += prob(o, sp[k]);
        return v;
    }
    // this thread's part of the loss; sp <- p_k
    __device__ __forceinline__ double terms(const Prob& o, double lse_t, double lse_z, int lane) {
        double v = 0.0;
        for (int k = lane; k < K; k += G) {
            const float t = sp[k], p = prob(o, t);
            sp[k] = p;
            if (p != 0.f)     // (a NaN comes through)
                v += (double)p * (((double)t * o.inv_tau - lse_t) - ((double)sz[k] * o.inv_tau - lse_z));
        }
        return v;
    }
    // the entries' own gradients, over what the row's stores have left there; an index that stands twice is written by
    // the first of its entries, with the sum of all
    __device__ __forceinline__ void write(T* g, float c2, const RowStat& r, float cq, float cp, int lane) const {
        for (int k = lane; k < K; k += G) {
            const int32_t i = si[k];
            if (i < 0) continue;
            float p = 0.f;
            bool first = true;
            for (int j = 0; j < K; j += 4) {
                const int4 o = *reinterpret_cast<const int4*>(si + j);
                const int32_t e[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (e[u] == i) {
                        if (j + u < k) first = false;
                        p += sp[j + u];
                    }
            }
            if (first) g[i] = from_float<T>(cq * (__builtin_amdgcn_exp2f((sz[k] - r.m) * c2) * r.rs) - cp * p);
        }
    }
};

// log sum e^{z / tau}; of a row of nothing but -inf 0, so that log q stays -inf there
__device__ __forceinline__ double row_lse(float m, float s, double inv_tau) {
    return s > 0.f || s != s ? (double)m * inv_tau + log((double)s) : 0.0;
}

// Behind the dense part of a row: its loss, and the K entries' own gradients.  (The logarithms in float64 and the float64
// terms stand here, where nothing else of the row is in registers any more: before the stores they cost 30 of them.)
template <typename T, int G, bool GRAD>
__device__ __forceinline__ void finish(const Args& a, Teacher<T, G>& te, const typename Teacher<T, G>::Prob& o, const RowStat& r,
                                       float ss, float st, float w, float cq, float cp, int64_t row, int lane, bool live,
                                       bool on, double* shd, int& turn) {
    const double lse_z = row_lse(r.m, ss, a.inv_tau), lse_t = o.given ? (double)o.lse : row_lse(o.mt, st, a.inv_tau);
    double v[1] = {te.terms(o, lse_t, lse_z, lane)};
    row_reduce<OpSum, G>(v, shd, (G < 256 ? 256 : G) / 64, turn);
    if (live && lane == 0) a.loss[row] = on ? (float)((double)w * v[0]) : 0.f;
    if constexpr (GRAD) {
        __syncthreads();        // the row's dense part stands in memory, its p in LDS
        if (on) te.write((T*)a.grad + row * a.ldg, o.c2, r, cq, cp, lane);
    }
}

// One row for every G threads, the row in their registers: NV whole pieces each, and of the last V % kN values one.
template <typename T, int G, int NV, bool GRAD>
__global__ __launch_bounds__(G < 256 ? 256 : G, NV <= 8 ? 8 : 4) void row_kernel(Args a) {
    constexpr int B = G < 256 ? 256 : G, W = B / 64, N = Piece<T>::kN;
    extern __shared__ char lds[];
    __shared__ float shf[2 * W * 2];
    __shared__ double shd[2 * W];
    int turn = 0, turnd = 0;
    const int lane = threadIdx.x % G, slot = __builtin_amdgcn_readfirstlane(threadIdx.x / G);
    const int V = (int)a.V, whole = V / N * N, tail = V - whole;
    const int64_t row = (int64_t)blockIdx.x * (B / G) + slot;
    const bool live = row < a.N;
    const float w = live ? a.weight ? a.weight[row] : 1.f : 0.f;
    const bool on = live && w != 0.f;      // a row of weight zero is not looked at
    const T* z = (const T*)a.z + (live ? row : 0) * a.ld;
    Piece<T> raw[NV];
    const int here = on ? whole : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * G + lane) * N;
        if (at < here) {
            const Raw16 x = *reinterpret_cast<const Raw16*>(z + at);
            __builtin_memcpy(&raw[v], &x, 16);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[v].w[j] = sizeof(T) == 4 ? kNegInf<T> : kNegInf<T> * 0x10001u;
        }
    }
    const float zt = on && lane < tail ? to_float(z[whole + lane]) : -INFINITY;
    Teacher<T, G> te(lds + slot * row_lds(a.K), a.K);
    const float c2 = (float)(a.inv_tau * 1.4426950408889634);
    float mx[2] = {zt, te.load(a, row, lane, on)};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < N; ++j) mx[0] = OpMax::f(mx[0], raw[v].f(j));
    row_reduce<OpMax, G>(mx, shf, 2 * W, turn);
    forget(raw);
    RowStat r;
    r.m = mx[0] == -INFINITY ? 0.f : mx[0];
    const float mt = mx[1] == -INFINITY ? 0.f : mx[1];
    float s[2] = {__builtin_amdgcn_exp2f((zt - r.m) * c2), a.lse ? 0.f : te.sum(mt, c2, lane)};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < N; ++j) s[0] += __builtin_amdgcn_exp2f((raw[v].f(j) - r.m) * c2);
    row_reduce<OpSum, G>(s, shf, 2 * W, turn);
    r.rs = s[0] > 0.f || s[0] != s[0] ? 1.f / s[0] : 0.f;
    typename Teacher<T, G>::Prob o{a.lse != nullptr, on && a.lse ? a.lse[row] : 0.f, mt, s[1] > 0.f || s[1] != s[1] ? 1.f / s[1] : 0.f,
                                   c2, a.inv_tau};
    float cp = 0.f, cq = 0.f;
    if constexpr (GRAD) {
        float mass[1] = {te.mass(o, lane)};
        row_reduce<OpSum, G>(mass, shf, 2 * W, turn);
        if (on) {
            cp = (float)(a.scale * (double)w);
            cq = (float)(a.scale * (double)w * (double)mass[0]);
        }
        T* g = (T*)a.grad + (live ? row : 0) * a.ldg;
        const float f = cq * r.rs;
        forget(raw);
        if (live) {
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at = (v * G + lane) * N;
                float o[N];
#pragma unroll
                for (int j = 0; j < N; ++j) o[j] = f * __builtin_amdgcn_exp2f((raw[v].f(j) - r.m) * c2);
                const Piece<T> p = pack<T>(o);
                if (at < whole) {
                    Raw16 x;
                    __builtin_memcpy(&x, &p, 16);
                    *reinterpret_cast<Raw16*>(g + at) = x;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (lane < tail) g[whole + lane] = from_float<T>(f * __builtin_amdgcn_exp2f((zt - r.m) * c2));
        }
    }
    finish<T, G, GRAD>(a, te, o, r, s[0], s[1], w, cq, cp, row, lane, live, on, shd, turnd);
}

// A row that does not fit: 1024 threads read it twice.
template <typename T, bool GRAD>
__global__ __launch_bounds__(1024) void wide_kernel(Args a) {
    constexpr int G = 1024, W = G / 64, N = Piece<T>::kN, U = 4;
    extern __shared__ char lds[];
    __shared__ float shf[2 * W * 2];
    __shared__ double shd[2 * W];
    int turn = 0, turnd = 0;
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const float w = a.weight ? a.weight[row] : 1.f;
    const bool on = w != 0.f;
    const T* z = (const T*)a.z + row * a.ld;
    Teacher<T, G> te(lds, a.K);
    const float c2 = (float)(a.inv_tau * 1.4426950408889634);
    float mx[2] = {-INFINITY, te.load(a, row, lane, on)}, part = 0.f;
    for (int64_t at = (int64_t)lane * N; on && at < a.V; at += (int64_t)U * G * N) {
        Piece<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = load_piece(z, at + (int64_t)u * G * N, a.V, kNegInf<T>);
        float m = mx[0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) m = OpMax::f(m, raw[u].f(j));
        const float mm = m == -INFINITY ? 0.f : m;
        part *= __builtin_amdgcn_exp2f((mx[0] - mm) * c2);      // (0 at first: 0 * e^-inf)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < N; ++j) part += __builtin_amdgcn_exp2f((raw[u].f(j) - mm) * c2);
        mx[0] = m;
    }
    const float own = mx[0];
    row_reduce<OpMax, G>(mx, shf, 2 * W, turn);
    RowStat r;
    r.m = mx[0] == -INFINITY ? 0.f : mx[0];
    const float mt = mx[1] == -INFINITY ? 0.f : mx[1];
    float s[2] = {part * __builtin_amdgcn_exp2f((own - r.m) * c2), a.lse ? 0.f : te.sum(mt, c2, lane)};
    row_reduce<OpSum, G>(s, shf, 2 * W, turn);
    r.rs = s[0] > 0.f || s[0] != s[0] ? 1.f / s[0] : 0.f;
    typename Teacher<T, G>::Prob o{a.lse != nullptr, on && a.lse ? a.lse[row] : 0.f, mt, s[1] > 0.f || s[1] != s[1] ? 1.f / s[1] : 0.f,
                                   c2, a.inv_tau};
    float cp = 0.f, cq = 0.f;
    if constexpr (GRAD) {
        float mass[1] = {te.mass(o, lane)};
        row_reduce<OpSum, G>(mass, shf, 2 * W, turn);
        if (on) {
            cp = (float)(a.scale * (double)w);
            cq = (float)(a.scale * (double)w * (double)mass[0]);
        }
        T* g = (T*)a.grad + row * a.ldg;
        const float f = cq * r.rs;
        for (int64_t at = (int64_t)lane * N; at < a.V; at += (int64_t)U * G * N) {
            Piece<T> raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load_piece(z, at + (int64_t)u * G * N, on ? a.V : 0, kNegInf<T>);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float o[N];
#pragma unroll
                for (int j = 0; j < N; ++j) o[j] = f * __builtin_amdgcn_exp2f((raw[u].f(j) - r.m) * c2);
                store_piece(g, at + (int64_t)u * G * N, a.V, pack<T>(o));
            }
        }
    }
    finish<T, G, GRAD>(a, te, o, r, s[0], s[1], w, cq, cp, row, lane, true, on, shd, turnd);
}

// The rows in launches of at most 2^31 threads, G for each row.  (Beyond 2^32 a launch reports nothing and leaves rows out.)
template <typename T, int G, typename Go>
int in_launches(const Args& all, Go go) {
    constexpr int64_t kMost = (int64_t(1) << 31) / G;
    for (int64_t at = 0; at < all.N; at += kMost) {
        Args a = all;
        a.N = all.N - at < kMost ? all.N - at : kMost;
        a.z = (const T*)all.z + at * all.ld;
        a.idx = all.idx + at * all.K;
        a.teacher = all.teacher + at * all.K;
        if (all.lse) a.lse = all.lse + at;
        if (all.weight) a.weight = all.weight + at;
        a.loss = all.loss + at;
        if (all.grad) a.grad = (T*)all.grad + at * all.ldg;
        go(a);
        SAMX_LAUNCH_CHECK();
    }
    return SAMX_OK;
}

template <typename T, int G, int NV, bool GRAD>
int launch_row(const Args& all, hipStream_t st) {
    constexpr int B = G < 256 ? 256 : G, R = B / G;
    return in_launches<T, G>(all, [&](const Args& a) {
        row_kernel<T, G, NV, GRAD><<<(unsigned)((a.N + R - 1) / R), B, R * row_lds(a.K), st>>>(a);
    });
}

template <typename T, bool GRAD>
int launch(const Args& a, hipStream_t st) {
    const int64_t n = a.V / Piece<T>::kN;   // whole pieces of a row
    if (n <= 64) return launch_row<T, 64, 1, GRAD>(a, st);
    if (n <= 128) return launch_row<T, 64, 2, GRAD>(a, st);
    if (n <= 256) return launch_row<T, 64, 4, GRAD>(a, st);
    if (n <= 512) return launch_row<T, 256, 2, GRAD>(a, st);
    if (n <= 1024) return launch_row<T, 256, 4, GRAD>(a, st);
    if (n <= 2048) return launch_row<T, 256, 8, GRAD>(a, st);
    if (n <= 4096) return launch_row<T, 512, 8, GRAD>(a, st);
    if (n <= 8192) return launch_row<T, 1024, 8, GRAD>(a, st);
    // Behind that 16 pieces a thread leave one row a unit, and nothing runs while it is reduced: two workgroups that read
    // their rows twice (the second time out of a cache) are as good or better, but for float32 gradients.  4096 x 128000
    // bf16: loss 286 -> 226 us, gradient 550 -> 519; 4096 x 64000 float32: loss 233 -> 183, gradient 453 against 485.
    if constexpr (GRAD && sizeof(T) == 4)
        if (n <= 16384) return launch_row<T, 1024, 16, GRAD>(a, st);
    return in_launches<T, 1024>(a, [&](const Args& p) { wide_kernel<T, GRAD><<<(unsigned)p.N, 1024, row_lds(p.K), st>>>(p); });
}

int distill(const char* who, const void* logits, int64_t ld, int dtype, int64_t N, int64_t V, const int32_t* idx,
            const float* teacher, int K, float tau, const float* lse, const float* weight, float scale, float* loss,
            void* grad, int64_t ldg, hipStream_t st) {
    SAMX_REQUIRE(N >= 0 && N < (int64_t(1) << 31) && V > 0 && V < (int64_t(1) << 31) - 64, "%s: N %lld, V %lld out of range", who, (long long)N,
                 (long long)V);
    SAMX_REQUIRE(K > 0 && K <= SAMX_DISTILL_MAX_K, "%s: K %d must be in [1, %d]", who, K, SAMX_DISTILL_MAX_K);
    SAMX_REQUIRE(ld >= V && (!grad || ldg >= V), "%s: a row stride is shorter than V", who);
    SAMX_REQUIRE(tau >= 1e-6f && tau <= 1e6f && isfinite(scale), "%s: tau must be in [1e-6, 1e6], scale finite", who);
    SAMX_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown element type %d", who, dtype);
    SAMX_REQUIRE(!grad || grad != logits || ldg == ld, "%s: a gradient in place of the logits has their row stride", who);
    if (N == 0) return SAMX_OK;
    SAMX_REQUIRE(logits && idx && teacher && loss, "%s: null pointer", who);
    const Args a{logits, ld, N, V, idx, teacher, K, 1.0 / (double)tau, lse, weight, (double)scale / (double)tau, loss, grad, ldg};
    if (dtype == kF32) return grad ? launch<float, true>(a, st) : launch<float, false>(a, st);
    if (dtype == kBF16) return grad ? launch<bf16, true>(a, st) : launch<bf16, false>(a, st);
    return grad ? launch<f16, true>(a, st) : launch<f16, false>(a, st);
}

}  // namespace

extern "C" {

int samx_distill_loss(const void* logits, int64_t ld, int dtype, int64_t N, int64_t V, const int32_t* idx,
                      const float* teacher, int K, float tau, const float* lse, const float* weight, float* loss,
                      void* stream) {
    return distill("samx_distill_loss", logits, ld, dtype, N, V, idx, teacher, K, tau, lse, weight, 1.f, loss, nullptr,
                   0, (hipStream_t)stream);
}

int samx_distill_grad(const void* logits, int64_t ld, int dtype, int64_t N, int64_t V, const int32_t* idx,
                      const float* teacher, int K, float tau, const float* lse, const float* weight, float scale,
                      float* loss, void* grad, int64_t ld_grad, void* stream) {
    SAMX_REQUIRE(grad || N == 0, "samx_distill_grad: null pointer");
    return distill("samx_distill_grad", logits, ld, dtype, N, V, idx, teacher, K, tau, lse, weight, scale, loss, grad,
                   ld_grad, (hipStream_t)stream);
}

}  // extern "C"
