// Linear attention with a decay for each head.  For a head with decay factor l = e^g:
//
//   S_t = l S_{t-1} + k_t v_t^T ;  o_t = c q_t^T S_t          (S: [D, Dv], S_{-1} the caller's state or zero)
//
// and backward, with G_t the gradient of S_t (G behind the last row: the caller's, without the factor l):
//
//   G_t = l G_{t+1} + c q_t do_t^T ;  dq_t = c S_t do_t ;  dk_t = G_t v_t ;  dv_t = G_t^T k_t ;  dS_{-1} = l G_0
//
// All four are one recurrence over positions p (rows forwards, or from the last one backwards),
//
//   out_p = ps sum_{s <= p} l^{p-s} (a_p . b_s) c_s + l^p so a_p^T X_0 ,
//
// with (a, b, c) = (q, k, v), (do, v, k), backwards (k, q, do) and (v, do, q).  X_p is the state a row at p finds,
// already decayed to it: X_{p+1} = l (X_p + kv b_p c_p^T).
//
// A chunk of 64 positions at a time, on the matrix cores: scores P = a b^T masked with l^{p-s}, out = P c + l^p a X,
// X <- l^64 X + sum_s l^{64-s} b_s c_s^T.  X stays in the registers of the workgroup (float32; each wave owns whole
// columns, and their part of out: the tiles it holds are operands of the product with a as they stand).  Operands of 16 bits
// enter the matrix cores as they are; P and X enter as two numbers of their type each, so that an output of 16 bits is rounded
// by half a step once (as one number each its error was 1.4 times that), and l^{64-s} c_s as the numbers of the type whose sum
// it is, so that the state, a float32 output, is one.  float16, which has too few exponents for any of these, takes each as
// fractions of a power of two (Scale).  float32 operands use the float32 matrix instructions throughout.
//
// Where batch times heads is less than the device holds, time is cut into segments: kv_kernel makes each segment's own
// contribution to the state behind it, join_kernel runs the recurrence over the segments, mix_kernel does the rest with
// a known state at each segment's start.
//
// Measured, 16 heads of 128, bf16.  32 x 1024 rows (two workgroups for each compute unit, no segments): 165 us, 3650 GB/s of
// 4750 that a large copy reaches.  2 x 4096 rows: 84 us in 8 segments (alone: kv 24, join 8, mix 54), the keys and values read
// twice.  Gradient of 4 x 2048 ragged rows: 131 us, two workgroups for each head's columns.  (P and X as one number each: 150,
// 78 and 111 us; X passed on through LDS as two: 190, 82 and 128, gradient of 32 x 1024 rows 519 against 432.)
// float32: its matrix instructions have a sixteenth of the rate, and its tiles leave LDS for one workgroup a unit
// (2 x 4096 rows 210 us).
#include "seq_dev.h"
#include "../../include/samx.h"
#include <type_traits>

namespace {

using namespace samx::seq;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 64, kMaxDim = 128;
constexpr int64_t kMaxHeads = 131072;   // of all sequences: three roles' workgroups of 256 threads are far fewer than 2^32 threads
constexpr int kWaves = 4, kThreads = kWaves * 64;   // a wave for each 16 rows of a chunk

// D += A B^T for 16 rows each and the kN * 4 inner values that 64 lanes' pieces hold: lane l has row l % 16, inner values
// (l / 16) * kN + [0, kN).  D: lane l has column l % 16 (B's row), rows (l / 16) * 4 + [0, 4).
__device__ __forceinline__ f32x4 mma(const Piece<bf16>& a, const Piece<bf16>& b, f32x4 d) {
    bf16x8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, d, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const Piece<f16>& a, const Piece<f16>& b, f32x4 d) {
    f16x8 x, y;
    __builtin_memcpy(&x, &a, 16);
    __builtin_memcpy(&y, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, d, 0, 0, 0);
}
// (four instructions of 4 inner values: each takes the j-th of every lane, an order of the inner values that A and B share)
__device__ __forceinline__ f32x4 mma(const Piece<float>& a, const Piece<float>& b, f32x4 d) {
#pragma unroll
    for (int j = 0; j < 4; ++j) d = __builtin_amdgcn_mfma_f32_16x16x4f32(a.f(j), b.f(j), d, 0, 0, 0);
    return d;
}

// [B, T, heads, dim], element strides; grp: query heads that share one of its heads
struct Mat { const void* p; int64_t sb, st, sh; int grp, dim; };

struct Role {
    Mat a, b, c;
    void* out; int out_f32;                    // [B, T, H, c.dim] dense, of the type or float32
    int rev;
    float kv, ps, so;                          // factors: of b c^T in the state, of the scores, of a X
    const float* s_in; int in_a, in_c;     // state before the first position, strides of a state's element (a, c)
    float* s_out;                              // state behind the last, strides as s_in's
    float* seg; int turned;                    // states at the segments' starts (workspace); turned: another role's, transposed
};

struct Args {
    Role r[3];
    int roles, H, B;
    int parts;                                 // workgroups that share the columns of c (and of the state)
    int64_t T, seg_len;
    int nseg;
    int64_t seg_size;                          // floats of a segment's state
    const float* decay;
    const int32_t* lengths;
};

__device__ __forceinline__ float power(float g, int64_t n) { return n == 0 ? 1.f : expf(g * (float)n); }

// where a workgroup works
struct Place { int role, part, b, h, seg; int64_t L; float g; };

// 8 workgroups that follow each other run on 8 dies: the roles of one (batch, head, segment) go to the same one
__device__ __forceinline__ bool place_of(const Args& a, int nseg, Place& p) {
    const int64_t units = (int64_t)a.B * a.H * nseg, id = blockIdx.x;
    const int64_t x = id & 7, k = id >> 3, unit = k / (a.roles * a.parts) * 8 + x;
    p.role = (int)(k % a.roles);
    p.part = (int)(k / a.roles % a.parts);
    if (unit >= units) return false;
    p.seg = (int)(unit % nseg);
    const int64_t bh = unit / nseg;
    p.h = (int)(bh % a.H);
    p.b = (int)(bh / a.H);
    p.L = a.T;
    if (a.lengths) {
        const int64_t n = a.lengths[p.b];
        p.L = n < 0 ? 0 : n < a.T ? n : a.T;
    }
    p.g = a.decay[p.h];
    return true;
}
inline unsigned grid_of(const Args& a, int nseg) {
    const int64_t units = (int64_t)a.B * a.H * nseg;
    return (unsigned)((units + 7) / 8 * 8 * a.roles * a.parts);
}

#define SAMX_GLOBAL __attribute__((address_space(1)))
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

// a matrix of this place in the order of positions.  EVEN: its rows are whole pieces and a chunk of them lies within 2^31
// bytes, so that a lane's place in a chunk is one offset to an address that all lanes share: no branch, nothing that waits.
// (The pointer says that it is one to global memory, which the compiler cannot see behind the choice of a role: it would
// use the instructions that may also mean LDS.)
template <typename T, bool EVEN>
struct Rows {
    static constexpr int kN = Piece<T>::kN;
    const SAMX_GLOBAL char* p;             // position 0
    int64_t step;                          // bytes from one position to the next
    int dim;
    // from column `from` on
    __device__ Rows(Mat m, Place q, int rev, int from = 0) : dim(m.dim - from) {
        p = (const SAMX_GLOBAL char*)m.p + (int64_t)sizeof(T) * (q.b * m.sb + (int64_t)(q.h / m.grp) * m.sh + from + (rev ? (q.L - 1) * m.st : 0));
        step = (int64_t)sizeof(T) * (rev ? -m.st : m.st);
    }
    // elements [at, at + kN) of position base + pos.  What lies behind the chunk's n positions or behind the row's end is
    // not what comes here: the caller does not use it.
    __device__ __forceinline__ Piece<T> piece(int64_t base, int pos, int at, int n) const {
        Piece<T> r;
        const int row = pos < n ? pos : n - 1;
        if constexpr (EVEN) {
            // (backwards the shared address is that of the chunk's last position, below which nothing lies)
            const bool back = step < 0;
            const SAMX_GLOBAL char* chunk = p + base * step + (back ? (n - 1) * step : 0);
            const uint32_t off = (back ? (uint32_t)(n - 1) * (uint32_t)-step : 0u) + (uint32_t)row * (uint32_t)step +
                                 (at < dim ? (uint32_t)at * (uint32_t)sizeof(T) : 0u);
            const u32x4 v = *(const SAMX_GLOBAL u32x4_any*)(chunk + off);
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[j] = v[j];
        } else {
            const SAMX_GLOBAL char* e = p + (base + row) * step + at * (int)sizeof(T);
            const int m = dim - at;
            if (m >= kN) {
                const u32x4 v = *(const SAMX_GLOBAL u32x4_any*)e;
#pragma unroll
                for (int j = 0; j < 4; ++j) r.w[j] = v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (sizeof(T) == 4) r.w[j] = j < m ? *(const SAMX_GLOBAL uint32_t*)(e + 4 * j) : 0u;
                    else r.w[j] = (2 * j < m ? (uint32_t)*(const SAMX_GLOBAL uint16_t*)(e + 4 * j) : 0u) |
                                  (2 * j + 1 < m ? (uint32_t)*(const SAMX_GLOBAL uint16_t*)(e + 4 * j + 2) : 0u) << 16;
                }
            }
        }
        return r;
    }
};

// 16 bytes, and 4 values, of LDS: every row and every column that comes here is a multiple of them
template <typename T>
__device__ __forceinline__ Piece<T> lds_piece(const T* p) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(p);
    Piece<T> r;
    __builtin_memcpy(&r, &v, 16);
    return r;
}
template <typename T>
__device__ __forceinline__ void lds_put(T* p, const Piece<T>& r) {
    u32x4 v;
    __builtin_memcpy(&v, &r, 16);
    *reinterpret_cast<u32x4*>(p) = v;
}
// 4 values, rounded; v: what of them that leaves
__device__ __forceinline__ void put_part(float* p, float (&v)[4]) { *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]}; }
template <typename T>
__device__ __forceinline__ void put_part(T* p, float (&v)[4]) {
    const u32x2 x = {pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
    *reinterpret_cast<u32x2*>(p) = x;
    Piece<T> r;
    r.w[0] = x[0];
    r.w[1] = x[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] -= r.f(e);
}
// A piece down a column: elements [0, kN) are rows[e][lane % 16].  16 bits: two transposing reads, in each of which 16
// lanes read 4 rows of 16 values and get a column each; with 4-byte values a read for each row.
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ Piece<T> lds_column(const T* rows, int stride) {
    const int r16 = threadIdx.x & 15;
    Piece<T> r;
    if constexpr (sizeof(T) == 2) {
        const T* p = rows + (r16 >> 2) * stride + (r16 & 3) * 4;
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + 4 * stride));
        __builtin_memcpy(&r.w[0], &a, 8);
        __builtin_memcpy(&r.w[2], &b, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) r.w[e] = __float_as_uint(rows[e * stride + r16]);
    }
    return r;
}

// float16: values that are to be rounded to it, or split into parts of it, are first taken to a power of two's fractions, so
// that the largest of those that share it stands in [2^14, 2^15): none overflows, and what is below 2^-39 of the largest is all
// that is lost.  One power for each column of c and of X and one for each row of P: lanes of one l % 16.  (Without it a value
// of the state beyond 65504 was an infinity to its rows, and the state of values around 1e-5 had a few per cent of error.)
// It costs: 32 x 1024 rows, 16 heads of 128, 204 us where bfloat16 takes 163; the gradient of 4 x 2048 rows 188, not 167.
template <typename T> constexpr bool kScaled = std::is_same<T, f16>::value;
struct Scale { float up, down; };              // the power and one over it
// of values whose magnitudes are at most `most` (in this lane); none below 2^(least - 127 - 14)
__device__ __forceinline__ Scale scale_of(float most, uint32_t least = 15) {
    // (rows of lanes exchanged by the vector unit; by LDS's permutation the gradient of 2 x 4096 rows took 197 us, not 184)
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(most), __float_as_uint(most), false, false);
    most = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
    most = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
    uint32_t e = __float_as_uint(most) >> 23;
    e = e < least ? least : e > 254u ? 254u : e;
    return {__uint_as_float((e - 14u) << 23), __uint_as_float((268u - e) << 23)};
}

// numbers that a score and a value of X are as they enter a product: two of 16 bits, the second what the first has left
template <typename T> constexpr int kHalves = sizeof(T) == 2 ? 2 : 1;

// LDS rows are 16 bytes longer than their contents: 16 lanes that read 16 rows at one column use all banks
template <typename T, int DP, int DC>
struct LdsKv {
    static constexpr int kRow = DP + Piece<T>::kN, kRowC = DC + Piece<T>::kN;
    T b[kChunk][kRow], c[kChunk][kRowC];                 // the chunk's rows
    float lam[2 * kChunk + 1];                           // l^(n - kChunk), 0 below kChunk
    uint32_t odd, pad[2];                                // 1 + the last chunk whose c has an infinity or a NaN
};
template <typename T, int DP, int DC>
struct Lds : LdsKv<T, DP, DC> {
    static constexpr int kTok = kChunk + Piece<T>::kN;
    static_assert(sizeof(LdsKv<T, DP, DC>) % 16 == 0, "pieces are read whole");
    T a[kChunk][LdsKv<T, DP, DC>::kRow];
    T p[kHalves<T>][kChunk][kTok];                       // scores
    float ps[kScaled<T> ? kChunk : 4], xs[kScaled<T> ? DC : 4];   // the powers of two of P's rows and X's columns
};

// N groups of products, group g's operands read (into buf[g % (AHEAD + 1)]) AHEAD groups before they are used; nothing is
// moved across the groups.  (Left to itself the compiler saves registers by reading what it multiplies next.)
template <int N, int AHEAD, int I = 0, typename Read, typename Use>
__device__ __forceinline__ void in_groups(Read read, Use use) {
    if constexpr (I == 0) {
#pragma unroll
        for (int g = 0; g < (AHEAD < N ? AHEAD : N); ++g) read(g, g % (AHEAD + 1));
        __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (I < N) {
        if constexpr (I + AHEAD < N) read(I + AHEAD, (I + AHEAD) % (AHEAD + 1));
        __builtin_amdgcn_sched_barrier(0);
        use(I, I % (AHEAD + 1));
        __builtin_amdgcn_sched_barrier(0);
        in_groups<N, AHEAD, I + 1>(read, use);
    }
}

// a bit of a dword's element(s) whose exponent is all ones, gathered by "or"
template <typename T>
__device__ __forceinline__ uint32_t odd_bits(uint32_t w) {
    constexpr uint32_t e = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, f16>::value ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t one = sizeof(T) == 4 ? 0x00800000u : std::is_same<T, f16>::value ? 0x04000400u : 0x00800080u;
    return ((w & e) + one) & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u);
}

// A chunk's rows of b and c, and of a as A says, on their way to LDS.  kByRow: each lane has pieces of one row of a, so that a row
// that is not whole pieces costs a lane one piece that waits for its elements, not four (100 of 128 dimensions, bfloat16,
// gradient of 4 x 2048 rows, 4 key heads: 350 us against 398); whole pieces do better side by side (4 x 2048 rows of 128: 167
// against 171; float32 519 against 568).
enum StageA { kNoA, kSideBySide, kByRow };
template <typename T, int DP, int DC, StageA A>
struct Staged {
    static constexpr int kN = Piece<T>::kN;
    static constexpr int kAcross = DP / kN, kDown = kThreads / kAcross, kPer = kChunk / kDown;
    static constexpr int kAcrossC = DC / kN, kDownC = kThreads / kAcrossC, kPerC = kChunk / kDownC;
    Piece<T> a[A == kNoA ? 1 : kPer], b[kPer], c[kPerC];
    static __device__ __forceinline__ int a_row(int u) {
        return A == kByRow ? threadIdx.x / 64 * 16 + threadIdx.x % 16 : threadIdx.x / kAcross + u * kDown;
    }
    static __device__ __forceinline__ int a_col(int u) {
        return (A == kByRow ? u * 4 + threadIdx.x % 64 / 16 : threadIdx.x % kAcross) * kN;
    }
    template <bool EVEN>
    __device__ __forceinline__ void load(const Rows<T, EVEN>& ma, const Rows<T, EVEN>& mb, const Rows<T, EVEN>& mc, int64_t base, int n) {
        const int t = threadIdx.x / kAcross, d = threadIdx.x % kAcross * kN;
        const int tc = threadIdx.x / kAcrossC, e = threadIdx.x % kAcrossC * kN;
        if constexpr (A != kNoA)
#pragma unroll
            for (int u = 0; u < kPer; ++u) a[u] = ma.piece(base, a_row(u), a_col(u), n);
#pragma unroll
        for (int u = 0; u < kPer; ++u) b[u] = mb.piece(base, t + u * kDown, d, n);
#pragma unroll
        for (int u = 0; u < kPerC; ++u) c[u] = mc.piece(base, tc + u * kDownC, e, n);
    }
    // zeros behind the rows' ends and behind the n positions (a and b are as wide)
    template <typename L>
    __device__ __forceinline__ uint32_t store(L& l, int db, int dc, int n) const {
        const int t = threadIdx.x / kAcross, d = threadIdx.x % kAcross * kN;
        const int tc = threadIdx.x / kAcrossC, e = threadIdx.x % kAcrossC * kN;
        uint32_t odd = 0;                 // whether c has something that is not finite
#pragma unroll
        for (int u = 0; u < kPer; ++u) {
            const uint32_t ka = a_col(u) < db && a_row(u) < n ? ~0u : 0u;
            const uint32_t kb = d < db && t + u * kDown < n ? ~0u : 0u, kc = e < dc && tc + u * kDownC < n ? ~0u : 0u;
            Piece<T> w, x, y;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (A != kNoA) w.w[j] = a[u].w[j] & ka;
                x.w[j] = b[u].w[j] & kb;
                if (u < kPerC) { y.w[j] = c[u].w[j] & kc; odd |= odd_bits<T>(y.w[j]); }
            }
            if constexpr (A != kNoA) lds_put(&l.a[a_row(u)][a_col(u)], w);
            lds_put(&l.b[t + u * kDown][d], x);
            if (u < kPerC) lds_put(&l.c[tc + u * kDownC][e], y);
        }
        return odd;
    }
};

// X of a workgroup: wave w owns the tiles of 16 columns w, w + kWaves, ...; tile (j, i): lane l has column l % 16, rows
// (l / 16) * 4 + [0, 4) of the a side
template <int DP, int DC>
struct State {
    static constexpr int kJ = DC / 16 / kWaves, kI = DP / 16;
    f32x4 x[kJ][kI];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int i = 0; i < kI; ++i) x[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
};

// Tile column j of X as it enters a product with a, inner values of mma m: the lane's own registers.  16 bits: the tiles 2m and
// 2m + 1, an order of the inner values that a_piece has too, rounded (X half 0) and what of it that leaves (half 1).
template <typename T, int DP, int DC>
__device__ __forceinline__ void x_pieces(const State<DP, DC>& S, int j, int m, float down, Piece<T> (&x)[kHalves<T>]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[0].w[e] = __float_as_uint(S.x[j][m][e]);
    } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = kScaled<T> ? S.x[j][2 * m + e / 4][e % 4] * down : S.x[j][2 * m + e / 4][e % 4];
        x[0] = pack<T>(v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] -= x[0].f(e);
        x[1] = pack<T>(v);
    }
}
template <typename T>
__device__ __forceinline__ Piece<T> a_piece(const T* row, int m, int q) {
    if constexpr (sizeof(T) == 4) return lds_piece(row + m * 16 + q * 4);
    else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(row + m * 32 + q * 4), y = *reinterpret_cast<const u32x2*>(row + m * 32 + 16 + q * 4);
        Piece<T> r;
        r.w[0] = x[0]; r.w[1] = x[1]; r.w[2] = y[0]; r.w[3] = y[1];
        return r;
    }
}

// numbers of the type whose sum a float32 is
template <typename T> constexpr int kParts = 1;
template <> inline constexpr int kParts<f16> = 3;
template <> inline constexpr int kParts<bf16> = 3;

// X <- l^end X + kv sum_s l^{end - s} b_s c_s^T, with l^{end - s} c_s in as many numbers of the type as it has
template <typename T, int DP, int DC, typename L>
__device__ __forceinline__ void update(State<DP, DC>& S, const L& l, int end, float kv) {
    constexpr int kN = Piece<T>::kN, kJ = State<DP, DC>::kJ, kI = State<DP, DC>::kI, kP = kParts<T>;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, q = lane >> 4;
    const float whole = l.lam[kChunk + end];
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int i = 0; i < kI; ++i) S.x[j][i] *= whole;
#pragma unroll
    for (int k = 0; k < kChunk; k += 4 * kN) {
        const int s0 = k + q * kN;
        float f[kN];
        Piece<T> c[kJ];
#pragma unroll
        for (int e = 0; e < kN; ++e) f[e] = l.lam[kChunk + end - s0 - e];   // (rows behind the end are zeros, and their factors)
#pragma unroll
        for (int j = 0; j < kJ; ++j) c[j] = lds_column(&l.c[s0][(w + kWaves * j) * 16], L::kRowC);
        __builtin_amdgcn_sched_barrier(0);
        Piece<T> part[kJ][kP];
        float up[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
            float v[kN];
#pragma unroll
            for (int e = 0; e < kN; ++e) v[e] = c[j].f(e) * (kv * f[e]);
            if constexpr (kScaled<T>) {
                float most = 0.f;
#pragma unroll
                for (int e = 0; e < kN; ++e) most = fmaxf(most, fabsf(v[e]));
                const Scale s = scale_of(most);
                up[j] = s.up;
#pragma unroll
                for (int e = 0; e < kN; ++e) v[e] *= s.down;
            }
#pragma unroll
            for (int u = 0; u < kP; ++u) {
                part[j][u] = pack<T>(v);
#pragma unroll
                for (int e = 0; e < kN; ++e) v[e] -= part[j][u].f(e);
            }
        }
        Piece<T> b[2][4];
        in_groups<kI / 4, 1>(
            [&](int g, int at) {
#pragma unroll
                for (int i = 0; i < 4; ++i) b[at][i] = lds_column(&l.b[s0][(g * 4 + i) * 16], L::kRow);
            },
            [&](int g, int at) {
                f32x4 d[kJ][4];
#pragma unroll
                for (int j = 0; j < kJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) d[j][i] = kScaled<T> ? f32x4{0.f, 0.f, 0.f, 0.f} : S.x[j][g * 4 + i];
#pragma unroll
                for (int u = 0; u < kP; ++u)
#pragma unroll
                    for (int j = 0; j < kJ; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[j][i] = mma(b[at][i], part[j][u], d[j][i]);
#pragma unroll
                for (int j = 0; j < kJ; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if constexpr (kScaled<T>) S.x[j][g * 4 + i] += up[j] * d[j][i];
                        else S.x[j][g * 4 + i] = d[j][i];
                    }
            });
    }
}

// A caller's state, [da, dc] values with the strides sa, sc: to and from a workgroup's registers.
template <int DP, int DC>
__device__ __forceinline__ void state_load(State<DP, DC>& S, const SAMX_GLOBAL float* m, int da, int dc, int sa, int sc, float f) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < State<DP, DC>::kJ; ++j)
#pragma unroll
        for (int i = 0; i < State<DP, DC>::kI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = (w + kWaves * j) * 16 + r16, a = i * 16 + q * 4 + e;
                const bool there = a < da && c < dc;
                const float v = m[(uint32_t)(there ? a * sa + c * sc : 0)];      // (no branch: the loads go out together)
                S.x[j][i][e] = there ? v * f : 0.f;
            }
}
template <int DP, int DC>
__device__ __forceinline__ void state_store(const State<DP, DC>& S, SAMX_GLOBAL float* m, int da, int dc, int sa, int sc) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < State<DP, DC>::kJ; ++j)
#pragma unroll
        for (int i = 0; i < State<DP, DC>::kI; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = (w + kWaves * j) * 16 + r16, a = i * 16 + q * 4 + e;
                if (a < da && c < dc) m[(uint32_t)(a * sa + c * sc)] = S.x[j][i][e];
            }
}
// A segment's state in the workspace: all tiles, [columns][rows] dense; `turned`: the matrix that is wanted is its transpose.
template <int DP, int DC>
__device__ __forceinline__ void seg_load(State<DP, DC>& S, const SAMX_GLOBAL float* m, bool turned) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < State<DP, DC>::kJ; ++j)
#pragma unroll
        for (int i = 0; i < State<DP, DC>::kI; ++i) {
            const uint32_t c = (w + kWaves * j) * 16 + r16, a = i * 16 + q * 4;
            if (!turned) {
                S.x[j][i] = *(const SAMX_GLOBAL f32x4*)(m + c * DP + a);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) S.x[j][i][e] = m[(a + e) * DP + c];
            }
        }
}
template <int DP, int DC>
__device__ __forceinline__ void seg_store(const State<DP, DC>& S, SAMX_GLOBAL float* m) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
#pragma unroll
    for (int j = 0; j < State<DP, DC>::kJ; ++j)
#pragma unroll
        for (int i = 0; i < State<DP, DC>::kI; ++i)
            *(SAMX_GLOBAL f32x4*)(m + (uint32_t)(((w + kWaves * j) * 16 + r16) * DP + i * 16 + q * 4)) = S.x[j][i];
}

template <typename T, int DP, bool EVEN>
__global__ __launch_bounds__(kThreads, 2) void kv_kernel(Args A) {
    extern __shared__ __attribute__((aligned(16))) char lds_[];
    LdsKv<T, DP, DP>& l = *reinterpret_cast<LdsKv<T, DP, DP>*>(lds_);
    Place p;
    if (!place_of(A, A.nseg - 1, p)) return;
    const int64_t at = (int64_t)p.seg * A.seg_len;
    if (p.L <= at + A.seg_len) return;                  // nobody follows
    const Role r = A.r[p.role];
    const Rows<T, EVEN> b(r.b, p, r.rev), c(r.c, p, r.rev);
    if (threadIdx.x <= 2 * kChunk) l.lam[threadIdx.x] = threadIdx.x < kChunk ? 0.f : power(p.g, threadIdx.x - kChunk);
    State<DP, DP> S;
    S.zero();
    Staged<T, DP, DP, kNoA> st;
    st.load(b, b, c, at, kChunk);
    for (int64_t k = 0; k < A.seg_len; k += kChunk) {
        __syncthreads();
        st.store(l, r.b.dim, r.c.dim, kChunk);
        __syncthreads();
        if (k + kChunk < A.seg_len) st.load(b, b, c, at + k + kChunk, kChunk);
        update<T, DP, DP>(S, l, kChunk, r.kv);
    }
    seg_store<DP, DP>(S, (SAMX_GLOBAL float*)r.seg + ((int64_t)(p.b * A.H + p.h) * (A.nseg - 1) + p.seg) * A.seg_size);
}

// states at the segments' starts: X_{j+1} = l^len X_j + (segment j's own), over the segments that have a follower
template <int DP>
__global__ __launch_bounds__(256) void join_kernel(Args A) {
    constexpr int U = 8;
    const Role& r = A.r[blockIdx.z];
    const int64_t bh = blockIdx.x;
    const int e = blockIdx.y * 256 + threadIdx.x, na = r.b.dim, nc = r.c.dim, states = A.nseg - 1;
    const int b = (int)(bh / A.H), h = (int)(bh % A.H);
    int64_t L = A.T;
    if (A.lengths) L = A.lengths[b] < A.T ? A.lengths[b] : A.T;
    const int i = e % DP, j = e / DP;
    if (i >= na || j >= nc) return;       // (kv_kernel has left zeros there)
    const float g = A.decay[h], f = power(g, A.seg_len);
    float x = 0.f;
    if (r.s_in) x = r.s_in[bh * na * nc + i * r.in_a + j * r.in_c] * (r.rev ? 1.f : power(g, 1));
    float* s = r.seg + bh * states * A.seg_size + e;
    int n = 0;                                          // states that are wanted
    while (n < states && (int64_t)(n + 1) * A.seg_len < L) ++n;
    for (int k = 0; k < n; k += U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = k + u < n ? s[(int64_t)(k + u) * A.seg_size] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x = f * x + v[u];
            if (k + u < n) s[(int64_t)(k + u) * A.seg_size] = x;
        }
    }
}

template <typename T, int DP, int DC, bool EVEN>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP == 128 ? 1 : 2) void mix_kernel(Args A) {
    constexpr int kN = Piece<T>::kN, kInner = 4 * kN, kK = DP / kInner;      // inner values of one mma
    extern __shared__ __attribute__((aligned(16))) char lds_[];
    Lds<T, DP, DC>& l = *reinterpret_cast<Lds<T, DP, DC>*>(lds_);
    constexpr int kRowC = LdsKv<T, DP, DC>::kRowC;
    Place p;
    if (!place_of(A, A.nseg, p)) return;
    // (by value: a reference into the arguments makes the compiler keep a copy of all of them in scratch memory)
    const Role r = A.r[p.role];
    // wave w: tiles w, w + kWaves of the columns, of the state and of out; of a chunk's scores, rows 16 w + [0, 16)
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int64_t at = (int64_t)p.seg * A.seg_len, bh = (int64_t)p.b * A.H + p.h;
    const int64_t to = at + A.seg_len < p.L ? at + A.seg_len : p.L;         // this segment's positions
    constexpr bool kShare = DC < DP;       // a workgroup has DC of the columns
    const int c0 = kShare ? p.part * DC : 0;
    const int da = r.a.dim, all = r.c.dim, dc = kShare && all - c0 > DC ? DC : all - c0;
    if (kShare && dc <= 0) return;
    const int64_t out_row = (int64_t)A.H * all;
    const int64_t out_at = ((int64_t)p.b * A.T * A.H + p.h) * all + c0;
    SAMX_GLOBAL char* const outp = (SAMX_GLOBAL char*)r.out + out_at * (r.out_f32 ? 4 : (int)sizeof(T));
    // four of a row's outputs from d on, those that exist; el: elements from the first row to it
    auto put4 = [=](auto f32, int64_t el, int d, f32x4 v) {
        if constexpr (decltype(f32)::value) {
            SAMX_GLOBAL float* o = (SAMX_GLOBAL float*)outp + el + d;
            if (EVEN) { if (d < dc) *(SAMX_GLOBAL f32x4_any*)o = v; return; }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d + e < dc) o[e] = v[e];
        } else if constexpr (sizeof(T) == 2) {
            SAMX_GLOBAL uint16_t* o = (SAMX_GLOBAL uint16_t*)outp + el + d;
            const uint32_t lo = pack2<T>(v[0], v[1]), hi = pack2<T>(v[2], v[3]);
            if (EVEN) { if (d < dc) *(SAMX_GLOBAL u32x2_any*)o = u32x2{lo, hi}; return; }
            if (d < dc) o[0] = (uint16_t)lo;
            if (d + 1 < dc) o[1] = (uint16_t)(lo >> 16);
            if (d + 2 < dc) o[2] = (uint16_t)hi;
            if (d + 3 < dc) o[3] = (uint16_t)(hi >> 16);
        }
    };
    const bool wide = sizeof(T) == 4 || r.out_f32;
    {   // rows behind the trajectory's end
        const int64_t z0 = at > p.L ? at : p.L, z1 = at + A.seg_len < A.T ? at + A.seg_len : A.T;
        for (int64_t t = z0 + w; t < z1; t += kWaves)
            for (int d = lane * 4; d < dc; d += 256) {
                if (wide) put4(std::true_type(), t * out_row, d, f32x4{0.f, 0.f, 0.f, 0.f});
                else put4(std::false_type(), t * out_row, d, f32x4{0.f, 0.f, 0.f, 0.f});
            }
    }
    State<DP, DC> S;
    const SAMX_GLOBAL float* s_in = r.s_in ? (const SAMX_GLOBAL float*)r.s_in + bh * da * all + c0 * r.in_c : nullptr;
    SAMX_GLOBAL float* s_out = r.s_out ? (SAMX_GLOBAL float*)r.s_out + bh * da * all + c0 * r.in_c : nullptr;
    if (p.L == 0) {    // nothing to read: the state goes through
        if (p.seg == 0 && s_out) {
            if (s_in) state_load<DP, DC>(S, s_in, da, dc, r.in_a, r.in_c, 1.f);
            else S.zero();
            state_store<DP, DC>(S, s_out, da, dc, r.in_a, r.in_c);
        }
        return;
    }
    if (at >= to) return;
    const Rows<T, EVEN> a(r.a, p, r.rev), b(r.b, p, r.rev), c(r.c, p, r.rev, c0);
    const int row = w * 16 + r16;          // of a chunk: the one whose scores this lane makes
    Staged<T, DP, DC, EVEN || sizeof(T) == 4 ? kSideBySide : kByRow> st;
    auto rows_at = [&](int64_t base) { return (int)(to - base < kChunk ? to - base : kChunk); };
    st.load(a, b, c, at, rows_at(at));
    const bool last = to == p.L;           // this segment makes the state behind the last position
    if (p.seg > 0) seg_load<DP, DC>(S, (const SAMX_GLOBAL float*)r.seg + (bh * (A.nseg - 1) + p.seg - 1) * A.seg_size +
                                           (r.turned ? c0 : c0 * DP), r.turned);
    else if (s_in) state_load<DP, DC>(S, s_in, da, dc, r.in_a, r.in_c, r.rev ? 1.f : power(p.g, 1));
    else S.zero();
    if (threadIdx.x <= 2 * kChunk) l.lam[threadIdx.x] = threadIdx.x < kChunk ? 0.f : power(p.g, threadIdx.x - kChunk);
    if (threadIdx.x == 0) l.odd = 0u;
    __syncthreads();
    constexpr int kJ = State<DP, DC>::kJ, kU = kHalves<T>;
    for (int64_t base = at; base < to; base += kChunk) {
        const int n = (int)(to - base < kChunk ? to - base : kChunk);
        const bool more = base + kChunk < to;
        const uint32_t chunk = (uint32_t)((base - at) / kChunk) + 1u;
        if (st.store(l, da, dc, n)) l.odd = chunk;
        __syncthreads();
        if (more) st.load(a, b, c, base + kChunk, rows_at(base + kChunk));
        // scores, transposed: column = this lane's row, rows = positions s.  (Nothing here branches on the wave: no read
        // would be ahead of its use across a branch.)
        f32x4 sc[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) sc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        {
            Piece<T> f[3][5];
            in_groups<kK, 2>(
                [&](int k, int at) {
                    f[at][4] = lds_piece(&l.a[row][k * kInner + q * kN]);
#pragma unroll
                    for (int t = 0; t < 4; ++t) f[at][t] = lds_piece(&l.b[t * 16 + r16][k * kInner + q * kN]);
                },
                [&](int k, int at) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) sc[t] = mma(f[at][t], f[at][4], sc[t]);
                });
        }
        {
            float v[4][4], most = 0.f;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // (l^d is 0 behind the row, but 0 times a NaN is none)
                    const float x = r.ps * l.lam[kChunk + row - (t * 16 + q * 4 + e)] * sc[t][e];
                    v[t][e] = row >= t * 16 + q * 4 + e ? x : 0.f;
                    if constexpr (kScaled<T>) most = fmaxf(most, fabsf(v[t][e]));
                }
            if constexpr (kScaled<T>) {
                // (not below 2^-54: a X is divided by it, and such scores add nothing to an output of this type)
                const Scale s = scale_of(most, 127 - 40);
                if (q == 0) l.ps[row] = s.up;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[t][e] *= s.down;
            }
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
                for (int t = 0; t < 4; ++t) put_part(&l.p[u][row][t * 16 + q * 4], v[t]);
        }
        float down[kJ];
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
            down[j] = 1.f;
            if constexpr (kScaled<T>) {
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < State<DP, DC>::kI; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) most = fmaxf(most, fabsf(S.x[j][i][e]));
                const Scale s = scale_of(most);
                down[j] = s.down;
                if (q == 0) l.xs[(w + kWaves * j) * 16 + r16] = s.up;
            }
        }
        // out, transposed, of this wave's columns: column = position t * 16 + lane % 16, rows = columns of c
        f32x4 o[4][kJ];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < kJ; ++j) o[t][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        {
            Piece<T> f[2][4];
            in_groups<kK, 1>(
                [&](int m, int at) {
#pragma unroll
                    for (int t = 0; t < 4; ++t) f[at][t] = a_piece(&l.a[t * 16 + r16][0], m, q);
                },
                [&](int m, int at) {
#pragma unroll
                    for (int j = 0; j < kJ; ++j) {
                        Piece<T> x[kU];
                        x_pieces<T, DP, DC>(S, j, m, down[j], x);
#pragma unroll
                        for (int u = 0; u < kU; ++u)
#pragma unroll
                            for (int t = 0; t < 4; ++t) o[t][j] = mma(x[u], f[at][t], o[t][j]);
                    }
                });
        }
        __syncthreads();                   // everybody's scores are there
        // of position t * 16 + lane % 16: a X's factor, and the power of two that the scores' row has been divided by
        const auto factors = [&](int t, float& d, float& up) {
            d = r.so * l.lam[kChunk + t * 16 + r16];
            up = 1.f;
            if constexpr (kScaled<T>) {
                up = l.ps[t * 16 + r16];
                d *= __uint_as_float((254u << 23) - __float_as_uint(up));        // one over a power of two
            }
        };
        const auto decayed = [&](int j, float d, f32x4 v) {
            // (one factor after the other: their product can be an infinity where v is 0)
            if constexpr (kScaled<T>) return (v * *reinterpret_cast<const f32x4*>(&l.xs[(w + kWaves * j) * 16 + q * 4])) * d;
            else return v * d;
        };
        float up[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            float d;
            factors(t, d, up[t]);
#pragma unroll
            for (int j = 0; j < kJ; ++j) o[t][j] = decayed(j, d, o[t][j]);
        }
        {
            Piece<T> fc[2][kJ], fp[2][4];
            in_groups<kChunk / kInner * kU, 1>(
                [&](int g, int at) {
                    const int k = g / kU, u = g % kU;
                    if (u == 0)
#pragma unroll
                        for (int j = 0; j < kJ; ++j) fc[k % 2][j] = lds_column(&l.c[k * kInner + q * kN][(w + kWaves * j) * 16], kRowC);
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        if (k * kInner < (t + 1) * 16) fp[at][t] = lds_piece(&l.p[u][t * 16 + r16][k * kInner + q * kN]);
                },
                [&](int g, int at) {
                    const int k = g / kU;
#pragma unroll
                    for (int j = 0; j < kJ; ++j)
#pragma unroll
                        for (int t = 0; t < 4; ++t)
                            if (k * kInner < (t + 1) * 16) o[t][j] = mma(fc[k % 2][j], fp[at][t], o[t][j]);
                });
        }
        // (elements from the first row of out to position `base`'s, and on from one position to the next)
        const int64_t o_base = (r.rev ? p.L - 1 - base : base) * out_row, o_step = r.rev ? -out_row : out_row;
        const int64_t o_lane = r16 * o_step;
        const auto put = [&](int t, int j, f32x4 v) {
            if (t * 16 + r16 >= n) return;
            const int64_t el = o_base + t * 16 * o_step + o_lane;
            if (wide) put4(std::true_type(), el, (w + kWaves * j) * 16 + q * 4, v);
            else put4(std::false_type(), el, (w + kWaves * j) * 16 + q * 4, v);
        };
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < kJ; ++j) put(t, j, kScaled<T> ? o[t][j] * up[t] : o[t][j]);
        if (__builtin_amdgcn_readfirstlane(l.odd) == chunk) {
            // Zeros behind a row's own position times an infinity or a NaN there were NaN in what has just been written: once
            // more, with the scores' products one after the other, up to the row.  (Kept out of the way of the products above: as
            // their other branch it cost them their reads ahead, a quarter more time for the gradient of 4 x 2048 rows.)
#pragma unroll 1
            for (int t = 0; t < 4; ++t) {
                float d, up;
                factors(t, d, up);
#pragma unroll
                for (int j = 0; j < kJ; ++j) {
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int m = 0; m < kK; ++m) {
                        Piece<T> x[kU];
                        x_pieces<T, DP, DC>(S, j, m, down[j], x);
                        const Piece<T> f = a_piece(&l.a[t * 16 + r16][0], m, q);
#pragma unroll
                        for (int u = 0; u < kU; ++u) v = mma(x[u], f, v);
                    }
                    v = decayed(j, d, v);
                    for (int i = 0; i <= t * 16 + r16; ++i) {
                        float x = 0.f;
#pragma unroll
                        for (int u = 0; u < kU; ++u) x += to_float(l.p[u][t * 16 + r16][i]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] += x * to_float(l.c[i][(w + kWaves * j) * 16 + q * 4 + e]);
                    }
                    put(t, j, v * up);
                }
            }
        }
        if (more || (last && s_out)) {
            // behind the last row the state of the forward recurrence has not been decayed once more
            update<T, DP, DC>(S, l, more ? kChunk : r.rev ? n : n - 1, r.kv);
        }
        if (more) __syncthreads();         // everybody has read the chunk
    }
    if (last && s_out) state_store<DP, DC>(S, s_out, da, dc, r.in_a, r.in_c);
}

// sums of the query heads that share a key head: float32 [rows, HK, grp, dim] -> [rows, HK, dim] of the type
template <typename T>
__global__ __launch_bounds__(256) void group_kernel(const float* __restrict__ in, T* __restrict__ out, int64_t n, int grp, int dim) {
    for (int64_t e = blockIdx.x * (int64_t)256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        const int64_t row = e / dim, d = e % dim;
        const float* p = in + row * grp * dim + d;
        float v = 0.f;
        for (int k = 0; k < grp; ++k) v += p[(int64_t)k * dim];
        out[e] = from_float<T>(v);
    }
}

// One row: S <- l S + k v^T, out = c q^T S, in place.  A workgroup has a head's state (four columns for each of cols / 4
// lanes); the other lanes take the rows by turns.  Bound: the state, read and written (192 sequences, 16 heads of 128 x 128:
// 84 us, 4800 GB/s); of a single sequence the launch.
template <typename T>
__global__ __launch_bounds__(256) void step_kernel(Mat Q, Mat K, Mat V, const float* __restrict__ decay, float* __restrict__ state,
                                                   T* __restrict__ out, int H, int D, int DV, float scale, int cols) {
    __shared__ float sq[kMaxDim], sk[kMaxDim];
    __shared__ float part[256 * 4];
    const int64_t unit = blockIdx.x;
    const int h = (int)(unit % H);
    const int64_t b = unit / H;
    const T* q = (const T*)Q.p + b * Q.sb + h * Q.sh;
    const T* k = (const T*)K.p + b * K.sb + (int64_t)(h / K.grp) * K.sh;
    const T* v = (const T*)V.p + b * V.sb + (int64_t)(h / V.grp) * V.sh;
    for (int i = threadIdx.x; i < D; i += 256) { sq[i] = to_float(q[i]); sk[i] = to_float(k[i]); }
    const int lanes = cols / 4, c = threadIdx.x % lanes * 4, rows = 256 / lanes;
    float ve[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) ve[e] = c + e < DV ? to_float(v[c + e]) : 0.f;
    const float l = power(decay[h], 1);
    float* s = state + unit * D * DV;
    __syncthreads();
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int i = threadIdx.x / lanes; i < D; i += rows) {
        const Piece<float> x = load_piece(s + (int64_t)i * DV, (int64_t)c, (int64_t)DV, 0u);
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = l * x.f(e) + sk[i] * ve[e];
            acc[e] += sq[i] * y[e];
        }
        store_piece(s + (int64_t)i * DV, (int64_t)c, (int64_t)DV, pack<float>(y));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[threadIdx.x * 4 + e] = acc[e];
    __syncthreads();
    const int col = threadIdx.x;
    if (col < DV) {
        float o = 0.f;
        for (int i = 0; i < rows; ++i) o += part[i * cols + col];
        out[(b * H + h) * DV + col] = from_float<T>(o * scale);
    }
}

// ---------------------------------------------------------------- host

// How many segments time is cut into.  In the time that a workgroup takes for a chunk (about 4 us at 128 dimensions of 16 bits):
// a sequence of c chunks takes c; in n segments it takes c / n, and half as much again for kv_kernel, 6 for the other two
// launches and the states' way through memory, times the rounds in which the device takes all the workgroups, one for each
// of its units (two at once take twice as long: they are bound by memory).  Measured (us), 2 x 4096 rows, 16 heads of 128,
// bfloat16: n = 4 109, 6 99, 8 85, 11 92, 16 85; gradient of 4 x 2048 ragged rows: n = 1 131, 2 163, 4 159 (n = 1 with two
// workgroups for a head's columns, 172 with one); float32, 3 x 1531 ragged rows of 6 heads: n = 4 104, 14 65.
void cut(Args& a) {
    const int64_t c = (a.T + kChunk - 1) / kChunk, units = (int64_t)a.B * a.H * a.roles, cu = cu_count();
    double best = 0.0;
    a.nseg = 1;
    a.parts = 1;
    a.seg_len = (c < 1 ? 1 : c) * kChunk;
    for (int64_t n = 1; n <= c && n <= 64; ++n) {
        const int64_t each = (c + n - 1) / n, rounds = (units * n + cu - 1) / cu;
        const double cost = (double)(each * rounds) * (n > 1 ? 1.5 : 1.0) + (n > 1 ? 6.0 : 0.0);
        if (n > 1 && cost >= best) continue;
        best = cost;
        a.seg_len = each * kChunk;
        a.nseg = (int)((c + each - 1) / each);
    }
}

template <typename T, int DP, bool EVEN>
int launch(Args& a, const int (&joined)[2], int joins, hipStream_t st) {
    if (a.nseg > 1) {
        Args k = a;
        k.roles = joins;
        k.parts = 1;
        for (int i = 0; i < joins; ++i) k.r[i] = a.r[joined[i]];
        static samx::LdsGrant grant;
        if (int rc = grant.ensure((const void*)kv_kernel<T, DP, EVEN>, sizeof(LdsKv<T, DP, DP>))) return rc;
        kv_kernel<T, DP, EVEN><<<grid_of(k, a.nseg - 1), kThreads, sizeof(LdsKv<T, DP, DP>), st>>>(k);
        SAMX_LAUNCH_CHECK();
        join_kernel<DP><<<dim3((unsigned)(a.B * a.H), DP * DP / 256, (unsigned)joins), 256, 0, st>>>(k);
        SAMX_LAUNCH_CHECK();
    }
    static samx::LdsGrant grant;
    // As long as the device has a unit for every workgroup two of them share a head's columns, each with all the scores: two
    // on a unit hide each other's waits.  Where it holds more anyway the scores made twice cost more.  One against two,
    // bf16, 16 heads of 128: 8 x 512 rows 53 and 40 us, 16 x 1024 108 and 105, 32 x 1024 165 and 205; gradient of 4 x 2048
    // ragged rows 172 and 131, of 16 x 1024 233 and 277.  float32's tiles leave LDS for one on a unit: there as long as both
    // halves have a unit of their own (8 x 512 rows 145 and 91, 16 x 1024 289 and 337; gradient of 4 x 512 rows, 8 heads of 72
    // and 88, 129 and 82).
    if constexpr (DP == 128) {
        if ((int64_t)a.B * a.H * a.roles * a.nseg * (sizeof(T) == 4 ? 2 : 1) <= cu_count()) {
            a.parts = 2;
            static samx::LdsGrant half;
            if (int rc = half.ensure((const void*)mix_kernel<T, DP, 64, EVEN>, sizeof(Lds<T, DP, 64>))) return rc;
            mix_kernel<T, DP, 64, EVEN><<<grid_of(a, a.nseg), kThreads, sizeof(Lds<T, DP, 64>), st>>>(a);
            SAMX_LAUNCH_CHECK();
            return SAMX_OK;
        }
    }
    if (int rc = grant.ensure((const void*)mix_kernel<T, DP, DP, EVEN>, sizeof(Lds<T, DP, DP>))) return rc;
    mix_kernel<T, DP, DP, EVEN><<<grid_of(a, a.nseg), kThreads, sizeof(Lds<T, DP, DP>), st>>>(a);
    SAMX_LAUNCH_CHECK();
    return SAMX_OK;
}

template <typename T>
int launch_dim(Args& a, int most, const int (&joined)[2], int joins, hipStream_t st) {
    const int n = Piece<T>::kN;
    bool even = true;
    for (int i = 0; i < a.roles; ++i)
        for (const Mat* m : {&a.r[i].a, &a.r[i].b, &a.r[i].c}) {
            const int64_t st = m->st < 0 ? -m->st : m->st;
            even = even && m->dim % n == 0 && st < (int64_t(1) << 31) / ((int64_t)sizeof(T) * kChunk) - kMaxDim;
        }
    if (even) return most <= 64 ? launch<T, 64, true>(a, joined, joins, st) : launch<T, 128, true>(a, joined, joins, st);
    return most <= 64 ? launch<T, 64, false>(a, joined, joins, st) : launch<T, 128, false>(a, joined, joins, st);
}

int launch_type(int dtype, Args& a, int most, const int (&joined)[2], int joins, hipStream_t st) {
    if (dtype == kF32) return launch_dim<float>(a, most, joined, joins, st);
    if (dtype == kBF16) return launch_dim<bf16>(a, most, joined, joins, st);
    return launch_dim<f16>(a, most, joined, joins, st);
}

// a segment's state: whole tiles of the kernel that takes these dimensions
int64_t seg_size(int D, int DV) { return D <= 64 && DV <= 64 ? 64 * 64 : kMaxDim * kMaxDim; }

int check(const char* who, const samx_linattn_shape* s) {
    SAMX_REQUIRE(s, "%s: null shape", who);
    SAMX_REQUIRE(s->dtype >= 0 && s->dtype <= 2, "%s: unknown element type %d", who, s->dtype);
    SAMX_REQUIRE(s->B >= 0 && s->T >= 0 && s->T < (int64_t(1) << 31) && s->H > 0 && s->HK > 0 && s->H % s->HK == 0,
                 "%s: bad sizes (B %lld, T %lld, H %d, HK %d; H has to be a multiple of HK)", who, (long long)s->B,
                 (long long)s->T, s->H, s->HK);
    SAMX_REQUIRE(s->D > 0 && s->D <= kMaxDim && s->DV > 0 && s->DV <= kMaxDim, "%s: head dimensions %d, %d must be in [1, %d]", who,
                 s->D, s->DV, kMaxDim);
    SAMX_REQUIRE(s->B <= kMaxHeads && s->B * s->H <= kMaxHeads, "%s: B %lld times H %d is more than %lld", who, (long long)s->B, s->H,
                 (long long)kMaxHeads);
    return SAMX_OK;
}

Mat mat(const void* p, const int64_t (&st)[3], int grp, int dim) { return Mat{p, st[0], st[1], st[2], grp, dim}; }

size_t seg_bytes(const Args& a, int D, int DV) {
    return a.nseg > 1 ? (size_t)a.B * a.H * (a.nseg - 1) * seg_size(D, DV) * sizeof(float) : 0;
}

}  // namespace

extern "C" {

size_t samx_linattn_ws_bytes(const samx_linattn_shape* s) {
    if (check("samx_linattn_ws_bytes", s)) return 0;
    Args a{};
    a.roles = 1; a.B = (int)s->B; a.H = s->H; a.T = s->T;
    cut(a);
    return seg_bytes(a, s->D, s->DV) + 256;
}

int samx_linattn(const samx_linattn_shape* s, const void* q, const void* k, const void* v, const float* decay, float scale,
                 const float* state_in, const int32_t* lengths, void* out, float* state_out, void* ws, size_t ws_bytes,
                 void* stream) {
    if (int rc = check("samx_linattn", s)) return rc;
    SAMX_REQUIRE(isfinite(scale), "samx_linattn: scale must be finite");
    if (s->B == 0) return SAMX_OK;
    SAMX_REQUIRE(((q && k && v && out) || s->T == 0) && decay && state_out, "samx_linattn: null pointer");
    Args a{};
    a.roles = 1; a.B = (int)s->B; a.H = s->H; a.T = s->T; a.decay = decay; a.lengths = lengths;
    cut(a);
    const size_t need = seg_bytes(a, s->D, s->DV);
    SAMX_REQUIRE(!need || ((uintptr_t)ws & 15) == 0, "samx_linattn: the workspace has to be 16-byte aligned");
    if (need && (!ws || ws_bytes < need))
        return samx::fail(SAMX_ERR_WORKSPACE, "samx_linattn: workspace %zu < %zu", ws_bytes, need);
    const int rep = s->H / s->HK;
    a.seg_size = seg_size(s->D, s->DV);
    Role& r = a.r[0];
    r.a = mat(q, s->q, 1, s->D); r.b = mat(k, s->k, rep, s->D); r.c = mat(v, s->v, rep, s->DV);
    r.out = out; r.kv = 1.f; r.ps = scale; r.so = scale;
    r.s_in = state_in; r.in_a = s->DV; r.in_c = 1; r.s_out = state_out;
    r.seg = (float*)ws;
    const int joined[2] = {0, 0};
    return launch_type(s->dtype, a, s->D > s->DV ? s->D : s->DV, joined, 1, (hipStream_t)stream);
}

size_t samx_linattn_grad_ws_bytes(const samx_linattn_shape* s) {
    if (check("samx_linattn_grad_ws_bytes", s)) return 0;
    Args a{};
    a.roles = 3; a.B = (int)s->B; a.H = s->H; a.T = s->T;
    cut(a);
    const size_t rows = s->H == s->HK ? 0 : (size_t)s->B * s->T * s->H;
    return 2 * seg_bytes(a, s->D, s->DV) + rows * (s->D + s->DV) * sizeof(float) + 256;
}

int samx_linattn_grad(const samx_linattn_shape* s, const void* q, const void* k, const void* v, const float* decay,
                      const void* dout, float scale, const float* state_in, const float* dstate, const int32_t* lengths,
                      void* dq, void* dk, void* dv, float* dstate_in, void* ws, size_t ws_bytes, void* stream) {
    if (int rc = check("samx_linattn_grad", s)) return rc;
    SAMX_REQUIRE(isfinite(scale), "samx_linattn_grad: scale must be finite");
    if (s->B == 0) return SAMX_OK;
    SAMX_REQUIRE(((q && k && v && dout && dq && dk && dv) || s->T == 0) && decay && dstate_in, "samx_linattn_grad: null pointer");
    const size_t need = samx_linattn_grad_ws_bytes(s) - 256;
    SAMX_REQUIRE(!need || ((uintptr_t)ws & 15) == 0, "samx_linattn_grad: the workspace has to be 16-byte aligned");
    if (need && (!ws || ws_bytes < need))
        return samx::fail(SAMX_ERR_WORKSPACE, "samx_linattn_grad: workspace %zu < %zu", ws_bytes, need);
    Args a{};
    a.roles = 3; a.B = (int)s->B; a.H = s->H; a.T = s->T; a.decay = decay; a.lengths = lengths;
    cut(a);
    const int rep = s->H / s->HK, D = s->D, DV = s->DV;
    const Mat Q = mat(q, s->q, 1, D), K = mat(k, s->k, rep, D), V = mat(v, s->v, rep, DV), O = mat(dout, s->o, 1, DV);
    a.seg_size = seg_size(D, DV);
    float* seg0 = (float*)ws;
    float* seg1 = seg0 + seg_bytes(a, D, DV) / sizeof(float);
    float* heads = seg1 + seg_bytes(a, D, DV) / sizeof(float);
    const int64_t rows = s->B * s->T;
    float* dk_h = heads;
    float* dv_h = heads + rows * s->H * D;
    // dq: the forward states, transposed
    Role& x = a.r[0];
    x.a = O; x.b = V; x.c = K; x.out = dq; x.kv = 1.f; x.ps = scale; x.so = scale;
    x.s_in = state_in; x.in_a = 1; x.in_c = DV; x.seg = seg0;
    // dv: the gradient's states; the last of them, decayed, is the gradient of the state before the first row
    Role& y = a.r[1];
    y.a = K; y.b = Q; y.c = O; y.out = rep > 1 ? (void*)dv_h : dv; y.out_f32 = rep > 1; y.rev = 1;
    y.kv = scale; y.ps = scale; y.so = 1.f;
    y.s_in = dstate; y.in_a = DV; y.in_c = 1; y.s_out = dstate_in; y.seg = seg1;
    // dk: the same states, transposed
    Role& z = a.r[2];
    z = y;
    z.a = V; z.b = O; z.c = Q; z.out = rep > 1 ? (void*)dk_h : dk; z.s_out = nullptr;
    z.in_a = 1; z.in_c = DV; z.turned = 1;
    const hipStream_t st = (hipStream_t)stream;
    const int joined[2] = {0, 1};
    if (int rc = launch_type(s->dtype, a, D > DV ? D : DV, joined, 2, st)) return rc;
    if (rep > 1 && rows > 0) {
        for (int i = 0; i < 2; ++i) {
            const int dim = i ? DV : D;
            const int64_t n = rows * s->HK * dim;
            const float* in = i ? dv_h : dk_h;
            void* out = i ? dv : dk;
            const int64_t want = (n + 255) / 256, most = int64_t(1) << 23;      // (a launch of 2^32 threads leaves some out)
            const unsigned g = (unsigned)(want < most ? want : most);
            if (s->dtype == kF32) group_kernel<float><<<g, 256, 0, st>>>(in, (float*)out, n, rep, dim);
            else if (s->dtype == kBF16) group_kernel<bf16><<<g, 256, 0, st>>>(in, (bf16*)out, n, rep, dim);
            else group_kernel<f16><<<g, 256, 0, st>>>(in, (f16*)out, n, rep, dim);
            SAMX_LAUNCH_CHECK();
        }
    }
    return SAMX_OK;
}

int samx_linattn_step(const samx_linattn_shape* s, const void* q, const void* k, const void* v, const float* decay, float scale,
                      float* state, void* out, void* stream) {
    if (int rc = check("samx_linattn_step", s)) return rc;
    SAMX_REQUIRE(isfinite(scale), "samx_linattn_step: scale must be finite");
    if (s->B == 0) return SAMX_OK;
    SAMX_REQUIRE(q && k && v && decay && state && out, "samx_linattn_step: null pointer");
    const int rep = s->H / s->HK;
    const Mat Q = mat(q, s->q, 1, s->D), K = mat(k, s->k, rep, s->D), V = mat(v, s->v, rep, s->DV);
    int cols = 16;
    while (cols < s->DV && cols < 128) cols *= 2;
    const unsigned g = (unsigned)(s->B * s->H);
    const hipStream_t st = (hipStream_t)stream;
    if (s->dtype == kF32) step_kernel<float><<<g, 256, 0, st>>>(Q, K, V, decay, state, (float*)out, s->H, s->D, s->DV, scale, cols);
    else if (s->dtype == kBF16) step_kernel<bf16><<<g, 256, 0, st>>>(Q, K, V, decay, state, (bf16*)out, s->H, s->D, s->DV, scale, cols);
    else step_kernel<f16><<<g, 256, 0, st>>>(Q, K, V, decay, state, (f16*)out, s->H, s->D, s->DV, scale, cols);
    SAMX_LAUNCH_CHECK();
    return SAMX_OK;
}

}  // extern "C"
