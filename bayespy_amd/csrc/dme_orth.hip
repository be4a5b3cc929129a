// dme_orth.hip — the orthogonalised step (include/dme_hip.h, dme_orthogonal_step): X = G / |G|, then `steps` times
// X <- a X + (b S + c S S) X with S = X X'.  The polynomial p(x) = a x + b x^3 + c x^5 acts on X's singular values and
// leaves its singular vectors alone (Carlson et al. 2015 take this step's limit as the steepest descent of log-sum-exp
// losses; the quintic iteration is Bjorck and Bowie's, 1971; the coefficients that bayespy_amd/regression.py begins with, 3.4445, -4.7750 and 2.0315,
// are those that Jordan et al. 2024 publish for the Muon optimiser: steep at 0; five steps take singular values
// from 0.005 of |G| on to between 0.68 and 1.16).
//
// S is the square of the smaller side: X X' for a wide X, X' X for a tall one (then X <- a X + X (b S + c S S)); X keeps G's
// orientation.
//
// The products run on the fp16 matrix instructions, sums in 32 bits.  A value v, scaled by a power of two, is kept as fp16 pairs
// hi + lo of 22 bits together; |X| = 1 at the start and singular values stay below 3 (checked), so nothing leaves fp16's range.
//   fp32 matrices  P Q = Ph Qh + Ph Ql + Pl Qh: what is dropped is 2^-22 of a product, less than 32-bit sums of as many terms round
//                  off, at 2.5 times the rate of the fp32 instructions.  X itself stays in 32 bits beside its pair.
//   bf16 matrices  P Q = Ph Qh; X itself keeps its lo part.
// What the operands drop of X then only passes through b S + c S S, which is small where X's singular values are, instead of being
// amplified by a at every step (fp32, 16 strong directions over weak noise: 1.7e-6 of the result when X was its pair alone).
// The diagonals of S and of b S + c S S are kept out of the operands and applied in 32 bits: where singular values are alike the diagonal is
// nearly one number, and its rounding would not average out (50000 x 256 of near-flat spectrum, five steps: 3.7e-3 of the result with
// the diagonal in fp16, below 1e-3 without).
#include <math.h>

#include <atomic>
#include <type_traits>

#include "dme_products.h"

namespace {

// Powers of two that keep the operands inside fp16: X and S hold values up to 3 and 9, b S + c S S up to 60 (checked on
// the host), and what falls below 2^-14 / scale is small beside their norms.
constexpr float SCALE_X = 4096.f, SCALE_S = 4096.f, SCALE_B = 1024.f;

typedef _Float16 half;

constexpr int NORM_BLOCKS = 256;

// Sums of squares of the workgroups' shares, in 64 bits.  lines x length values, those of a line `step` apart.  One read of G: 50000 x 256 in
// bf16 takes 7 us (3.7 TB/s).
template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* G, long long sb, long long line, long long step, long long lines, long long length, double* part) {
    __shared__ double sums[4];
    const T* g = G + blockIdx.y * sb;
    double s = 0.0;
    constexpr int VEC = 16 / sizeof(T);
    typedef T tv __attribute__((ext_vector_type(VEC)));
    if (lines == 1 && step == 1 && (uintptr_t)g % 16 == 0) {  // contiguous: 16 bytes a lane
        const long long n = length / VEC;
        const tv* v = (const tv*)g;
        constexpr int DEEP = 4;  // loads on their way at a time
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += DEEP * NORM_BLOCKS * 256) {
            tv x[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; ++u) x[u] = i + u * NORM_BLOCKS * 256 < n ? v[i + u * NORM_BLOCKS * 256] : tv{};
#pragma unroll
            for (int u = 0; u < DEEP; ++u)
#pragma unroll
                for (int q = 0; q < VEC; ++q) s += (double)(float)x[u][q] * (double)(float)x[u][q];
        }
        const long long i = n * VEC + threadIdx.x;
        if (blockIdx.x == 0 && i < length) s += (double)(float)g[i] * (double)(float)g[i];
    } else {  // a workgroup's lines one after the other, or pieces of a single one
        const long long l0 = lines > 1 ? blockIdx.x : 0, ls = lines > 1 ? NORM_BLOCKS : 1;
        const long long i0 = lines > 1 ? threadIdx.x : (long long)blockIdx.x * 256 + threadIdx.x, is = lines > 1 ? 256 : NORM_BLOCKS * 256;
        for (long long l = l0; l < lines; l += ls)
            for (long long i = i0; i < length; i += is) {
                const double x = (double)(float)g[l * line + i * step];
                s += x * x;
            }
    }
    s = dme_wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

typedef half f16x8 __attribute__((ext_vector_type(8)));

// hi + lo of eight values, 16 bytes each
__device__ __forceinline__ void split8(half* hi, half* lo, const float (&v)[8]) {
    f16x8 h, l;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        h[q] = (half)v[q];
        l[q] = (half)(v[q] - (float)h[q]);
    }
    *(f16x8*)hi = h;
    *(f16x8*)lo = l;
}
// hi + lo of four values
__device__ __forceinline__ void split4(half* hi, half* lo, f32x4 v) {
    f16x4 h, l;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        h[q] = (half)v[q];
        l[q] = (half)(v[q] - (float)h[q]);
    }
    *(f16x4*)hi = h;
    *(f16x4*)lo = l;
}
__device__ __forceinline__ void split1(half* hi, half* lo, float v) {
    const half h = (half)v;
    *hi = h;
    if (lo) *lo = (half)(v - (float)h);
}

struct Matrices {
    half* X[2][2];  // [which of two][hi, lo]: [rows][ldx], read and written in turn
    float* Xf;      // fp32 matrices: X itself, scaled like its pair
    float* S;       // fp32 matrices: [m][lds], on and below the diagonal
    half* Sw[2];    // [hi, lo]: S without its diagonal; lo for fp32 matrices
    half* Bw[2];    // b S + c S S without its diagonal
    float* Sd;      // [lds]: the diagonals
    float* Bd;
    float* part;    // [split][m][lds]: pieces of S
    long long stride_x, stride_s, stride_part;  // from matrix to matrix
    long long rows, cols, ldx, m, lds;
};

// X = G / |G|, zero in the padding of its pitch.  One read of G, one write of the pairs: 50000 x 256 in bf16 takes 18 us (4.2 TB/s).
template <class T, int PARTS>
__global__ __launch_bounds__(256) void begin_kernel(const T* G, long long sb, long long rs, long long cs, const double* part, Matrices a) {
    __shared__ float tile[64][65];
    __shared__ double sums[4];
    double s = dme_wave_sum_f64(part[blockIdx.y * NORM_BLOCKS + threadIdx.x]);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const double scale = s > 0.0 || s != s ? (double)SCALE_X / sqrt(s) : 0.0;
    const T* g = G + blockIdx.y * sb;
    const long long xo = blockIdx.y * a.stride_x;
    const bool along = cs == 1 || a.cols == 1;  // neighbouring values are neighbours in G too; otherwise tiles are turned in LDS
    const long long tiles_c = (a.ldx + 63) / 64, tiles_r = (a.rows + 63) / 64;
    const int row = threadIdx.x >> 4, col = (threadIdx.x & 15) * 4;  // four neighbouring values a thread
    for (long long t = blockIdx.x; t < tiles_c * tiles_r; t += gridDim.x) {
        const long long r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;
        if (!along) {
            __syncthreads();
            for (int q = threadIdx.x >> 6; q < 64; q += 4) {
                const long long r = r0 + (threadIdx.x & 63), c = c0 + q;
                if (r < a.rows && c < a.cols) tile[threadIdx.x & 63][q] = (float)g[r * rs + c * cs];
            }
            __syncthreads();
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long long r = r0 + row + q * 16, c = c0 + col;
            if (r >= a.rows || c >= a.ldx) continue;
            f32x4 v;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                v[u] = c + u < a.cols ? (float)((double)(along ? (float)g[r * rs + (c + u) * cs] : tile[row + q * 16][col + u]) * scale) : 0.f;
            split4(a.X[0][0] + xo + r * a.ldx + c, a.X[0][1] + xo + r * a.ldx + c, v);
            if (PARTS == 2) *(f32x4*)(a.Xf + xo + r * a.ldx + c) = v;
        }
    }
}

template <class T>
struct StepArgs {
    Matrices mat;
    float a, b, c;
    int from;  // which of X is read
    T* out;    // the last step's result, or null
    long long out_batch;
    int vector;  // its rows are aligned to 16 bytes
    long long tiles_r, tiles_c, batch;
    int slices, per_split;
};

// acc = P Q' of operands in one part or two
template <int PARTS, class Tile>
__device__ __forceinline__ void multiply(Tile& t, half* const* P, const DmeOperand& p, half* const* Q, const DmeOperand& q, long long po, long long qo,
                                         long long K, char* lds, long long r0, long long c0, int s0, int s1) {
    t.clear();
    if constexpr (PARTS == 2) {
        const char* const x[3] = {(const char*)(P[0] + po), (const char*)(P[0] + po), (const char*)(P[1] + po)};
        const char* const y[3] = {(const char*)(Q[0] + qo), (const char*)(Q[1] + qo), (const char*)(Q[0] + qo)};
        t.run(p, q, x, y, K, lds, r0, c0, s0, s1);
    } else {
        t.run(DmeOperand{(const char*)(P[0] + po), p.ld, p.rows}, DmeOperand{(const char*)(Q[0] + qo), q.ld, q.rows}, K, lds, r0, c0, s0, s1);
    }
}

// The tiles of the lower triangle of a square of n x n tiles, numbered along its rows; XCDs take eighths of them (dme_xcd_order).
__device__ __forceinline__ void triangle_tile(u32 block, u32 n, long long& tr, long long& tc) {
    const u32 t = dme_xcd_order(block, n * (n + 1) / 2);
    u32 r = (u32)((__builtin_sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);  // near enough: set right below
    while (r * (r + 1) / 2 > t) --r;
    while ((r + 1) * (r + 2) / 2 <= t) ++r;
    tr = r;
    tc = t - r * (r + 1) / 2;
}

// what becomes of S[r][c] = v
template <int PARTS>
__device__ __forceinline__ void put_s(const Matrices& x, long long so, long long mo, long long r, long long c, float v) {
    const long long at = so + r * x.lds + c;
    if (PARTS == 2) x.S[at] = v;
    split1(x.Sw[0] + at, PARTS == 2 ? x.Sw[1] + at : nullptr, r == c ? 0.f : v * SCALE_S);
    if (r == c) x.Sd[mo + r] = v;
}

__device__ __forceinline__ void wave_fence() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// How a wave's part of a tile, which the matrix instructions leave in groups of four values of 16 rows, goes through LDS so that its lanes
// store 16 bytes beside each other.
template <class Tile>
struct Turn {
    static constexpr int ROWS = 16, PITCH = Tile::WTC + 4;                   // 16 rows in 32 bits at a time
    static constexpr int PER = Tile::WTC / 8, ITEMS = ROWS * PER, ITER = (ITEMS + 63) / 64;  // groups of eight values
    static constexpr int HALVES = (Tile::WTR * (Tile::WTC + 8) > Tile::WTC * (Tile::WTR + 8) ? Tile::WTR * (Tile::WTC + 8) : Tile::WTC * (Tile::WTR + 8));
    static constexpr int LDS = Tile::NW * (HALVES * 2 > ROWS * PITCH * 4 ? HALVES * 2 : ROWS * PITCH * 4);
};

// The wave's part v of the tile at (r0, c0) into a symmetric matrix of halves, and its mirror image for a tile beside the diagonal.  v is zero
// outside the m x m values; the pitch's padding gets its zeros here.
template <class Tile>
__device__ __forceinline__ void store_symmetric(char* lds, half* M, long long ld, long long m, const f16x4 (&v)[Tile::NI][Tile::NJ], long long r0,
                                                long long c0, bool mirror) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    half* mine = (half*)lds + wave * Turn<Tile>::HALVES;
    const long long r1 = r0 + wave / (Tile::TC_ / Tile::WTC) * Tile::WTR, c1 = c0 + wave % (Tile::TC_ / Tile::WTC) * Tile::WTC;
    {
        constexpr int PITCH = Tile::WTC + 8, PER = Tile::WTC / 8, ITEMS = Tile::WTR * PER;
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j)
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i) *(f16x4*)(mine + (j * 16 + c) * PITCH + i * 16 + g * 4) = v[i][j];
        wave_fence();
#pragma unroll
        for (int it = 0; it < (ITEMS + 63) / 64; ++it) {
            const int f = it * 64 + lane;
            if (ITEMS % 64 && f >= ITEMS) break;
            const long long r = r1 + f / PER, k = c1 + f % PER * 8;
            if (r < m && k < ld) *(u32q*)(M + r * ld + k) = *(const u32q*)(mine + f / PER * PITCH + f % PER * 8);
        }
        wave_fence();
    }
    if (mirror) {
        constexpr int PITCH = Tile::WTR + 8, PER = Tile::WTR / 8, ITEMS = Tile::WTC * PER;
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j)
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) mine[(i * 16 + g * 4 + q) * PITCH + j * 16 + c] = v[i][j][q];
        wave_fence();
#pragma unroll
        for (int it = 0; it < (ITEMS + 63) / 64; ++it) {
            const int f = it * 64 + lane;
            if (ITEMS % 64 && f >= ITEMS) break;
            const long long r = c1 + f / PER, k = r1 + f % PER * 8;
            if (r < m && k < ld) *(u32q*)(M + r * ld + k) = *(const u32q*)(mine + f / PER * PITCH + f % PER * 8);
        }
        wave_fence();
    }
}

// the halves of a matrix of 32-bit values, part 0 or 1 of their pairs
template <class Tile>
__device__ __forceinline__ void halves(f16x4 (&h)[Tile::NI][Tile::NJ], const f32x4 (&v)[Tile::NI][Tile::NJ], int part) {
#pragma unroll
    for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const half hi = (half)v[i][j][q];
                h[i][j][q] = part ? (half)(v[i][j][q] - (float)hi) : hi;
            }
}

// S = X X' (X' X for a tall X), the tiles on and below the diagonal; what lies above is their mirror image.  Where the tiles are
// too few for the card, k is split and join_kernel adds the pieces.  4096 x 4096 (253 tiles of 192, one to a CU) takes 73 us (940 TFLOP/s of
// the half that is made); 50000 x 256 (10 tiles in 25 pieces) 18 us and the join 5, bound by how fast one workgroup a CU takes its slices.
template <class T, int PARTS, int SIDE, bool TALL>
__global__ __launch_bounds__(SIDE >= 192 ? 512 : 256) void square_kernel(StepArgs<T> a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeSquare<half, SIDE, TALL, TALL> Tile;
    const Matrices& x = a.mat;
    const long long so = blockIdx.y * x.stride_s, mo = blockIdx.y * x.lds, xo = blockIdx.y * x.stride_x;
    const DmeOperand op{nullptr, x.ldx * 2, x.m};
    long long tr, tc;
    triangle_tile(blockIdx.x, (u32)a.tiles_r, tr, tc);
    const int s0 = (int)blockIdx.z * a.per_split;
    int s1 = s0 + a.per_split;
    s1 = s1 < a.slices ? s1 : a.slices;
    Tile t;
    multiply<PARTS>(t, x.X[a.from], op, x.X[a.from], op, xo, xo, TALL ? x.rows : x.cols, lds, tr * SIDE, tc * SIDE, s0, s1);
    constexpr float UNIT = 1.f / (SCALE_X * SCALE_X);
    const bool split = gridDim.z > 1;
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = tr * SIDE + Tile::row_of(j);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const long long c = tc * SIDE + Tile::col_of(i);
            f32x4& v = t.acc[i][j];
            v *= UNIT;
            const bool in = r < x.m && c < x.lds;
            if (split) {
                if (in) *(f32x4*)(x.part + blockIdx.y * x.stride_part + blockIdx.z * x.stride_s + r * x.lds + c) = v;
                continue;
            }
            if (PARTS == 2 && in) *(f32x4*)(x.S + so + r * x.lds + c) = v;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (in && c + q == r) x.Sd[mo + r] = v[q];
                v[q] = r < x.m && c + q < x.m && c + q != r ? v[q] * SCALE_S : 0.f;
            }
        }
    }
    if (split) return;
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        f16x4 h[Tile::NI][Tile::NJ];
        halves<Tile>(h, t.acc, part);
        store_symmetric<Tile>(lds, x.Sw[part] + so, x.lds, x.m, h, tr * SIDE, tc * SIDE, tr != tc);
    }
}

// 16 x 16 values of S on and below the diagonal, and their mirror image.
template <int PARTS>
__global__ __launch_bounds__(256) void join_kernel(Matrices x, int splits) {
    __shared__ float turn[16][17];
    const long long so = blockIdx.y * x.stride_s, mo = blockIdx.y * x.lds;
    long long tr, tc;
    triangle_tile(blockIdx.x, (u32)((x.lds + 15) / 16), tr, tc);
    const int lo = threadIdx.x & 15, hi = threadIdx.x >> 4;
    const long long r = tr * 16 + hi, c = tc * 16 + lo;
    float v = 0.f;
    if (r < x.m && c < x.m) {
        const float* at = x.part + blockIdx.y * x.stride_part + (r > c ? r * x.lds + c : c * x.lds + r);  // above the diagonal: the same sum
        const auto some = [&](int s, auto count, bool last) {  // loads without branches: all on their way at once
            constexpr int N = decltype(count)::value;
            float p[N];
#pragma unroll
            for (int u = 0; u < N; ++u) p[u] = at[(!last || s + u < splits ? s + u : s) * x.stride_s];
#pragma unroll
            for (int u = 0; u < N; ++u) v += !last || s + u < splits ? p[u] : 0.f;
        };
        int s = 0;
        for (; s + 8 <= splits; s += 8) some(s, std::integral_constant<int, 8>(), false);
        if (splits - s > 2)
            some(s, std::integral_constant<int, 8>(), true);
        else if (splits - s > 0)
            some(s, std::integral_constant<int, 2>(), true);
    }
    turn[hi][lo] = v;
    if (r < x.m && c < x.lds) put_s<PARTS>(x, so, mo, r, c, v);
    if (tr == tc) return;  // uniform
    __syncthreads();
    const long long rr = tc * 16 + hi, cc = tr * 16 + lo;
    if (rr < x.m && cc < x.lds) put_s<PARTS>(x, so, mo, rr, cc, turn[lo][hi]);
}

// (4096 x 4096: 80 us.)  B = b S + c S S.  With S = d + O (diagonal, rest): (S S)[r][c] = (O O)[r][c] + (d_r + d_c) O[r][c], + d_r^2 where r = c.
template <class T, int PARTS, int SIDE>
__global__ __launch_bounds__(SIDE >= 192 ? 512 : 256) void poly_kernel(StepArgs<T> a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeSquare<half, SIDE> Tile;
    const Matrices& x = a.mat;
    const long long so = blockIdx.y * x.stride_s, mo = blockIdx.y * x.lds;
    const DmeOperand op{nullptr, x.lds * 2, x.m};
    long long tr, tc;
    triangle_tile(blockIdx.x, (u32)a.tiles_r, tr, tc);
    Tile t;
    // S[r][c ...]; edge: in a tile on the diagonal or at the end, where S above the diagonal is what lies below it
    const auto own = [&](long long r, long long c, bool edge) {
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        if (edge && (r >= x.m || c >= x.lds)) return v;
        if (PARTS == 1) {
            const f16x4 h = *(const f16x4*)(x.Sw[0] + so + r * x.lds + c);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = (float)h[q] * (1.f / SCALE_S);
        } else if (!edge) {
            v = *(const f32x4*)(x.S + so + r * x.lds + c);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < x.m) v[q] = x.S[so + (c + q > r ? (c + q) * x.lds + r : r * x.lds + c + q)];
        }
        return v;
    };
    const bool edge = tr == tc || (tr + 1) * SIDE > x.m;  // tc <= tr
    // a small tile's own values are on their way while it is made
    constexpr bool EARLY = SIDE == 64;
    f32x4 early[EARLY ? Tile::NI : 1][EARLY ? Tile::NJ : 1];
    if constexpr (EARLY) {
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j)
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i) early[i][j] = own(tr * SIDE + Tile::row_of(j), tc * SIDE + Tile::col_of(i), edge);
    }
    multiply<PARTS>(t, x.Sw, op, x.Sw, op, so, so, x.m, lds, tr * SIDE, tc * SIDE, 0, a.slices);
    constexpr float UNIT = 1.f / (SCALE_S * SCALE_S);
    const auto finish = [&](auto at_edge) {
        constexpr bool EDGE = decltype(at_edge)::value;
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j) {
            if (!EARLY) __builtin_amdgcn_sched_barrier(0);  // or all blocks' values are loaded first, and there are no registers for them
            const long long r = tr * SIDE + Tile::row_of(j);
            const float dr = !EDGE || r < x.m ? x.Sd[mo + r] : 0.f;
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i) {
                const long long c = tc * SIDE + Tile::col_of(i);
                f32x4 s, &v = t.acc[i][j], dc = f32x4{0.f, 0.f, 0.f, 0.f};
                if constexpr (EARLY)
                    s = early[i][j];
                else
                    s = own(r, c, EDGE);
                if (!EDGE || c < x.lds) dc = *(const f32x4*)(x.Sd + mo + c);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const bool in = !EDGE || (r < x.m && c + q < x.m), on = EDGE && in && c + q == r;
                    const float sq = on ? dr : s[q], ss = v[q] * UNIT + (on ? dr * dr : (dr + dc[q]) * sq);
                    const float poly = __builtin_fmaf(a.c, ss, a.b * sq);
                    if (on) x.Bd[mo + r] = poly;
                    v[q] = in && !on ? poly * SCALE_B : 0.f;
                }
            }
        }
    };
    if (edge)
        finish(std::true_type());
    else
        finish(std::false_type());
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
        f16x4 h[Tile::NI][Tile::NJ];
        halves<Tile>(h, t.acc, part);
        store_symmetric<Tile>(lds, x.Bw[part] + so, x.lds, x.m, h, tr * SIDE, tc * SIDE, tr != tc);
    }
}

// X <- a X + B X (a X + X B for a tall X).  EU: waves that a SIMD shall have room for.  4096 x 4096 takes 122 us, 96 of them the matrix
// instructions' and most of the rest 134 MB of X read and written behind them (155 before the values went through LDS).  50000 x 256
// is bound by memory: slabs of 64 lines read X once and take 26 us for 102 MB (3.9 TB/s; tiles of 64 x 64 took 43).
template <class T, int PARTS, class Tile, bool TALL, int EU>
__global__ __launch_bounds__(Tile::NT, EU) void update_kernel(StepArgs<T> a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef Turn<Tile> Way;
    const Matrices& x = a.mat;
    const long long xo = blockIdx.y * x.stride_x, so = blockIdx.y * x.stride_s, mo = blockIdx.y * x.lds;
    const DmeOperand b{nullptr, x.lds * 2, x.m}, y{nullptr, x.ldx * 2, TALL ? x.rows : x.cols};
    half* const* X = x.X[a.from];
    long long tr, tc;
    dme_tile_of(blockIdx.x, (u32)a.tiles_r, (u32)a.tiles_c, tr, tc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const long long r0 = tr * Tile::TR_, c0 = tc * Tile::TC_;
    const long long r1 = r0 + wave / (Tile::TC_ / Tile::WTC) * Tile::WTR, c1 = c0 + wave % (Tile::TC_ / Tile::WTC) * Tile::WTC;
    // X's own values, eight of a row for a lane, 16 rows of the wave at a time: the next ones on their way while these are made
    struct Own {
        u32q at[2];  // hi, lo; fp32 matrices: X itself
    };
    const auto load = [&](int j, Own (&o)[Way::ITER]) {
#pragma unroll
        for (int it = 0; it < Way::ITER; ++it) {
            const int f = it * 64 + lane;
            const long long r = r1 + j * 16 + f / Way::PER, c = c1 + f % Way::PER * 8, at = xo + r * x.ldx + c;
            o[it].at[0] = o[it].at[1] = u32q{0, 0, 0, 0};
            if (f >= Way::ITEMS || r >= x.rows || c >= x.ldx) continue;
            o[it].at[0] = PARTS == 2 ? *(const u32q*)(x.Xf + at) : *(const u32q*)(X[0] + at);
            o[it].at[1] = PARTS == 2 ? *(const u32q*)(x.Xf + at + 4) : *(const u32q*)(X[1] + at);
        }
    };
    constexpr bool EARLY = Tile::NI * Tile::NJ <= 8;  // a small tile leaves registers for them while it is made
    Own own[Way::ITER], next[Way::ITER];
    Tile t;
    if (EARLY) load(0, own);
    if (TALL)
        multiply<PARTS>(t, X, y, x.Bw, b, xo, so, x.m, lds, r0, c0, 0, a.slices);
    else
        multiply<PARTS>(t, x.Bw, b, X, y, so, xo, x.m, lds, r0, c0, 0, a.slices);
    if (!EARLY) load(0, own);
    constexpr float UNIT = 1.f / SCALE_B;  // X's scale stays
    half *hi = x.X[a.from ^ 1][0] + xo, *lo = x.X[a.from ^ 1][1] + xo;
    float* mine = (float*)lds + wave * Way::ROWS * Way::PITCH;
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        if (j + 1 < Tile::NJ) load(j + 1, next);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) *(f32x4*)(mine + (lane & 15) * Way::PITCH + i * 16 + g * 4) = t.acc[i][j] * UNIT;
        wave_fence();
#pragma unroll
        for (int it = 0; it < Way::ITER; ++it) {
            const int f = it * 64 + lane, row = f / Way::PER, col = f % Way::PER * 8;
            const long long r = r1 + j * 16 + row, c = c1 + col, at = r * x.ldx + c;
            if (f >= Way::ITEMS || r >= x.rows || c >= x.ldx) continue;
            const f32x4 left = *(const f32x4*)(mine + row * Way::PITCH + col), right = *(const f32x4*)(mine + row * Way::PITCH + col + 4);
            const f16x8 h = __builtin_bit_cast(f16x8, own[it].at[0]), l = __builtin_bit_cast(f16x8, own[it].at[1]);
            const f32x4 o0 = __builtin_bit_cast(f32x4, own[it].at[0]), o1 = __builtin_bit_cast(f32x4, own[it].at[1]);
            f32x4 d0, d1;
            if (TALL) {  // c < ldx = lds
                d0 = *(const f32x4*)(x.Bd + mo + c);
                d1 = *(const f32x4*)(x.Bd + mo + c + 4);
            } else {
                const float d = x.Bd[mo + r];
                d0 = d1 = f32x4{d, d, d, d};
            }
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float old = PARTS == 2 ? (q < 4 ? o0[q & 3] : o1[q & 3]) : (float)h[q] + (float)l[q];
                const float d = a.a + (q < 4 ? d0[q & 3] : d1[q & 3]), product = q < 4 ? left[q & 3] : right[q & 3];
                v[q] = c + q < x.cols ? __builtin_fmaf(d, old, product) : 0.f;
            }
            if (!a.out) {
                split8(hi + at, lo + at, v);
                if (PARTS == 2) {
                    *(f32x4*)(x.Xf + xo + at) = f32x4{v[0], v[1], v[2], v[3]};
                    *(f32x4*)(x.Xf + xo + at + 4) = f32x4{v[4], v[5], v[6], v[7]};
                }
                continue;
            }
            T* to = a.out + blockIdx.y * a.out_batch + r * x.cols + c;  // the result has no padding
            if (a.vector) {
                constexpr int VEC = 16 / sizeof(T);
                typedef T tv __attribute__((ext_vector_type(VEC)));
#pragma unroll
                for (int q = 0; q < 8; q += VEC) {
                    tv w;
#pragma unroll
                    for (int u = 0; u < VEC; ++u) w[u] = (T)(v[q + u] * (1.f / SCALE_X));
                    if (c + q < x.cols) *(tv*)(to + q) = w;
                }
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c + q < x.cols) to[q] = (T)(v[q] * (1.f / SCALE_X));
            }
        }
        wave_fence();
#pragma unroll
        for (int it = 0; it < Way::ITER; ++it) own[it] = next[it];
    }
}

// ---- up to 64 singular values, up to 4096 the other way ---------------------------------------------------------------
//
// Such a matrix is all latency: the launches of a step above take 15 us (79 x 75), most of it waiting for memory once or twice each.  Here
// a step is one launch, 9 us at 1000 x 64: the products 2.6 (fp32 instructions), the rest the launch and two rounds to memory.  X lies n x 64 in 32 bits, a workgroup owns tiles of 64 lines of it; it adds up the workgroups' pieces of S, makes
// the polynomial of S for itself (64 x 64 x 64 products in LDS, fp32 instructions), updates its tiles and leaves its piece of the next S.

constexpr int SMALL = 64, SMALL_GROUPS = 16, SP = SMALL + 4;  // SP: pitch in LDS, a multiple of 16 bytes that spreads the lines over the banks

struct SmallArgs {
    float* X;             // [batch][n][64]
    const float* part;    // [batch][groups][64][64]
    float* next;
    long long n, m, tiles;
    int groups;
    float a, b, c;
    void* out;            // the last step's result, or null
    long long out_batch, out_n, out_m;
};

// Sixteen waves, each with 16 x 16 of the 64 x 64 values: a thread has one group of four of everything, so that all pieces of S are on their
// way at once.
constexpr int SMALL_THREADS = 1024;

// acc += P[r][k] Q[c][k] over 64 k.  P, Q: lines of SP values in LDS.
__device__ __forceinline__ void small_product(f32x4& acc, const float* P, const float* Q) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int k = 0; k < SMALL; k += 16)
        acc = dme_mma(*(const u32q*)(Q + ((wave & 3) * 16 + c) * SP + k + g * 4), *(const u32q*)(P + ((wave >> 2) * 16 + c) * SP + k + g * 4), acc, float());
}

// acc += X[k][r] X[k][c] over 64 lines k
__device__ __forceinline__ void small_square(f32x4& acc, const float* X) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int k = 0; k < SMALL; k += 4) {
        const float* line = X + (k + g) * SP + c;
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(line[(wave & 3) * 16], line[(wave >> 2) * 16], acc, 0, 0, 0);
    }
}

// where this lane's four values are: row, first column
__device__ __forceinline__ int small_row() { return (threadIdx.x >> 8) * 16 + (threadIdx.x & 15); }
__device__ __forceinline__ int small_col() { return (threadIdx.x >> 6 & 3) * 16 + (threadIdx.x >> 4 & 3) * 4; }

template <class T>
__global__ __launch_bounds__(SMALL_THREADS) void small_begin_kernel(const T* G, long long sb, long long sn, long long sm, const double* norm, SmallArgs a) {
    __shared__ __attribute__((aligned(16))) float tile[SMALL * SP];
    __shared__ double sums[4];
    const int tid = threadIdx.x;
    if (tid < NORM_BLOCKS) {
        const double s = dme_wave_sum_f64(norm[blockIdx.y * NORM_BLOCKS + tid]);
        if ((tid & 63) == 0) sums[tid >> 6] = s;
    }
    __syncthreads();
    const double s = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    const double scale = s > 0.0 || s != s ? 1.0 / sqrt(s) : 0.0;
    const T* g = G + blockIdx.y * sb;
    f32x4 acc = {};
    const int lo = tid & 63, hi = tid >> 6;
    for (long long t = blockIdx.x; t < a.tiles; t += a.groups) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < SMALL; u += 16) {  // neighbouring lanes along G's contiguous direction
            const int y = sm == 1 ? hi + u : lo, x = sm == 1 ? lo : hi + u;
            const long long r = t * SMALL + y;
            tile[y * SP + x] = r < a.n && x < a.m ? (float)((double)(float)g[r * sn + x * sm] * scale) : 0.f;
        }
        __syncthreads();
        *(f32x4*)(a.X + (blockIdx.y * a.tiles + t) * SMALL * SMALL + tid * 4) = *(const f32x4*)(tile + (tid >> 4) * SP + (tid & 15) * 4);
        small_square(acc, tile);
    }
    *(f32x4*)(a.next + (blockIdx.y * a.groups + blockIdx.x) * SMALL * SMALL + small_row() * SMALL + small_col()) = acc;
}

template <class T>
__global__ __launch_bounds__(SMALL_THREADS) void small_step_kernel(SmallArgs a) {
    __shared__ __attribute__((aligned(16))) float S[SMALL * SP], B[SMALL * SP], X[SMALL * SP];
    const int tid = threadIdx.x, r = small_row(), k = small_col();
    const int at = (tid >> 4) * SP + (tid & 15) * 4;  // of this thread's four values, counted along the lines
    float* mine = a.X + blockIdx.y * a.tiles * SMALL * SMALL + tid * 4;
    f32x4 x = *(const f32x4*)(mine + blockIdx.x * SMALL * SMALL);  // the first tile is on its way while S is added up
    {
        const float* part = a.part + blockIdx.y * a.groups * SMALL * SMALL + tid * 4;
        f32x4 p[SMALL_GROUPS], s = {};
#pragma unroll
        for (int u = 0; u < SMALL_GROUPS; ++u) p[u] = *(const f32x4*)(part + (u < a.groups ? u : 0) * SMALL * SMALL);
#pragma unroll
        for (int u = 0; u < SMALL_GROUPS; ++u)
            if (u < a.groups) s += p[u];
        *(f32x4*)(S + at) = s;
    }
    __syncthreads();
    {
        f32x4 acc = {};
        small_product(acc, S, S);
        const f32x4 s = *(const f32x4*)(S + r * SP + k);
        f32x4 v;
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = __builtin_fmaf(a.c, acc[q], a.b * s[q]) + (k + q == r ? a.a : 0.f);
        *(f32x4*)(B + r * SP + k) = v;
    }
    f32x4 next = {};
    for (long long t = blockIdx.x; t < a.tiles; t += a.groups) {
        if (t != blockIdx.x) x = *(const f32x4*)(mine + t * SMALL * SMALL);
        __syncthreads();  // X of the tile before is read
        *(f32x4*)(X + at) = x;
        __syncthreads();  // and B is written
        f32x4 acc = {};
        small_product(acc, X, B);  // B is symmetric
        if (a.out) {
            const long long line = t * SMALL + r;
            T* o = (T*)a.out + blockIdx.y * a.out_batch + line * a.out_n;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (line < a.n && k + q < a.m) o[(k + q) * a.out_m] = (T)acc[q];
            continue;
        }
        __syncthreads();
        *(f32x4*)(X + r * SP + k) = acc;
        __syncthreads();
        *(f32x4*)(mine + t * SMALL * SMALL) = *(const f32x4*)(X + at);
        small_square(next, X);
    }
    if (!a.out) *(f32x4*)(a.next + (blockIdx.y * a.groups + blockIdx.x) * SMALL * SMALL + r * SMALL + k) = next;
}

inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct StepPlan {
    bool small;
    long long tiles;  // small: of 64 lines
    int groups;
    long long m, n, ldx, lds;
    DmeCut square, poly, update;
    bool slab;        // the update by slabs of 64 lines
    long long norm, X[2][2], Xf, S, Sw[2], Bw[2], Sd, Bd, part, bytes;
};

StepPlan plan_of(int type, long long batch, long long rows, long long cols) {
    StepPlan p{};
    const int parts = type == DME_TYPE_BF16 ? 1 : 2;
    p.m = rows < cols ? rows : cols;
    p.n = rows < cols ? cols : rows;
    p.ldx = up(cols, 8);
    p.lds = up(p.m, 8);
    const int products = parts == 2 ? 3 : 1;
    const auto slices = [](long long k) { return (k * 2 + DME_SLICE - 1) / DME_SLICE; };
    p.square = dme_cut(p.m, p.m, slices(p.n), 2, true, 0.0, true, batch, products);
    p.poly = dme_cut(p.m, p.m, slices(p.m), 2, false, 0.0, true, batch, products);
    p.update = dme_cut(rows, cols, slices(p.m), 2, false, 0.0, false, batch, products);
    // a slab of X with all its singular values is one tile, and X is read once: where there are slabs enough for the card
    p.slab = p.m <= 256 && batch * ((p.n + 63) / 64) >= 256;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.norm = take(batch * NORM_BLOCKS * 8);
    p.small = p.m <= SMALL && p.n <= 4096;
    if (p.small) {
        p.tiles = (p.n + SMALL - 1) / SMALL;
        p.groups = (int)(p.tiles < SMALL_GROUPS ? p.tiles : SMALL_GROUPS);
        p.S = take(batch * p.tiles * SMALL * SMALL * 4);                        // X
        p.part = take(2 * batch * p.groups * SMALL * SMALL * 4);  // the pieces of S, read and written in turn
        p.bytes = at;
        return p;
    }
    for (int i = 0; i < 4; ++i) p.X[i / 2][i % 2] = take(batch * rows * p.ldx * 2);
    if (parts == 2) p.Xf = take(batch * rows * p.ldx * 4);
    if (parts == 2) p.S = take(batch * p.m * p.lds * 4);
    for (int i = 0; i < parts; ++i) {
        p.Sw[i] = take(batch * p.m * p.lds * 2);
        p.Bw[i] = take(batch * p.m * p.lds * 2);
    }
    p.Sd = take(batch * p.lds * 4);
    p.Bd = take(batch * p.lds * 4);
    if (p.square.splits > 1) p.part = take(batch * p.square.splits * p.m * p.lds * 4);
    p.bytes = at;
    return p;
}

template <class Tile, class F, class A>
int launch(F kernel, std::atomic<bool>* done, const A& a, long long tiles, int splits, hipStream_t s) {
    constexpr int bytes = Tile::LDS > Turn<Tile>::LDS ? Tile::LDS : Turn<Tile>::LDS;
    static_assert(bytes <= 160 * 1024, "more than a CU has");
    int dev = 0;
    DME_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        DME_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)a.batch, (unsigned)splits), dim3(Tile::NT), bytes, s, a);
    return DME_OK;
}

template <class T, int PARTS, int SIDE, bool TALL>
int square(StepArgs<T> a, const DmeCut& cut, hipStream_t s) {
    static std::atomic<bool> done[64];
    a.tiles_r = (a.mat.m + SIDE - 1) / SIDE;
    a.slices = (int)(((TALL ? a.mat.rows : a.mat.cols) * 2 + DME_SLICE - 1) / DME_SLICE);
    a.per_split = (a.slices + cut.splits - 1) / cut.splits;
    return launch<DmeSquare<half, SIDE>>(square_kernel<T, PARTS, SIDE, TALL>, done, a, a.tiles_r * (a.tiles_r + 1) / 2, cut.splits, s);
}

template <class T, int PARTS, int SIDE>
int poly(StepArgs<T> a, hipStream_t s) {
    static std::atomic<bool> done[64];
    a.tiles_r = (a.mat.m + SIDE - 1) / SIDE;
    a.slices = (int)((a.mat.m * 2 + DME_SLICE - 1) / DME_SLICE);
    return launch<DmeSquare<half, SIDE>>(poly_kernel<T, PARTS, SIDE>, done, a, a.tiles_r * (a.tiles_r + 1) / 2, 1, s);
}

template <class T, int PARTS, class Tile, bool TALL, int EU>
int update_by(StepArgs<T> a, hipStream_t s) {
    static std::atomic<bool> done[64];
    a.tiles_r = (a.mat.rows + Tile::TR_ - 1) / Tile::TR_;
    a.tiles_c = (a.mat.cols + Tile::TC_ - 1) / Tile::TC_;
    a.slices = (int)((a.mat.m * 2 + DME_SLICE - 1) / DME_SLICE);
    return launch<Tile>(update_kernel<T, PARTS, Tile, TALL, EU>, done, a, a.tiles_r * a.tiles_c, 1, s);
}

template <class T, int PARTS, int SIDE, bool TALL>
int update(StepArgs<T> a, hipStream_t s) {
    // small tiles: a deep pipeline where a CU has one or two of them, two buffers where it can hold five
    if constexpr (SIDE == 64)
        if ((a.mat.rows + 63) / 64 * ((a.mat.cols + 63) / 64) * a.batch > 512) return update_by<T, PARTS, DmeSquare<half, SIDE, false, !TALL, 2>, TALL, 1>(a, s);
    return update_by<T, PARTS, DmeSquare<half, SIDE, false, !TALL>, TALL, 1>(a, s);
}

template <class T, int PARTS, bool TALL>
int one_step(const StepArgs<T>& k, const StepPlan& p, hipStream_t s) {
    int rc = p.square.side == 256   ? square<T, PARTS, 256, TALL>(k, p.square, s)
             : p.square.side == 192 ? square<T, PARTS, 192, TALL>(k, p.square, s)
             : p.square.side == 128 ? square<T, PARTS, 128, TALL>(k, p.square, s)
                                    : square<T, PARTS, 64, TALL>(k, p.square, s);
    if (rc) return rc;
    if (p.square.splits > 1) {
        const long long along = (p.lds + 15) / 16;
        hipLaunchKernelGGL(join_kernel<PARTS>, dim3((unsigned)(along * (along + 1) / 2), (unsigned)k.batch), dim3(256), 0, s, k.mat, p.square.splits);
    }
    rc = p.poly.side == 256   ? poly<T, PARTS, 256>(k, s)
         : p.poly.side == 192 ? poly<T, PARTS, 192>(k, s)
         : p.poly.side == 128 ? poly<T, PARTS, 128>(k, s)
                              : poly<T, PARTS, 64>(k, s);
    if (rc) return rc;
    if (p.slab) {
        if constexpr (TALL)
            return p.m <= 128 ? update_by<T, PARTS, DmeTile<half, 64, 128, 4, 2, false, false, 2>, true, 4>(k, s)
                              : update_by<T, PARTS, DmeTile<half, 64, 256, 4, 2, false, false, 2>, true, 4>(k, s);
        else
            return p.m <= 128 ? update_by<T, PARTS, DmeTile<half, 128, 64, 8, 1, false, true, 2>, false, 4>(k, s)
                              : update_by<T, PARTS, DmeTile<half, 256, 64, 8, 1, false, true, 2>, false, 4>(k, s);
    }
    return p.update.side == 256   ? update<T, PARTS, 256, TALL>(k, s)
           : p.update.side == 192 ? update<T, PARTS, 192, TALL>(k, s)
           : p.update.side == 128 ? update<T, PARTS, 128, TALL>(k, s)
                                  : update<T, PARTS, 64, TALL>(k, s);
}

template <class T, int PARTS>
int run(const T* G, long long sb, long long rs, long long cs, long long batch, long long rows, long long cols, int steps, double a, double b, double c,
        T* out, char* ws, const StepPlan& p, hipStream_t s) {
    const bool tall = rows > cols;
    StepArgs<T> k{};
    Matrices& x = k.mat;
    for (int i = 0; i < 4; ++i) x.X[i / 2][i % 2] = (half*)(ws + p.X[i / 2][i % 2]);
    for (int i = 0; i < PARTS; ++i) {
        x.Sw[i] = (half*)(ws + p.Sw[i]);
        x.Bw[i] = (half*)(ws + p.Bw[i]);
    }
    x.Xf = (float*)(ws + p.Xf);
    x.S = (float*)(ws + p.S);
    x.Sd = (float*)(ws + p.Sd);
    x.Bd = (float*)(ws + p.Bd);
    x.part = (float*)(ws + p.part);
    x.rows = rows;
    x.cols = cols;
    x.ldx = p.ldx;
    x.m = p.m;
    x.lds = p.lds;
    x.stride_x = rows * p.ldx;
    x.stride_s = p.m * p.lds;
    x.stride_part = p.square.splits * p.m * p.lds;
    k.a = (float)a;
    k.b = (float)b;
    k.c = (float)c;
    k.out_batch = rows * cols;
    k.vector = cols * sizeof(T) % 16 == 0 && (uintptr_t)out % 16 == 0;
    k.batch = batch;
    double* part = (double*)(ws + p.norm);
    // the norm is read along G's contiguous direction, as one line where G has no gaps
    const bool turn = rs == 1 && cs != 1;
    const long long line = turn ? cs : rs, step = turn ? rs : cs, lines = turn ? cols : rows, length = turn ? rows : cols;
    const bool whole = step == 1 && line == length;
    hipLaunchKernelGGL(norm_kernel<T>, dim3(NORM_BLOCKS, (unsigned)batch), dim3(256), 0, s, G, sb, line, step, whole ? 1 : lines,
                       whole ? lines * length : length, part);
    if (p.small) {
        SmallArgs y{};
        float* pieces[2] = {(float*)(ws + p.part), (float*)(ws + p.part) + batch * p.groups * SMALL * SMALL};
        y.X = (float*)(ws + p.S);
        y.next = pieces[0];
        y.n = p.n;
        y.m = p.m;
        y.tiles = p.tiles;
        y.groups = p.groups;
        y.a = (float)a;
        y.b = (float)b;
        y.c = (float)c;
        y.out_batch = rows * cols;
        y.out_n = tall ? cols : 1;
        y.out_m = tall ? 1 : cols;
        const dim3 grid((unsigned)p.groups, (unsigned)batch);
        hipLaunchKernelGGL(small_begin_kernel<T>, grid, dim3(SMALL_THREADS), 0, s, G, sb, tall ? rs : cs, tall ? cs : rs, part, y);
        for (int i = 0; i < steps; ++i) {
            y.part = pieces[i & 1];
            y.next = pieces[(i & 1) ^ 1];
            y.out = i + 1 < steps ? nullptr : out;
            hipLaunchKernelGGL(small_step_kernel<T>, grid, dim3(SMALL_THREADS), 0, s, y);
        }
        DME_HIP_CHECK(hipGetLastError());
        return DME_OK;
    }
    const long long tiles = (p.ldx + 63) / 64 * ((rows + 63) / 64);
    hipLaunchKernelGGL((begin_kernel<T, PARTS>), dim3((unsigned)(tiles < 4096 ? tiles : 4096), (unsigned)batch), dim3(256), 0, s, G, sb, rs, cs, part, x);
    for (int i = 0; i < steps; ++i) {
        k.from = i & 1;
        k.out = i + 1 < steps ? nullptr : out;
        const int rc = tall ? one_step<T, PARTS, true>(k, p, s) : one_step<T, PARTS, false>(k, p, s);
        if (rc) return rc;
    }
    DME_HIP_CHECK(hipGetLastError());
    return DME_OK;
}

// Whether the polynomial keeps singular values that begin in [0, 1] (|X| = 1) where the operands can hold them.
bool in_range(int steps, double a, double b, double c) {
    if (!isfinite(a) || !isfinite(b) || !isfinite(c)) return false;
    double top = 1.0;
    for (int i = 0; i < steps && i < 64; ++i) {
        double next = 0.0;
        for (int q = 0; q <= 512; ++q) {
            const double x = top * q / 512.0, even = x * x * (b + c * x * x), y = fabs(x * (a + even));
            if (fabs(even) > 60.0) return false;
            next = y > next ? y : next;
        }
        if (next > 3.0) return false;
        top = next;
    }
    return true;
}

int check(int type, int64_t batch, int64_t rows, int64_t cols) {
    DME_REQUIRE(type == DME_TYPE_BF16 || type == DME_TYPE_F32, "the matrix is bf16 or fp32");
    DME_REQUIRE(batch >= 0 && batch <= 65535 && rows >= 1 && cols >= 1, "bad shape: %lld x %lld x %lld", (long long)batch, (long long)rows, (long long)cols);
    DME_REQUIRE(rows <= (1ll << 28) && cols <= (1ll << 28) && (rows < cols ? rows : cols) <= (1ll << 16), "shape out of range");
    return DME_OK;
}

}  // namespace

extern "C" int64_t dme_orthogonal_step_workspace_bytes(int type, int64_t batch, int64_t rows, int64_t cols) {
    if (check(type, batch, rows, cols) != DME_OK) return -1;
    return plan_of(type, batch, rows, cols).bytes;
}

extern "C" int dme_orthogonal_step(const void* G, int64_t batch_stride, int64_t row_stride, int64_t col_stride, int type, int64_t batch, int64_t rows,
                                   int64_t cols, int steps, double a, double b, double c, void* out, void* ws, int64_t ws_bytes, void* stream) {
    const int rc = check(type, batch, rows, cols);
    if (rc) return rc;
    DME_REQUIRE(steps >= 1 && steps <= 64, "steps must be in 1..64");
    DME_REQUIRE(in_range(steps, a, b, c), "the coefficients let singular values leave [0, 3]");
    if (batch == 0) return DME_OK;
    DME_REQUIRE(G != nullptr && out != nullptr, "null pointer");
    const StepPlan p = plan_of(type, batch, rows, cols);
    if (ws == nullptr || (uintptr_t)ws % 256 != 0 || ws_bytes < p.bytes)
        return dme_set_error(DME_ERR_WORKSPACE, "workspace of %lld bytes, aligned to 256, needed", p.bytes);
    if (type == DME_TYPE_BF16)
        return run<__bf16, 1>((const __bf16*)G, batch_stride, row_stride, col_stride, batch, rows, cols, steps, a, b, c, (__bf16*)out, (char*)ws, p,
                              (hipStream_t)stream);
    return run<float, 2>((const float*)G, batch_stride, row_stride, col_stride, batch, rows, cols, steps, a, b, c, (float*)out, (char*)ws, p,
                         (hipStream_t)stream);
}
