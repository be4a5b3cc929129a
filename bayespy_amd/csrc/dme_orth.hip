// dme_orth.hip — the orthogonalised step (include/dme_hip.h, dme_orthogonal_step): X = G / |G|, then `steps` times
// X <- a X + (b S + c S S) X with S = X X'.  The polynomial p(x) = a x + b x^3 + c x^5 acts on X's singular values and
// leaves its singular vectors alone (Carlson et al. 2015 take this step's limit as the steepest descent of log-sum-exp
// losses; the quintic iteration is Bjorck and Bowie's, 1971).
//
// X is kept m x n with m <= n (G transposed where it is tall), so S is the smaller square.  Operands of the products are
// fp16 for bf16 matrices, scaled by powers of two, and X itself stays in 32 bits beside them: what fp16 drops of X then
// only passes through (b S + c S S), which is small where X's singular values are, instead of being amplified by a at every
// step.  For fp32 matrices everything is fp32.
#include <math.h>

#include <atomic>

#include "dme_products.h"

namespace {

// Powers of two that keep the operands inside fp16: X and S hold values up to 3 and 9, b S + c S S up to 60 (checked on
// the host), and what falls below 2^-14 / scale is small beside their norms.
template <class W>
struct Scale {
    static constexpr float X = 1.f, S = 1.f, B = 1.f;
};
template <>
struct Scale<_Float16> {
    static constexpr float X = 4096.f, S = 4096.f, B = 1024.f;
};

constexpr int NORM_BLOCKS = 64;

template <class T>
__global__ __launch_bounds__(256) void norm_kernel(const T* G, long long sb, long long rs, long long cs, long long m, long long n, double* part) {
    __shared__ double sums[4];
    const T* g = G + blockIdx.y * sb;
    double s = 0.0;
    const long long total = m * n;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const long long r = i / n, c = i - r * n;
        const double v = (double)(float)g[r * rs + c * cs];
        s += v * v;
    }
    s = dme_wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) part[blockIdx.y * NORM_BLOCKS + blockIdx.x] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

template <class W>
struct Matrices {
    float* X;      // [m][ldn] in 32 bits; for fp32 matrices also the operand
    W* Xw;         // [m][ldn]
    W* Xt[2];      // [n][ldm]
    float* S;      // [m][ldm]
    W* Sw;         // [m][ldm]
    W* Bw;         // [m][ldm]
    long long stride_x, stride_t, stride_s;  // from matrix to matrix
    long long m, n, ldm, ldn;
};

// X = G / |G| and its transpose, zero in the padding of their pitches.
template <class T, class W>
__global__ __launch_bounds__(256) void begin_kernel(const T* G, long long sb, long long rs, long long cs, const double* part, Matrices<W> a) {
    __shared__ float tile[64][65];
    double s = 0.0;
    for (int i = 0; i < NORM_BLOCKS; ++i) s += part[blockIdx.y * NORM_BLOCKS + i];
    const double scale = s > 0.0 || s != s ? 1.0 / sqrt(s) : 0.0;
    const T* g = G + blockIdx.y * sb;
    const long long xo = blockIdx.y * a.stride_x, to = blockIdx.y * a.stride_t;
    const int lo = threadIdx.x & 63, hi = threadIdx.x >> 6;
    const bool along = cs == 1;  // neighbouring lanes read neighbouring values
    const long long tiles_c = (a.ldn + 63) / 64, tiles_r = (a.ldm + 63) / 64;
    for (long long t = blockIdx.x; t < tiles_c * tiles_r; t += gridDim.x) {
        const long long r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;
        for (int q = hi; q < 64; q += 4) {
            const int y = along ? q : lo, x = along ? lo : q;
            const long long r = r0 + y, c = c0 + x;
            tile[y][x] = r < a.m && c < a.n ? (float)((double)(float)g[r * rs + c * cs] * scale) : 0.f;
        }
        __syncthreads();
        for (int q = hi; q < 64; q += 4) {
            const long long r = r0 + q, c = c0 + lo;
            if (r < a.m && c < a.ldn) {
                a.X[xo + r * a.ldn + c] = tile[q][lo];
                if ((void*)a.Xw != (void*)a.X) a.Xw[xo + r * a.ldn + c] = (W)(tile[q][lo] * Scale<W>::X);
            }
            const long long rr = r0 + lo, cc = c0 + q;
            if (cc < a.n && rr < a.ldm) a.Xt[0][to + cc * a.ldm + rr] = (W)(tile[lo][q] * Scale<W>::X);
        }
        __syncthreads();
    }
}

enum { MAKE_S, MAKE_B, MAKE_X, MAKE_LAST };

template <class T, class W>
struct StepArgs {
    Matrices<W> mat;
    const char* zeros;
    float a, b, c;
    int from;  // which of Xt is read
    T* out;    // MAKE_LAST
    long long out_batch, out_row, out_col;
    long long tiles_r, tiles_c;
};

// One of a step's three products with what follows it: S = X X', B = b S + c S S, X = a X + B X.
template <class T, class W, int MAKE>
__global__ __launch_bounds__(256, 2) void step_kernel(StepArgs<T, W> a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<W, 128, 128, 2, 2> Tile;
    const Matrices<W>& x = a.mat;
    const long long xo = blockIdx.y * x.stride_x, to = blockIdx.y * x.stride_t, so = blockIdx.y * x.stride_s;
    constexpr long long size = sizeof(W);
    DmeOperands op;
    if (MAKE == MAKE_S) {
        const char* p = (const char*)(x.Xw + xo);
        op = DmeOperands{p, p, x.ldn * size, x.ldn * size, x.m, x.m, x.ldn * size, a.zeros};
    } else if (MAKE == MAKE_B) {
        const char* p = (const char*)(x.Sw + so);
        op = DmeOperands{p, p, x.ldm * size, x.ldm * size, x.m, x.m, x.ldm * size, a.zeros};
    } else {
        op = DmeOperands{(const char*)(x.Bw + so), (const char*)(x.Xt[a.from] + to), x.ldm * size, x.ldm * size, x.m, x.n, x.ldm * size, a.zeros};
    }
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    Tile t;
    t.run(op, lds, tr * 128, tc * 128, 0, (int)((op.kbytes + DME_SLICE - 1) / DME_SLICE));
    typedef Scale<W> K;
    const long long width = MAKE == MAKE_S || MAKE == MAKE_B ? x.m : x.n, pitch = MAKE == MAKE_S || MAKE == MAKE_B ? x.ldm : x.ldn;
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = tr * 128 + Tile::row_of(j);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const long long c = tc * 128 + Tile::col_of(i);
            if (c >= pitch) continue;
            f32x4 v = t.acc[i][j];
            if (MAKE == MAKE_S) {
                if (r >= x.m) continue;
                v *= 1.f / (K::X * K::X);
            } else if (MAKE == MAKE_B) {
                if (r >= x.m) continue;
                const f32x4 s = *(const f32x4*)(x.S + so + r * pitch + c);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = __builtin_fmaf(a.c, v[q] * (1.f / (K::S * K::S)), a.b * s[q]);
            } else if (r < x.m) {
                const f32x4 s = *(const f32x4*)(x.X + xo + r * pitch + c);
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = __builtin_fmaf(a.a, s[q], v[q] * (1.f / (K::B * K::X)));
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = r < x.m && c + q < width ? v[q] : 0.f;
            if (MAKE == MAKE_S) {
                *(f32x4*)(x.S + so + r * pitch + c) = v;
                if ((void*)x.Sw != (void*)x.S) dme_store4(x.Sw + so + r * pitch + c, v * K::S);
            } else if (MAKE == MAKE_B) {
                dme_store4(x.Bw + so + r * pitch + c, v * K::B);
            } else if (MAKE == MAKE_X) {
                if (r < x.m) {
                    *(f32x4*)(x.X + xo + r * pitch + c) = v;
                    if ((void*)x.Xw != (void*)x.X) dme_store4(x.Xw + xo + r * pitch + c, v * K::X);
                }
                if (r < x.ldm) {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (c + q < x.n) x.Xt[a.from ^ 1][to + (c + q) * x.ldm + r] = (W)(v[q] * K::X);
                }
            } else if (r < x.m) {
                T* o = a.out + blockIdx.y * a.out_batch + r * a.out_row + c * a.out_col;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (c + q < x.n) o[q * a.out_col] = (T)v[q];
            }
        }
    }
}

__global__ void zeros_kernel(u32* p) { p[threadIdx.x] = 0; }

inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }

struct StepPlan {
    long long m, n, ldm, ldn;
    long long zeros, norm, X, Xw, Xt[2], S, Sw, Bw, bytes;
};

StepPlan plan_of(int type, long long batch, long long rows, long long cols) {
    StepPlan p{};
    const bool half = type == DME_TYPE_BF16;
    const long long size = half ? 2 : 4, per = 16 / size;
    p.m = rows < cols ? rows : cols;
    p.n = rows < cols ? cols : rows;
    p.ldm = up(p.m, per);
    p.ldn = up(p.n, per);
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.zeros = take(256);
    p.norm = take(batch * NORM_BLOCKS * 8);
    p.X = take(batch * p.m * p.ldn * 4);
    p.Xw = half ? take(batch * p.m * p.ldn * 2) : p.X;
    for (int i = 0; i < 2; ++i) p.Xt[i] = take(batch * p.n * p.ldm * size);
    p.S = take(batch * p.m * p.ldm * 4);
    p.Sw = half ? take(batch * p.m * p.ldm * 2) : p.S;
    p.Bw = take(batch * p.m * p.ldm * size);
    p.bytes = at;
    return p;
}

template <class T, class W, int MAKE>
int launch(StepArgs<T, W> a, long long batch, hipStream_t s) {
    typedef DmeTile<W, 128, 128, 2, 2> Tile;
    a.tiles_r = (a.mat.m + 127) / 128;
    a.tiles_c = ((MAKE == MAKE_S || MAKE == MAKE_B ? a.mat.m : a.mat.n) + 127) / 128;
    static std::atomic<bool> done[64];
    int dev = 0;
    DME_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        DME_HIP_CHECK(hipFuncSetAttribute((const void*)step_kernel<T, W, MAKE>, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * Tile::STAGE));
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    hipLaunchKernelGGL((step_kernel<T, W, MAKE>), dim3((unsigned)(a.tiles_r * a.tiles_c), (unsigned)batch), dim3(256), 2 * Tile::STAGE, s, a);
    return DME_OK;
}

template <class T, class W>
int run(const T* G, long long sb, long long rs, long long cs, long long batch, long long rows, long long cols, int steps, double a, double b, double c,
        T* out, char* ws, const StepPlan& p, hipStream_t s) {
    const bool tall = rows > cols;
    const long long row = tall ? cs : rs, col = tall ? rs : cs;  // of X
    StepArgs<T, W> k{};
    Matrices<W>& x = k.mat;
    x.X = (float*)(ws + p.X);
    x.Xw = (W*)(ws + p.Xw);
    for (int i = 0; i < 2; ++i) x.Xt[i] = (W*)(ws + p.Xt[i]);
    x.S = (float*)(ws + p.S);
    x.Sw = (W*)(ws + p.Sw);
    x.Bw = (W*)(ws + p.Bw);
    x.m = p.m;
    x.n = p.n;
    x.ldm = p.ldm;
    x.ldn = p.ldn;
    x.stride_x = p.m * p.ldn;
    x.stride_t = p.n * p.ldm;
    x.stride_s = p.m * p.ldm;
    k.zeros = ws + p.zeros;
    k.a = (float)a;
    k.b = (float)b;
    k.c = (float)c;
    k.out = out;
    k.out_batch = rows * cols;
    k.out_row = tall ? 1 : cols;
    k.out_col = tall ? cols : 1;
    hipLaunchKernelGGL(zeros_kernel, dim3(1), dim3(64), 0, s, (u32*)(ws + p.zeros));
    double* part = (double*)(ws + p.norm);
    // the norm is read in G's own order
    if (tall)
        hipLaunchKernelGGL(norm_kernel<T>, dim3(NORM_BLOCKS, (unsigned)batch), dim3(256), 0, s, G, sb, rs, cs, rows, cols, part);
    else
        hipLaunchKernelGGL(norm_kernel<T>, dim3(NORM_BLOCKS, (unsigned)batch), dim3(256), 0, s, G, sb, row, col, p.m, p.n, part);
    const long long tiles = (p.ldn + 63) / 64 * ((p.ldm + 63) / 64);
    hipLaunchKernelGGL((begin_kernel<T, W>), dim3((unsigned)(tiles < 4096 ? tiles : 4096), (unsigned)batch), dim3(256), 0, s, G, sb, row, col, part, x);
    for (int i = 0; i < steps; ++i) {
        k.from = i & 1;
        int rc = launch<T, W, MAKE_S>(k, batch, s);
        if (!rc) rc = launch<T, W, MAKE_B>(k, batch, s);
        if (!rc) rc = i + 1 < steps ? launch<T, W, MAKE_X>(k, batch, s) : launch<T, W, MAKE_LAST>(k, batch, s);
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
        return run<__bf16, _Float16>((const __bf16*)G, batch_stride, row_stride, col_stride, batch, rows, cols, steps, a, b, c, (__bf16*)out, (char*)ws, p,
                                     (hipStream_t)stream);
    return run<float, float>((const float*)G, batch_stride, row_stride, col_stride, batch, rows, cols, steps, a, b, c, (float*)out, (char*)ws, p,
                             (hipStream_t)stream);
}
