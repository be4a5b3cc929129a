// dme_regress.hip — the log loss of count rows under a linear predictor, and its gradient (include/dme_hip.h,
// dme_log_loss*).  z = H W' + b is never kept: a workgroup makes a tile of it on the matrix cores, reduces it to a
// maximum, a sum of exponentials and what the row's counts need of it, and drops it.  The gradient makes the tiles of a
// piece of the columns again, turns them into d loss / d z, and multiplies that piece with W and H.
//
// With l = log sum_k exp z_k and T the row's total (DirichletEstimation/dirichletMultinomialEstimation.py:16-48 is the
// Dirichlet likelihood with one z for all rows):
//     loss = F(l, T) - sum_k F(z_k, x_k)         d loss / d z_k = exp(z_k - l) G(l, T) - G(z_k, x_k)
//     multinomial  F = x z, G = x;               Dirichlet  F = lgamma(e^z + x) - lgamma(e^z), G = dF/dz
// so both likelihoods share the pass over the columns; F and G are needed at the counts alone, in 64 bits.
#include <math.h>

#include <atomic>

#include "dme_products.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr long long ROW_BLOCK = 16384;             // rows worked on at a time
constexpr long long PIECE_BYTES = 512ll << 20;     // of d loss / d z held at a time

enum { LABELS = DME_ROWS_LABELS, CSR = DME_ROWS_CSR, DENSE = DME_ROWS_DENSE };

// 1 / (12 v) - 1 / (360 v^3) + 1 / (1260 v^5): what Stirling's formula leaves of lgamma (v >= 16: below 3e-12).
__device__ double stirling_rest(double v) {
    const double i = 1.0 / v, q = i * i;
    return i * (1.0 / 12.0 - q * (1.0 / 360.0 - q * (1.0 / 1260.0)));
}

// F of the Dirichlet likelihood: sum_{n < x} log(e^z + n).  The first 16 terms are multiplied out (n = 0 gives z itself,
// however small e^z), the rest is a difference of two Stirling formulas written without their cancelling parts.
__device__ __attribute__((noinline)) double dirichlet_f(double z, double x) {
    if (!(x > 0.0)) return 0.0 * x;
    if (z > 60.0) return x * z;  // e^z + n is e^z in 64 bits
    const double a = exp(z);
    double r = z, prod = 1.0;
    const int head = x < 16.0 ? (int)x : 16;
    for (int n = 1; n < head; ++n) {
        prod *= a + n;
        if ((n & 3) == 0) {
            r += log(prod);
            prod = 1.0;
        }
    }
    r += log(prod);
    if (x > 16.0) {
        const double y = a + 16.0, h = x - 16.0;
        r += h * log(y) + ((y + h - 0.5) * log1p(h / y) - h) + (stirling_rest(y + h) - stirling_rest(y));
    }
    return r;
}

// G = dF/dz = sum_{n < x} e^z / (e^z + n), each term as 1 / (1 + n e^-z) so that neither end of z overflows.
__device__ __attribute__((noinline)) double dirichlet_g(double z, double x) {
    if (!(x > 0.0)) return 0.0 * x;
    if (z > 60.0) return x;
    const double q = exp(-z);
    double g = 1.0;
    const int head = x < 16.0 ? (int)x : 16;
    for (int n = 1; n < head; ++n) g += 1.0 / (1.0 + n * q);
    if (x > 16.0) {
        const double a = exp(z), y = a + 16.0, h = x - 16.0, i = 1.0 / y, j = 1.0 / (y + h);
        const double psi = log1p(h / y) + 0.5 * (i - j) + (i * i - j * j) * (1.0 / 12.0) - (i * i * i * i - j * j * j * j) * (1.0 / 120.0);
        g += a * psi;
    }
    return g;
}

__device__ __forceinline__ double f_of(int likelihood, double z, double x) {
    if (likelihood == DME_LIKELIHOOD_DIRICHLET) return dirichlet_f(z, x);
    return x == 0.0 ? 0.0 : x * z;
}
__device__ __forceinline__ double g_of(int likelihood, double z, double x) {
    return likelihood == DME_LIKELIHOOD_DIRICHLET ? dirichlet_g(z, x) : x;
}

// Reductions over the 16 lanes that share a row.
template <int CTRL>
__device__ __forceinline__ float dpp_f32(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, dpp_f32<DME_DPP_QUAD_XOR1>(v));
    v = fmaxf(v, dpp_f32<DME_DPP_QUAD_XOR2>(v));
    v = fmaxf(v, dpp_f32<DME_DPP_HALF_MIRROR>(v));
    return fmaxf(v, dpp_f32<DME_DPP_MIRROR>(v));
}
__device__ __forceinline__ float sum16(float v) {
    v += dpp_f32<DME_DPP_QUAD_XOR1>(v);
    v += dpp_f32<DME_DPP_QUAD_XOR2>(v);
    v += dpp_f32<DME_DPP_HALF_MIRROR>(v);
    return v + dpp_f32<DME_DPP_MIRROR>(v);
}
__device__ __forceinline__ double sum16(double v) {
    v += dme_dpp_f64<DME_DPP_QUAD_XOR1>(v);
    v += dme_dpp_f64<DME_DPP_QUAD_XOR2>(v);
    v += dme_dpp_f64<DME_DPP_HALF_MIRROR>(v);
    return v + dme_dpp_f64<DME_DPP_MIRROR>(v);
}

// The count rows of one block of rows, as the kernels take them.
struct Rows {
    const long long* rowptr;  // CSR: of the block's first row
    const int* col;
    const int* val;
    long long nnz;
    const long long* labels;  // LABELS: of the block's first row
    const char* X;            // DENSE: of the block's first row
    long long ldx;
    int elem;                 // DENSE: bytes of a count
};

__device__ __forceinline__ long long row_begin(const Rows& rows, long long r) {
    const long long p = rows.rowptr[r];
    return p < 0 ? 0 : p < rows.nnz ? p : rows.nnz;
}

__device__ __forceinline__ int count_at(const Rows& rows, long long r, long long k) {
    return rows.elem == 2 ? (int)((const unsigned short*)rows.X)[r * rows.ldx + k] : ((const int*)rows.X)[r * rows.ldx + k];
}

struct TileArgs {
    DmeOperand h, w;
    long long D;
    const char* zeros;
    long long tiles_r, tiles_c;
    int slices;
    const float* bias;
    long long nb;      // rows of the block
    long long K;
    long long column;  // first column of the piece
    Rows rows;
    // forward
    f32x2* part;       // [tile][nb]: largest z log2 e, sum of 2^(z log2 e - that)
    double* part_f;    // DENSE: [tile][nb]: sum F(z, x)
    double* part_t;    // DENSE: [tile][nb]: sum x, NaN where a count is negative
    float* entry_z;    // CSR: [nnz], LABELS: [nb]: z at the counts
    int likelihood;
    // backward
    const float* lse2;     // [nb]: l * log2 e
    const float* coef;     // [nb]: weight * G(l, T) * 2^(lse2 - l log2 e)
    const float* weight;   // [nb]
    void* dz;              // [nb][lddz]
    long long lddz;
    float* dbias;          // [tiles_r][K] or null
};

// bias of four columns; columns from K on get -inf, which leaves them out of every sum
__device__ __forceinline__ f32x4 bias_of(const TileArgs& a, long long k) {
    typedef f32x4 f32x4_u __attribute__((aligned(4)));
    f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k + 4 <= a.K) {
        if (a.bias) b = *(const f32x4_u*)(a.bias + k);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) b[q] = k + q < a.K ? (a.bias ? a.bias[k + q] : 0.f) : -INFINITY;
    }
    return b;
}

__device__ __forceinline__ float dot_step(const u32q& h, const u32q& w, float s, __bf16) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        s = __builtin_fmaf(__builtin_bit_cast(float, h[q] << 16), __builtin_bit_cast(float, w[q] << 16), s);
        s = __builtin_fmaf(__builtin_bit_cast(float, h[q] & 0xffff0000u), __builtin_bit_cast(float, w[q] & 0xffff0000u), s);
    }
    return s;
}
__device__ __forceinline__ float dot_step(const u32q& h, const u32q& w, float s, float) {
    // the whole vector is cast: a cast of one element reads the first one, whatever its index (clang 22)
    const f32x4 x = __builtin_bit_cast(f32x4, h), y = __builtin_bit_cast(f32x4, w);
#pragma unroll
    for (int q = 0; q < 4; ++q) s = __builtin_fmaf(x[q], y[q], s);
    return s;
}

// z at a row's counts: a scalar product for each, 16 lanes an entry.  There are few of them beside the N K values of z that the
// tiles make (and drop), so they are made once more here instead of being looked for in every tile.  `first` of every
// `step` entries, by the caller's 16-lane group.
template <class T, int KIND>
__device__ __forceinline__ void entries_of(const TileArgs& a, long long r, int first, int step) {
    const int sub = threadIdx.x & 15;
    const int chunks = (int)((a.D * (long long)sizeof(T) + 15) / 16);
    const u32q* h = (const u32q*)(a.h.at + r * a.h.ld);
    const long long p0 = KIND == CSR ? row_begin(a.rows, r) : r, p1 = KIND == CSR ? row_begin(a.rows, r + 1) : r + 1;
    for (long long e = p0 + first; e < p1; e += step) {
        const long long k = KIND == CSR ? (long long)a.rows.col[e] : a.rows.labels[r];
        if (k < 0 || k >= a.K) continue;  // the row's 16 lanes together
        const u32q* w = (const u32q*)(a.w.at + k * a.w.ld);
        float s = 0.f;
        for (int q = sub; q < chunks; q += 16) s = dot_step(h[q], w[q], s, T());
        s = sum16(s);
        if (sub == 0) a.entry_z[e] = s + (a.bias ? a.bias[k] : 0.f);
    }
}

template <class T, int KIND>
__global__ __launch_bounds__(256) void entry_kernel(TileArgs a) {
    const long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r < a.nb) entries_of<T, KIND>(a, r, (threadIdx.x & 63) >> 4, 4);
}

// Tiles of z, reduced where the matrix instructions left them: a lane has NJ rows and 4 NI columns of each.
//   forward   largest exponent and sum of exponentials of each row: 2^(z log2 e - M) with M = max z log2 e rounded to 32 bits,
//             the same M that the sum is kept with, so that its rounding costs nothing
//   backward  2^(z log2 e - l log2 e) coef, rounded to T (the gradient's one rounding before its products), and the columns' sums
//             of the unrounded values.  The counts are not looked at: patch_kernel puts them in.
// With TR = 16 (few rows) the weights are read once from memory and each workgroup beyond the tiles makes one row's z at
// its counts, so that a call has two launches.
template <class T, int TR, int TC, int WR, int WC, int KIND, bool BACKWARD>
__global__ __launch_bounds__(WR * WC * 64) void tile_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, TR, TC, WR, WC> Tile;
    if (TR == 16 && !BACKWARD && blockIdx.x >= a.tiles_r * a.tiles_c) {
        if constexpr (KIND != DENSE) entries_of<T, KIND>(a, blockIdx.x - a.tiles_r * a.tiles_c, threadIdx.x >> 4, WR * WC * 4);
        return;
    }
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    const long long r0 = tr * TR, c0 = tc * TC, k0 = a.column + c0;
    Tile t;
    t.run(a.h, a.w, a.D, a.zeros, lds, r0, c0, 0, a.slices);
    const int tid = threadIdx.x, g = (tid & 63) >> 4, wc = (tid >> 6) % WC, wr = (tid >> 6) / WC;
#pragma unroll
    for (int i = 0; i < Tile::NI; ++i) {
        const f32x4 b = bias_of(a, k0 + Tile::col_of(i));
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j) t.acc[i][j] += b;
    }
    if (!BACKWARD) {
        f32x2* seen = (f32x2*)lds;  // [WC][TR]
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = fmaxf(m, t.acc[i][j][q]);
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            m *= LOG2E;
            const float base = m == -INFINITY ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) s += __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][q], LOG2E, -base));
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (g == 0) seen[wc * TR + wr * Tile::WTR + j * 16 + (tid & 15)] = f32x2{m, s};
        }
        __syncthreads();
        if (tid < TR && r0 + tid < a.nb) {
            f32x2 v = seen[tid];
#pragma unroll
            for (int w = 1; w < WC; ++w) {
                const f32x2 o = seen[w * TR + tid];
                const float m = fmaxf(v[0], o[0]), base = m == -INFINITY ? 0.f : m;
                v[1] = v[1] * __builtin_amdgcn_exp2f(v[0] - base) + o[1] * __builtin_amdgcn_exp2f(o[0] - base);
                v[0] = m;
            }
            a.part[tc * a.nb + r0 + tid] = v;
        }
        return;
    }
    float l2[Tile::NJ], cf[Tile::NJ];
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = r0 + Tile::row_of(j);
        l2[j] = r < a.nb ? a.lse2[r] : INFINITY;
        cf[j] = r < a.nb ? a.coef[r] : 0.f;
    }
    float* sums = (float*)lds;  // [WR][TC]
#pragma unroll
    for (int i = 0; i < Tile::NI; ++i) {
        f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j) {
            f32x4 d;
#pragma unroll
            for (int q = 0; q < 4; ++q) d[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(t.acc[i][j][q], LOG2E, -l2[j])) * cf[j];
            const long long r = r0 + Tile::row_of(j);
            if (r < a.nb) {
                sum += d;
                dme_store4((T*)a.dz + r * a.lddz + c0 + Tile::col_of(i), d);
            }
        }
        if (a.dbias) {
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[q] = sum16(sum[q]);
            if ((tid & 15) == 0) *(f32x4*)(sums + wr * TC + Tile::col_of(i)) = sum;
        }
    }
    if (a.dbias) {
        __syncthreads();
        for (int c = tid; c < TC; c += Tile::NT) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WR; ++w) v += sums[w * TC + c];
            if (k0 + c < a.K) a.dbias[tr * a.K + k0 + c] = v;
        }
    }
}

constexpr int DT = 128;      // columns of a tile with dense counts
constexpr int ZP = DT + 4;   // its pitch in LDS (a multiple of 16 bytes that spreads the rows over the banks)

// Tiles of z with a dense matrix of counts: every value of z may meet a count, so the tile lies in LDS in 32 bits, where a row's
// 16 lanes read it beside the counts (both in order of the columns) in a loop short enough for F and G.
template <class T, int TR, bool BACKWARD>
__global__ __launch_bounds__(256, 2) void dense_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, TR, DT, (TR == 16 ? 1 : 2), (TR == 16 ? 4 : 2)> Tile;
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    const long long r0 = tr * TR, c0 = tc * DT, k0 = a.column + c0;
    float* z = (float*)lds;
    {
        Tile t;
        t.run(a.h, a.w, a.D, a.zeros, lds, r0, c0, 0, a.slices);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const int c = Tile::col_of(i);
            const f32x4 b = bias_of(a, k0 + c);
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j) *(f32x4*)(z + Tile::row_of(j) * ZP + c) = t.acc[i][j] + b;
        }
    }
    __syncthreads();
    const int tid = threadIdx.x, sub = tid & 15;
    if (!BACKWARD) {
#pragma unroll 1
        for (int row = tid >> 4; row < TR; row += 16) {
            const long long r = r0 + row;
            if (r >= a.nb) break;  // all of a row's lanes, and rows only ascend
            const float* zr = z + row * ZP;
            const f32x4 u = *(const f32x4*)(zr + sub * 4), w = *(const f32x4*)(zr + 64 + sub * 4);
            const float m = LOG2E * max16(fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))));
            const float base = m == -INFINITY ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                s += __builtin_amdgcn_exp2f(__builtin_fmaf(u[q], LOG2E, -base)) + __builtin_amdgcn_exp2f(__builtin_fmaf(w[q], LOG2E, -base));
            s = sum16(s);
            double f = 0.0, t = 0.0;
            bool bad = false;
#pragma unroll 1
            for (int q = 0; q < 8; ++q) {
                const int c = q * 16 + sub;
                if (k0 + c >= a.K) break;
                const int x = count_at(a.rows, r, k0 + c);
                if (x < 0) bad = true;
                if (x > 0) {
                    t += (double)x;
                    f += f_of(a.likelihood, (double)zr[c], (double)x);
                }
            }
            f = sum16(f);
            t = sum16(bad ? __builtin_nan("") : t);
            if (sub == 0) {
                a.part[tc * a.nb + r] = f32x2{m, s};
                a.part_f[tc * a.nb + r] = f;
                a.part_t[tc * a.nb + r] = t;
            }
        }
        return;
    }
    T* dz = (T*)a.dz;
#pragma unroll 1
    for (int row = tid >> 4; row < TR; row += 16) {
        const long long r = r0 + row;
        const bool real = r < a.nb;
        const float l2 = real ? a.lse2[r] : INFINITY, cf = real ? a.coef[r] : 0.f, weight = real ? a.weight[r] : 0.f;
        float* zr = z + row * ZP;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int c = h * 64 + sub * 4;
            const f32x4 v = *(const f32x4*)(zr + c);
            f32x4 d;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                d[q] = real ? __builtin_amdgcn_exp2f(__builtin_fmaf(v[q], LOG2E, -l2)) * cf : 0.f;
                if (real && k0 + c + q < a.K) {
                    const int x = count_at(a.rows, r, k0 + c + q);
                    if (x != 0) d[q] -= weight * (float)g_of(a.likelihood, (double)v[q], (double)x);
                }
            }
            *(f32x4*)(zr + c) = d;
            if (real) dme_store4(dz + r * a.lddz + c0 + c, d);
        }
    }
    if (!a.dbias) return;
    __syncthreads();
    const int c = tid & 127, half = tid >> 7;
    float sum = 0.f;
#pragma unroll 4
    for (int row = half * (TR / 2); row < (half + 1) * (TR / 2); ++row) sum += z[row * ZP + c];
    __syncthreads();
    if (half) z[c] = sum;
    __syncthreads();
    if (!half && k0 + c < a.K) a.dbias[tr * a.K + k0 + c] = sum + z[c];
}

// Reductions over the lanes that share a row: 16, or a workgroup's 256.
template <int LANES>
struct Together {
    double* shared;  // [4] (LANES == 256)
    template <class F>
    __device__ __forceinline__ double over_waves(double v, F f) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
        __syncthreads();
        return f(f(shared[0], shared[1]), f(shared[2], shared[3]));
    }
    __device__ __forceinline__ double sum(double v) {
        if constexpr (LANES == 16) return sum16(v);
        return over_waves(dme_wave_sum_f64(v), [](double x, double y) { return x + y; });
    }
    __device__ __forceinline__ float max(float v) {
        v = max16(v);
        if constexpr (LANES == 16) return v;
        v = fmaxf(v, __shfl_xor(v, 16));
        v = fmaxf(v, __shfl_xor(v, 32));
        return (float)over_waves((double)v, [](double x, double y) { return x > y ? x : y; });
    }
};

struct RowArgs {
    long long nb, K;
    int tiles, kind, likelihood;
    const f32x2* part;
    const double* part_f;
    const double* part_t;
    const float* entry_z;
    Rows rows;
    const float* weights;  // [nb] or null
    float* loss;           // [nb]
    float* lse2;           // [nb] or null: no gradient is wanted
    float* coef;
    float* weight;
    float* entry_g;        // CSR: [nnz], LABELS: [nb]: weight * G(z, x)
    u32* largest;          // the largest |entry_g| so far, as the bits of a float
};

// The row's pieces become l, the loss, and what the gradient needs of them, in 64 bits.  CSR rows are checked here: columns
// strictly ascending and below K, no negative count, rowptr in order; a row that breaks this has total NaN.
template <int LANES>
__global__ __launch_bounds__(256) void row_kernel(RowArgs a) {
    __shared__ double shared[4];
    Together<LANES> row{shared};
    const int sub = threadIdx.x % LANES;
    const long long r = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    const bool real = r < a.nb;
    const long long rr = real ? r : a.nb - 1;
    float m = -INFINITY;
    for (int t = sub; t < a.tiles; t += LANES) m = fmaxf(m, a.part[t * a.nb + rr][0]);
    m = row.max(m);
    const float base = m == -INFINITY ? 0.f : m;
    double s = 0.0, f = 0.0, total = 0.0;
    for (int t = sub; t < a.tiles; t += LANES) {
        const f32x2 p = a.part[t * a.nb + rr];
        s += (double)p[1] * (double)__builtin_amdgcn_exp2f(p[0] - base);
    }
    s = row.sum(s);
    const double exact2 = s == 0.0 ? -INFINITY : (double)base + log2(s), lse = exact2 * (1.0 / (double)LOG2E);
    const float weight = a.weights ? a.weights[rr] : 1.f;
    float most = 0.f;
    if (a.kind == DENSE) {
        for (int t = sub; t < a.tiles; t += LANES) {
            f += a.part_f[t * a.nb + rr];
            total += a.part_t[t * a.nb + rr];
        }
        f = row.sum(f);
        total = row.sum(total);
    } else if (a.kind == CSR) {
        const long long q0 = a.rows.rowptr[rr], q1 = a.rows.rowptr[rr + 1];
        const long long e0 = row_begin(a.rows, rr), e1 = row_begin(a.rows, rr + 1);
        bool bad = q0 < 0 || q1 < q0 || q1 > a.rows.nnz;
        for (long long e = e0 + sub; e < e1; e += LANES) {
            const int k = a.rows.col[e], x = a.rows.val[e], before = e > e0 ? a.rows.col[e - 1] : -1;
            if (k <= before || k >= a.K || x < 0) {
                bad = true;
                continue;
            }
            const double z = (double)a.entry_z[e];
            total += (double)x;
            f += f_of(a.likelihood, z, (double)x);
            if (a.lse2 && real) {
                const float v = weight * (float)g_of(a.likelihood, z, (double)x);
                a.entry_g[e] = v;
                most = fmaxf(most, fabsf(v));
            }
        }
        f = row.sum(f);
        total = row.sum(bad ? __builtin_nan("") : total);
    } else {
        const long long k = a.rows.labels[rr];
        total = k < 0 ? 0.0 : k < a.K ? 1.0 : __builtin_nan("");
        f = k >= 0 && k < a.K ? (double)a.entry_z[rr] : 0.0;  // F(z, 1) = z, G(z, 1) = 1 in both likelihoods
        if (a.lse2 && real && sub == 0) {
            a.entry_g[r] = weight;
            most = k >= 0 ? fabsf(weight) : 0.f;
        }
    }
    if (a.lse2 && a.kind != DENSE) {
        most = row.max(most);
        if (LANES == 16) {  // one atomic a wave
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
        }
        if ((threadIdx.x & 63) == 0 && most > 0.f && (LANES == 16 || threadIdx.x == 0)) atomicMax(a.largest, __builtin_bit_cast(u32, most));
    }
    if (!real || sub != 0) return;
    a.loss[r] = total == 0.0 ? 0.f : (float)(f_of(a.likelihood, lse, total) - f);
    if (!a.lse2) return;
    // what lse2's rounding to 32 bits drops goes into the coefficient
    const float l2 = total == 0.0 ? INFINITY : (float)exact2;
    a.lse2[r] = l2;
    a.coef[r] = total == 0.0 ? 0.f : (float)((double)weight * g_of(a.likelihood, lse, total) * exp2((double)l2 - exact2));
    a.weight[r] = weight;
}

struct PatchArgs {
    long long nb, K, column, width;
    Rows rows;
    const float* entry_z;
    const float* entry_g;
    const float* lse2;
    const float* coef;
    void* dz;
    long long lddz;
    long long* fixed;  // [K] or null
    const u32* largest;
    int headroom;      // bits that the sum of all entries may need above one entry
};

// The exponent of the fixed-point sums of entry_g: the largest one takes 62 - headroom bits, whatever its size.
__device__ __forceinline__ int fixed_shift(const u32* largest, int headroom) {
    const float v = __builtin_bit_cast(float, *largest);
    return 62 - headroom - (v > 0.f && v < INFINITY ? ilogbf(v) + 1 : 0);
}

// d loss / d z at the counts: the tiles' value made again, minus G, in its place.  What dbias needs of G is added up in fixed
// point, 64 bits wide: sums of whole numbers do not depend on their order.  16 lanes a row.
template <class T, int KIND>
__global__ __launch_bounds__(256) void patch_kernel(PatchArgs a) {
    const int sub = threadIdx.x & 15;
    const long long r = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (r >= a.nb) return;
    const float l2 = a.lse2[r], cf = a.coef[r];
    const int shift = a.fixed ? fixed_shift(a.largest, a.headroom) : 0;
    const long long p0 = KIND == CSR ? row_begin(a.rows, r) : r, p1 = KIND == CSR ? row_begin(a.rows, r + 1) : r + 1;
    for (long long e = p0 + sub; e < p1; e += 16) {
        const long long k = KIND == CSR ? (long long)a.rows.col[e] : a.rows.labels[r];
        const long long c = k - a.column;
        if (c < 0 || c >= a.width || k >= a.K) continue;
        const float g = a.entry_g[e];
        ((T*)a.dz)[r * a.lddz + c] = (T)(__builtin_amdgcn_exp2f(__builtin_fmaf(a.entry_z[e], LOG2E, -l2)) * cf - g);
        if (a.fixed && __builtin_isfinite(g)) atomicAdd((u64*)(a.fixed + k), (u64)llrint(ldexp((double)g, shift)));
    }
}

struct ProductArgs {
    DmeOperand p, q;
    long long k;
    const char* zeros;
    long long tiles_r, tiles_c;
    int slices, per_split;
    float* part;        // [split][R][ldpart], or null: the result goes to out in T
    long long ldpart, split_stride;
    int add;            // part holds sums already
    void* out;
    long long ldout;
    int vector;         // out's rows are aligned to four values
};

// out = P Q' (R x C), Q k-major, in T, or as 32-bit pieces where k is split over workgroups or over launches.
template <class T, int SIDE, bool PK>
__global__ __launch_bounds__(SIDE == 256 ? 512 : 256) void product_kernel(ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, SIDE, SIDE, (SIDE == 256 ? 4 : 2), 2, PK, true> Tile;
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    const int s0 = (int)blockIdx.y * a.per_split;
    int s1 = s0 + a.per_split;
    s1 = s1 < a.slices ? s1 : a.slices;
    Tile t;
    t.run(a.p, a.q, a.k, a.zeros, lds, tr * SIDE, tc * SIDE, s0, s1);
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = tr * SIDE + Tile::row_of(j);
        if (r >= a.p.rows) continue;
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const long long c = tc * SIDE + Tile::col_of(i);
            if (c >= a.q.rows) continue;
            f32x4 v = t.acc[i][j];
            if (a.part) {  // the pitch is a multiple of four: a row's last vector stays inside it
                f32x4* to = (f32x4*)(a.part + blockIdx.y * a.split_stride + r * a.ldpart + c);
                if (a.add) v += *to;
                *to = v;
            } else if (a.vector) {
                dme_store4((T*)a.out + r * a.ldout + c, v);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (c + q < a.q.rows) ((T*)a.out)[r * a.ldout + c + q] = (T)v[q];
            }
        }
    }
}

// out [R][C] = the sum of `splits` pieces, in their order.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(const float* part, long long ldpart, long long split_stride, int splits, long long R, long long C,
                                                   T* out) {
    const long long n = R * C;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const long long r = i / C, c = i - r * C;
        const float* at = part + r * ldpart + c;
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += at[s * split_stride];
        out[i] = (T)v;
    }
}

// dbias [K] (+)= the row tiles' sums, in their order, minus the counts' (fixed, null for dense rows).
__global__ __launch_bounds__(256) void bias_kernel(const float* part, long long tiles, long long K, const long long* fixed, const u32* largest,
                                                   int headroom, int add, float* dbias) {
    const long long k = (long long)blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    double v = add ? (double)dbias[k] : 0.0;
    for (long long t = 0; t < tiles; ++t) v += (double)part[t * K + k];
    if (fixed) v -= ldexp((double)fixed[k], -fixed_shift(largest, headroom));
    dbias[k] = (float)v;
}

__global__ void zero_kernel(u32* p, long long words) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (long long)gridDim.x * blockDim.x) p[i] = 0;
}

inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }

// Everything a call decides before its first launch.
struct Plan {
    int size;                 // bytes of a value
    bool pack_h, pack_w;      // the operand is copied with a pitch of whole 16-byte chunks first
    long long dpad;           // k of the first product in a packed operand
    long long nb;             // rows of a block
    int side;                 // of the tiles of z: 256, 128, or 16 rows x 128 columns
    long long tile_rows, tile_cols, tiles;
    long long chunk;          // columns of a piece of d loss / d z
    DmeCut cut_w, cut_h;
    bool part_w, part_h;      // the products leave 32-bit pieces
    long long ldpart;
    int headroom;
    // places in the workspace
    long long zeros, h, w, part, part_f, part_t, entry_z, entry_g, lse2, coef, weight, dbias, fixed, dz, pw, ph, bytes;
    long long zero_words;     // from the beginning: the zeros, the largest entry, the fixed-point sums
};

Plan make_plan(const void* H, long long ldh, const void* W, long long ldw, int type, long long N, long long K, long long D,
               const dme_count_rows_t* rows, bool gradient) {
    Plan p{};
    p.size = type == DME_TYPE_BF16 ? 2 : 4;
    const auto loose = [&](const void* at, long long ld) {
        return ((uintptr_t)at | (uintptr_t)(ld * p.size) | (uintptr_t)(D * p.size)) % 16 != 0;
    };
    p.pack_h = loose(H, ldh);
    p.pack_w = loose(W, ldw);
    p.dpad = up(D, 16 / p.size);
    p.nb = N < 1 ? 1 : N < ROW_BLOCK ? N : ROW_BLOCK;
    const long long slices = (D * p.size + DME_SLICE - 1) / DME_SLICE;
    p.side = p.nb <= 16 ? 16 : rows->kind == DENSE ? 128 : dme_cut(p.nb, K, slices, p.size, false, 4.0).side < 256 ? 128 : 256;
    p.tile_rows = p.side;
    p.tile_cols = p.side == 16 ? 128 : p.side;
    p.tiles = (K + p.tile_cols - 1) / p.tile_cols;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.zeros = take(256);
    if (gradient && rows->kind != DENSE) p.fixed = take(K * 8);
    p.zero_words = at / 4;
    if (p.pack_h) p.h = take(p.nb * p.dpad * p.size);
    if (p.pack_w) p.w = take(K * p.dpad * p.size);
    p.part = take(p.tiles * p.nb * 8);
    if (rows->kind == CSR) {
        p.entry_z = take(rows->nnz * 4);
    } else if (rows->kind == DENSE) {
        p.part_f = take(p.tiles * p.nb * 8);
        p.part_t = take(p.tiles * p.nb * 8);
    } else {
        p.entry_z = take(p.nb * 4);
    }
    if (gradient) {
        if (rows->kind != DENSE) p.entry_g = take((rows->kind == CSR ? rows->nnz : p.nb) * 4);
        for (p.headroom = 1; (rows->kind == CSR ? rows->nnz : N) >> p.headroom; ++p.headroom) {}
        p.lse2 = take(p.nb * 4);
        p.coef = take(p.nb * 4);
        p.weight = take(p.nb * 4);
        p.dbias = take((p.nb + p.tile_rows - 1) / p.tile_rows * K * 4);
        long long c = PIECE_BYTES / (p.nb * p.size) / p.tile_cols;
        if (c < 1) c = 1;
        if (c > p.tiles) c = p.tiles;
        const long long pieces = (p.tiles + c - 1) / c;
        p.chunk = (p.tiles + pieces - 1) / pieces * p.tile_cols;  // pieces of like width
        p.dz = take(p.nb * p.chunk * p.size);
        p.ldpart = up(D, 4);
        p.cut_w = dme_cut(p.chunk < K ? p.chunk : K, D, (p.nb * p.size + DME_SLICE - 1) / DME_SLICE, p.size, true);
        p.cut_h = dme_cut(p.nb, D, (p.chunk * p.size + DME_SLICE - 1) / DME_SLICE, p.size, true);
        p.part_w = p.cut_w.splits > 1 || N > p.nb;
        p.part_h = p.cut_h.splits > 1 || p.chunk < p.tiles * p.tile_cols;
        if (p.part_w) p.pw = take((long long)p.cut_w.splits * K * p.ldpart * 4);
        if (p.part_h) p.ph = take((long long)p.cut_h.splits * p.nb * p.ldpart * 4);
    }
    p.bytes = at;
    return p;
}

template <class F>
int set_lds(std::atomic<bool>* done, F kernel, int bytes) {
    int dev = 0;
    DME_HIP_CHECK(hipGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
        DME_HIP_CHECK(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_release);
    }
    return DME_OK;
}

template <class T, int TR, int TC, int WR, int WC, int KIND, bool BACKWARD>
int launch_tile(const TileArgs& a, hipStream_t s) {
    typedef DmeTile<T, TR, TC, WR, WC> Tile;
    static_assert(2 * Tile::STAGE >= WC * TR * 8 && 2 * Tile::STAGE >= WR * TC * 4, "the reductions use the tiles' LDS");
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, tile_kernel<T, TR, TC, WR, WC, KIND, BACKWARD>, 2 * Tile::STAGE);
    if (rc) return rc;
    const long long blocks = a.tiles_r * a.tiles_c + (TR == 16 && !BACKWARD ? a.nb : 0);
    hipLaunchKernelGGL((tile_kernel<T, TR, TC, WR, WC, KIND, BACKWARD>), dim3((unsigned)blocks), dim3(Tile::NT), 2 * Tile::STAGE, s, a);
    return DME_OK;
}

template <class T, int TR, bool BACKWARD>
int launch_dense(const TileArgs& a, hipStream_t s) {
    typedef DmeTile<T, TR, DT, (TR == 16 ? 1 : 2), (TR == 16 ? 4 : 2)> Tile;
    constexpr int bytes = 2 * Tile::STAGE > TR * ZP * 4 ? 2 * Tile::STAGE : TR * ZP * 4;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, dense_kernel<T, TR, BACKWARD>, bytes);
    if (rc) return rc;
    hipLaunchKernelGGL((dense_kernel<T, TR, BACKWARD>), dim3((unsigned)(a.tiles_r * a.tiles_c)), dim3(256), bytes, s, a);
    return DME_OK;
}

template <class T, int KIND, bool BACKWARD>
int launch_side(const TileArgs& a, int side, hipStream_t s) {
    if (side == 256) return launch_tile<T, 256, 256, 4, 2, KIND, BACKWARD>(a, s);
    if (side == 128) return launch_tile<T, 128, 128, 2, 2, KIND, BACKWARD>(a, s);
    return launch_tile<T, 16, 128, 1, 4, KIND, BACKWARD>(a, s);
}

// The tiles of z (the workgroups that make z at the counts are part of the forward launch where rows are few).
template <class T, bool BACKWARD>
int tiles_of_z(const TileArgs& a, int kind, int side, hipStream_t s) {
    if (kind == DENSE) return side == 16 ? launch_dense<T, 16, BACKWARD>(a, s) : launch_dense<T, 128, BACKWARD>(a, s);
    if (BACKWARD || side != 16) return launch_side<T, LABELS, BACKWARD>(a, side, s);  // the kind does not matter
    return kind == CSR ? launch_side<T, CSR, false>(a, 16, s) : launch_side<T, LABELS, false>(a, 16, s);
}

template <class T, int SIDE, bool PK>
int launch_product(const ProductArgs& a, int splits, hipStream_t s) {
    typedef DmeTile<T, SIDE, SIDE, (SIDE == 256 ? 4 : 2), 2, PK, true> Tile;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, product_kernel<T, SIDE, PK>, 2 * Tile::STAGE);
    if (rc) return rc;
    hipLaunchKernelGGL((product_kernel<T, SIDE, PK>), dim3((unsigned)(a.tiles_r * a.tiles_c), (unsigned)splits), dim3(Tile::NT), 2 * Tile::STAGE, s, a);
    return DME_OK;
}

template <class T, bool PK>
int product(ProductArgs a, const DmeCut& cut, hipStream_t s) {
    a.tiles_r = (a.p.rows + cut.side - 1) / cut.side;
    a.tiles_c = (a.q.rows + cut.side - 1) / cut.side;
    a.slices = (int)((a.k * (long long)sizeof(T) + DME_SLICE - 1) / DME_SLICE);
    a.per_split = (a.slices + cut.splits - 1) / cut.splits;
    if (cut.side == 256) return launch_product<T, 256, PK>(a, cut.splits, s);
    if (cut.side == 128) return launch_product<T, 128, PK>(a, cut.splits, s);
    return launch_product<T, 64, PK>(a, cut.splits, s);
}

struct Call {
    const void* H;
    long long ldh;
    const void* W;
    long long ldw;
    const float* bias;
    long long N, K, D;
    const dme_count_rows_t* rows;
    int likelihood;
    const float* weights;
    float* loss;
    void* dH;
    void* dW;
    float* dbias;
    char* ws;
};

template <class T>
int work(const Call& c, const Plan& p, bool gradient, hipStream_t s) {
    const int size = p.size, kind = c.rows->kind;
    char* ws = c.ws;
    DmeOperand w{(const char*)c.W, c.ldw * size, c.K};
    if (p.pack_w) {
        hipLaunchKernelGGL(dme_pack_kernel<T>, dim3(dme_blocks(c.K * p.dpad, 1024, 8192)), dim3(256), 0, s, (const T*)c.W, c.ldw, c.K, c.D,
                           (T*)(ws + p.w), p.dpad);
        w = DmeOperand{ws + p.w, p.dpad * size, c.K};
    }
    u32* largest = (u32*)(ws + p.zeros) + 32;  // the zeros are its first bytes
    long long* fixed = gradient && kind != DENSE && c.dbias ? (long long*)(ws + p.fixed) : nullptr;
    for (long long n0 = 0; n0 < c.N; n0 += p.nb) {
        const long long nb = c.N - n0 < p.nb ? c.N - n0 : p.nb;
        // each block of rows has fixed-point sums of its own: their scale is the block's
        hipLaunchKernelGGL(zero_kernel, dim3(dme_blocks(p.zero_words, 1024, 1024)), dim3(256), 0, s, (u32*)ws, p.zero_words);
        DmeOperand h{(const char*)c.H + n0 * c.ldh * size, c.ldh * size, nb};
        if (p.pack_h) {
            hipLaunchKernelGGL(dme_pack_kernel<T>, dim3(dme_blocks(nb * p.dpad, 1024, 8192)), dim3(256), 0, s, (const T*)h.at, c.ldh, nb, c.D,
                               (T*)(ws + p.h), p.dpad);
            h = DmeOperand{ws + p.h, p.dpad * size, nb};
        }
        TileArgs a{};
        a.h = h;
        a.w = w;
        a.D = c.D;
        a.zeros = ws + p.zeros;
        a.tiles_r = (nb + p.tile_rows - 1) / p.tile_rows;
        a.tiles_c = p.tiles;
        a.slices = (int)((c.D * size + DME_SLICE - 1) / DME_SLICE);
        a.bias = c.bias;
        a.nb = nb;
        a.K = c.K;
        a.likelihood = c.likelihood;
        Rows& rows = a.rows;
        if (kind == CSR) {
            rows.rowptr = (const long long*)c.rows->rowptr + n0;
            rows.col = (const int*)c.rows->colidx;
            rows.val = (const int*)c.rows->vals;
            rows.nnz = c.rows->nnz;
        } else if (kind == DENSE) {
            rows.elem = c.rows->elem;
            rows.ldx = c.rows->ld;
            rows.X = (const char*)c.rows->X + n0 * rows.ldx * rows.elem;
        } else {
            rows.labels = (const long long*)c.rows->labels + n0;
        }
        a.part = (f32x2*)(ws + p.part);
        a.part_f = (double*)(ws + p.part_f);
        a.part_t = (double*)(ws + p.part_t);
        a.entry_z = (float*)(ws + p.entry_z);
        if (kind == CSR && p.side != 16)
            hipLaunchKernelGGL((entry_kernel<T, CSR>), dim3((unsigned)((nb + 3) / 4)), dim3(256), 0, s, a);
        else if (kind == LABELS && p.side != 16)
            hipLaunchKernelGGL((entry_kernel<T, LABELS>), dim3((unsigned)((nb + 3) / 4)), dim3(256), 0, s, a);
        int rc = tiles_of_z<T, false>(a, kind, p.side, s);
        if (rc) return rc;
        RowArgs ra{};
        ra.nb = nb;
        ra.K = c.K;
        ra.tiles = (int)p.tiles;
        ra.kind = kind;
        ra.likelihood = c.likelihood;
        ra.part = a.part;
        ra.part_f = a.part_f;
        ra.part_t = a.part_t;
        ra.entry_z = a.entry_z;
        ra.rows = rows;
        ra.loss = c.loss + n0;
        if (gradient) {
            ra.weights = c.weights ? c.weights + n0 : nullptr;
            ra.lse2 = (float*)(ws + p.lse2);
            ra.coef = (float*)(ws + p.coef);
            ra.weight = (float*)(ws + p.weight);
            ra.entry_g = (float*)(ws + p.entry_g);
            ra.largest = largest;
        }
        if (nb <= 1024)  // too few rows to fill the card with 16 lanes each
            hipLaunchKernelGGL(row_kernel<256>, dim3((unsigned)nb), dim3(256), 0, s, ra);
        else
            hipLaunchKernelGGL(row_kernel<16>, dim3((unsigned)((nb + 15) / 16)), dim3(256), 0, s, ra);
        if (!gradient) continue;
        a.lse2 = ra.lse2;
        a.coef = ra.coef;
        a.weight = ra.weight;
        a.dz = ws + p.dz;
        a.dbias = c.dbias ? (float*)(ws + p.dbias) : nullptr;
        for (long long k0 = 0; k0 < c.K; k0 += p.chunk) {
            const long long width = c.K - k0 < p.chunk ? c.K - k0 : p.chunk;
            a.column = k0;
            a.w = DmeOperand{w.at + k0 * w.ld, w.ld, width};
            a.tiles_c = (width + p.tile_cols - 1) / p.tile_cols;
            a.lddz = a.tiles_c * p.tile_cols;
            rc = tiles_of_z<T, true>(a, kind, p.side, s);
            if (rc) return rc;
            if (kind != DENSE) {
                PatchArgs pa{nb, c.K, k0, width, rows, a.entry_z, ra.entry_g, ra.lse2, ra.coef, a.dz, a.lddz, fixed, largest, p.headroom};
                if (kind == CSR)
                    hipLaunchKernelGGL((patch_kernel<T, CSR>), dim3((unsigned)((nb + 15) / 16)), dim3(256), 0, s, pa);
                else
                    hipLaunchKernelGGL((patch_kernel<T, LABELS>), dim3((unsigned)((nb + 15) / 16)), dim3(256), 0, s, pa);
            }
            const char* dz = (const char*)a.dz;
            ProductArgs m{};  // dW of the piece = dz' H
            m.p = DmeOperand{dz, a.lddz * size, width};
            m.q = DmeOperand{h.at, h.ld, c.D};
            m.k = nb;
            m.zeros = a.zeros;
            if (p.part_w) {
                m.part = (float*)(ws + p.pw) + k0 * p.ldpart;
                m.ldpart = p.ldpart;
                m.split_stride = c.K * p.ldpart;
                m.add = n0 > 0;
            } else {
                m.out = (T*)c.dW + k0 * c.D;
                m.ldout = c.D;
                m.vector = c.D % 4 == 0;
            }
            rc = product<T, true>(m, p.cut_w, s);
            if (rc) return rc;
            m = ProductArgs{};  // dH (+)= dz W
            m.p = DmeOperand{dz, a.lddz * size, nb};
            m.q = DmeOperand{a.w.at, a.w.ld, c.D};
            m.k = width;
            m.zeros = a.zeros;
            if (p.part_h) {
                m.part = (float*)(ws + p.ph);
                m.ldpart = p.ldpart;
                m.split_stride = p.nb * p.ldpart;
                m.add = k0 > 0;
            } else {
                m.out = (T*)c.dH + n0 * c.D;
                m.ldout = c.D;
                m.vector = c.D % 4 == 0;
            }
            rc = product<T, false>(m, p.cut_h, s);
            if (rc) return rc;
        }
        if (p.part_h)
            hipLaunchKernelGGL(join_kernel<T>, dim3(dme_blocks(nb * c.D, 1024, 8192)), dim3(256), 0, s, (const float*)(ws + p.ph), p.ldpart,
                               p.nb * p.ldpart, p.cut_h.splits, nb, c.D, (T*)c.dH + n0 * c.D);
        if (c.dbias)
            hipLaunchKernelGGL(bias_kernel, dim3((unsigned)((c.K + 255) / 256)), dim3(256), 0, s, (const float*)a.dbias, a.tiles_r, c.K,
                               fixed, largest, p.headroom, (int)(n0 > 0), c.dbias);
    }
    if (gradient && p.part_w)
        hipLaunchKernelGGL(join_kernel<T>, dim3(dme_blocks(c.K * c.D, 1024, 8192)), dim3(256), 0, s, (const float*)(ws + p.pw), p.ldpart,
                           c.K * p.ldpart, p.cut_w.splits, c.K, c.D, (T*)c.dW);
    DME_HIP_CHECK(hipGetLastError());
    return DME_OK;
}

int check_call(const void* H, int64_t ldh, const void* W, int64_t ldw, int type, int64_t N, int64_t K, int64_t D, const dme_count_rows_t* rows,
               int likelihood) {
    DME_REQUIRE(type == DME_TYPE_BF16 || type == DME_TYPE_F32, "features and weights are bf16 or fp32");
    DME_REQUIRE(N >= 0 && K >= 1 && D >= 1, "bad shape: N = %lld, K = %lld, D = %lld", (long long)N, (long long)K, (long long)D);
    DME_REQUIRE(K <= 0x7fffffffll && D <= (1ll << 20) && N <= (1ll << 40), "shape out of range");
    DME_REQUIRE(ldh >= D && ldw >= D, "pitch smaller than a row");
    DME_REQUIRE(likelihood == DME_LIKELIHOOD_MULTINOMIAL || likelihood == DME_LIKELIHOOD_DIRICHLET, "unknown likelihood %d", likelihood);
    DME_REQUIRE(rows != nullptr, "no count rows");
    DME_REQUIRE((N == 0 || H != nullptr) && W != nullptr, "null pointer");
    const uintptr_t size = type == DME_TYPE_BF16 ? 2 : 4;
    DME_REQUIRE((uintptr_t)H % size == 0 && (uintptr_t)W % size == 0, "operand not aligned to its values");
    if (rows->kind == CSR) {
        DME_REQUIRE(N == 0 || rows->rowptr != nullptr, "null rowptr");
        DME_REQUIRE(rows->nnz >= 0 && rows->nnz <= (1ll << 36) && (rows->nnz == 0 || (rows->colidx != nullptr && rows->vals != nullptr)), "bad CSR entries");
    } else if (rows->kind == DENSE) {
        DME_REQUIRE(N == 0 || rows->X != nullptr, "null count matrix");
        DME_REQUIRE(rows->elem == 2 || rows->elem == 4, "counts have 2 or 4 bytes");
        DME_REQUIRE(rows->ld >= K, "count matrix narrower than K");
    } else {
        DME_REQUIRE(rows->kind == LABELS, "unknown kind of rows %d", (int)rows->kind);
        DME_REQUIRE(N == 0 || rows->labels != nullptr, "null labels");
    }
    return DME_OK;
}

}  // namespace

extern "C" int64_t dme_log_loss_workspace_bytes(const void* H, int64_t ldh, const void* W, int64_t ldw, int type, int64_t N, int64_t K, int64_t D,
                                                const dme_count_rows_t* rows, int gradient) {
    if (check_call(H, ldh, W, ldw, type, N, K, D, rows, DME_LIKELIHOOD_MULTINOMIAL) != DME_OK) return -1;
    return make_plan(H, ldh, W, ldw, type, N, K, D, rows, gradient != 0).bytes;
}

extern "C" int dme_log_loss(const void* H, int64_t ldh, const void* W, int64_t ldw, const float* bias, int type, int64_t N, int64_t K, int64_t D,
                            const dme_count_rows_t* rows, int likelihood, float* loss, void* ws, int64_t ws_bytes, void* stream) {
    const int rc = check_call(H, ldh, W, ldw, type, N, K, D, rows, likelihood);
    if (rc) return rc;
    if (N == 0) return DME_OK;
    DME_REQUIRE(loss != nullptr, "null loss");
    const Plan p = make_plan(H, ldh, W, ldw, type, N, K, D, rows, false);
    if (ws == nullptr || (uintptr_t)ws % 256 != 0 || ws_bytes < p.bytes)
        return dme_set_error(DME_ERR_WORKSPACE, "workspace of %lld bytes, aligned to 256, needed", p.bytes);
    Call c{H, ldh, W, ldw, bias, N, K, D, rows, likelihood, nullptr, loss, nullptr, nullptr, nullptr, (char*)ws};
    return type == DME_TYPE_BF16 ? work<__bf16>(c, p, false, (hipStream_t)stream) : work<float>(c, p, false, (hipStream_t)stream);
}

extern "C" int dme_log_loss_gradient(const void* H, int64_t ldh, const void* W, int64_t ldw, const float* bias, int type, int64_t N, int64_t K,
                                     int64_t D, const dme_count_rows_t* rows, int likelihood, const float* row_weights, float* loss, void* dH,
                                     void* dW, float* dbias, void* ws, int64_t ws_bytes, void* stream) {
    const int rc = check_call(H, ldh, W, ldw, type, N, K, D, rows, likelihood);
    if (rc) return rc;
    DME_REQUIRE(dW != nullptr, "null gradient");
    const long long size = type == DME_TYPE_BF16 ? 2 : 4;
    DME_REQUIRE((uintptr_t)dW % 16 == 0 && (uintptr_t)dH % 16 == 0, "gradients must be aligned to 16 bytes");
    if (N == 0) {  // a sum over no rows
        hipLaunchKernelGGL(dme_pack_kernel<char>, dim3(dme_blocks(K * D * size, 4096, 8192)), dim3(256), 0, (hipStream_t)stream, (const char*)nullptr, 0,
                           K * D * size, 0, (char*)dW, 1);
        if (dbias) hipLaunchKernelGGL(zero_kernel, dim3(dme_blocks(K, 1024, 4096)), dim3(256), 0, (hipStream_t)stream, (u32*)dbias, K);
        DME_HIP_CHECK(hipGetLastError());
        return DME_OK;
    }
    DME_REQUIRE(loss != nullptr && dH != nullptr, "null output");
    const Plan p = make_plan(H, ldh, W, ldw, type, N, K, D, rows, true);
    if (ws == nullptr || (uintptr_t)ws % 256 != 0 || ws_bytes < p.bytes)
        return dme_set_error(DME_ERR_WORKSPACE, "workspace of %lld bytes, aligned to 256, needed", p.bytes);
    Call c{H, ldh, W, ldw, bias, N, K, D, rows, likelihood, row_weights, loss, dH, dW, dbias, (char*)ws};
    return type == DME_TYPE_BF16 ? work<__bf16>(c, p, true, (hipStream_t)stream) : work<float>(c, p, true, (hipStream_t)stream);
}
