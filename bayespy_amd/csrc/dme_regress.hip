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
#include <atomic>

#include "dme_products.h"

namespace {

constexpr int TCOLS = 128;          // columns of a tile
constexpr int ZP = TCOLS + 4;       // pitch of the tile in LDS (a multiple of 16 bytes that spreads the rows over the banks)
constexpr float LOG2E = 1.44269504088896341f;
constexpr long long ROW_BLOCK = 16384;             // rows worked on at a time
constexpr long long PIECE_BYTES = 512ll << 20;     // of d loss / d z and its transpose held at a time

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
    const int* table;         // CSR: [tiles + 1][nb], where tile t of a row's entries begins, from the row's first entry
    const double* total;      // CSR: [nb], NaN for a row that breaks the format
};

__device__ __forceinline__ long long row_begin(const Rows& rows, long long r) {
    const long long p = rows.rowptr[r];
    return p < 0 ? 0 : p < rows.nnz ? p : rows.nnz;
}

__device__ __forceinline__ int count_at(const Rows& rows, long long r, long long k) {
    return rows.elem == 2 ? (int)((const unsigned short*)rows.X)[r * rows.ldx + k] : ((const int*)rows.X)[r * rows.ldx + k];
}

// CSR rows: totals, the check of the format (columns strictly ascending and below K, no negative count), and the table
// of where each tile of TCOLS columns begins in a row.  16 lanes a row.  A row that breaks the format gets an empty
// table and a total of NaN, so that its loss is NaN and no column out of range is ever followed.
__global__ __launch_bounds__(256) void rows_kernel(Rows rows, long long nb, long long K, int tiles, int* table, double* total) {
    const int sub = threadIdx.x & 15;
    const long long r = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool real = r < nb;
    long long p0 = 0, p1 = 0;
    bool bad = false;
    if (real) {
        const long long q0 = rows.rowptr[r], q1 = rows.rowptr[r + 1];
        bad = q0 < 0 || q1 < q0 || q1 > rows.nnz;
        p0 = row_begin(rows, r);
        p1 = bad ? p0 : q1;
    }
    double t = 0.0;
    for (long long e = p0 + sub; e < p1; e += 16) {
        const int c = rows.col[e], v = rows.val[e], before = e > p0 ? rows.col[e - 1] : -1;
        if (c < 0 || c >= K || c <= before || v < 0) {
            bad = true;
        } else {
            const int tile = c / TCOLS;
            for (int q = before < 0 ? 0 : before / TCOLS + 1; q <= tile; ++q) table[(long long)q * nb + r] = (int)(e - p0);
            if (e == p1 - 1)
                for (int q = tile + 1; q <= tiles; ++q) table[(long long)q * nb + r] = (int)(p1 - p0);
        }
        t += (double)v;
    }
    t = sum16(t);
    const unsigned long long any = __ballot(bad);
    const bool row_bad = (any >> (threadIdx.x & 48)) & 0xffff;
    if (!real) return;
    if (row_bad || p1 == p0)
        for (int q = sub; q <= tiles; q += 16) table[(long long)q * nb + r] = 0;
    if (sub == 0) total[r] = row_bad ? __builtin_nan("") : t;
}

struct TileArgs {
    DmeOperands op;
    long long tiles_r, tiles_c;
    int slices;
    const float* bias;
    long long nb;      // rows of the block
    long long K;
    long long column;  // first column of the piece
    Rows rows;
    // forward
    f32x2* part;       // [tile][nb]: maximum, sum of exponentials
    double* part_f;    // DENSE: [tile][nb]: sum F(z, x)
    double* part_t;    // DENSE: [tile][nb]: sum x, NaN where a count is negative
    float* entry_z;    // CSR: [nnz], LABELS: [nb]: z at the counts
    int likelihood;
    // backward
    const float* lse2;     // [nb]: l * log2 e
    const float* coef;     // [nb]: weight * G(l, T) * 2^(lse2 - l log2 e)
    const float* weight;   // [nb]
    const float* entry_g;  // CSR: [nnz]: weight * G(z, x)
    void* dz;              // [nb][lddz]
    long long lddz;
    void* dzt;             // [columns of the piece][lddzt]
    long long lddzt;
    float* dbias;          // [tiles_r][K] or null
};

// One tile of z.  The products end in registers; the tile then lies in LDS in 32 bits, where the row's 16 lanes reduce
// it, the counts find their values, and (backward) columns are summed and both orders written out.
template <class T, int TR, int KIND, bool BACKWARD>
__global__ __launch_bounds__(256, 2) void tile_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, TR, TCOLS, (TR == 16 ? 1 : 2), (TR == 16 ? 4 : 2)> Tile;
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    const long long r0 = tr * TR, c0 = tc * TCOLS, k0 = a.column + c0;
    float* z = (float*)lds;
    {
        Tile t;
        t.run(a.op, lds, r0, c0, 0, a.slices);
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const int c = Tile::col_of(i);
            f32x4 b;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const long long k = k0 + c + q;
                b[q] = k < a.K ? (a.bias ? a.bias[k] : 0.f) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j) {
                f32x4 v = t.acc[i][j] + b;
#pragma unroll
                for (int q = 0; q < 4; ++q) v[q] = k0 + c + q < a.K ? v[q] : -INFINITY;
                *(f32x4*)(z + Tile::row_of(j) * ZP + c) = v;
            }
        }
    }
    __syncthreads();
    const int tid = threadIdx.x, sub = tid & 15;
    const long long gtile = k0 / TCOLS;
    if (!BACKWARD) {
#pragma unroll 1
        for (int row = tid >> 4; row < TR; row += 16) {
            const long long r = r0 + row;
            if (r >= a.nb) break;  // all of a row's lanes, and rows only ascend
            const float* zr = z + row * ZP;
            const f32x4 u = *(const f32x4*)(zr + sub * 4), w = *(const f32x4*)(zr + 64 + sub * 4);
            const float m = max16(fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]))));
            const float base = m == -INFINITY ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) s += __builtin_amdgcn_exp2f((u[q] - base) * LOG2E) + __builtin_amdgcn_exp2f((w[q] - base) * LOG2E);
            s = sum16(s);
            if (sub == 0) a.part[gtile * a.nb + r] = f32x2{m, s};
            if (KIND == DENSE) {
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
                    a.part_f[gtile * a.nb + r] = f;
                    a.part_t[gtile * a.nb + r] = t;
                }
            }
            if (KIND == CSR) {
                const int e1 = a.rows.table[(gtile + 1) * a.nb + r];
                for (int e = a.rows.table[gtile * a.nb + r] + sub; e < e1; e += 16) {
                    const long long at = row_begin(a.rows, r) + e;
                    const long long c = a.rows.col[at] - k0;
                    if (c >= 0 && c < TCOLS) a.entry_z[at] = zr[c];
                }
            }
            if (KIND == LABELS && sub == 0) {
                const long long k = a.rows.labels[r];
                if (k >= k0 && k < k0 + TCOLS && k < a.K) a.entry_z[r] = zr[k - k0];
            }
        }
        return;
    }
    // d loss / d z in place of z; rows beyond the block and columns beyond K become zero
#pragma unroll 1
    for (int row = tid >> 4; row < TR; row += 16) {
        const long long r = r0 + row;
        const bool real = r < a.nb;
        const float l2 = real ? a.lse2[r] : INFINITY, cf = real ? a.coef[r] : 0.f;
        float* zr = z + row * ZP;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 v = *(const f32x4*)(zr + h * 64 + sub * 4);
            f32x4 d;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                d[q] = real ? __builtin_amdgcn_exp2f(__builtin_fmaf(v[q], LOG2E, -l2)) * cf : 0.f;
                if (KIND == DENSE) {
                    const long long k = k0 + h * 64 + sub * 4 + q;
                    if (real && k < a.K) {
                        const int x = count_at(a.rows, r, k);
                        if (x != 0) d[q] -= a.weight[r] * (float)g_of(a.likelihood, (double)v[q], (double)x);
                    }
                }
            }
            *(f32x4*)(zr + h * 64 + sub * 4) = d;
        }
        // the row's counts: its own 16 lanes wrote the row, in one wave
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (KIND == CSR && real) {
            const int e1 = a.rows.table[(gtile + 1) * a.nb + r];
            for (int e = a.rows.table[gtile * a.nb + r] + sub; e < e1; e += 16) {
                const long long at = row_begin(a.rows, r) + e;
                const long long c = a.rows.col[at] - k0;
                if (c >= 0 && c < TCOLS) zr[c] -= a.entry_g[at];
            }
        }
        if (KIND == LABELS && real && sub == 0) {
            const long long k = a.rows.labels[r];
            if (k >= k0 && k < k0 + TCOLS && k < a.K) zr[k - k0] -= a.weight[r];
        }
    }
    __syncthreads();
    // rounding to T here is the gradient's one rounding before its products, as the operands' own type allows
    T* dz = (T*)a.dz;
#pragma unroll 1
    for (int row = tid >> 4; row < TR; row += 16) {
        if (r0 + row >= a.nb) break;
#pragma unroll
        for (int h = 0; h < 2; ++h) dme_store4(dz + (r0 + row) * a.lddz + c0 + h * 64 + sub * 4, *(const f32x4*)(z + row * ZP + h * 64 + sub * 4));
    }
    T* dzt = (T*)a.dzt;
    const int c = tid & 127, half = tid >> 7;
    float sum = 0.f;
    constexpr int ROWS = TR / 2;
    if (k0 + c < a.K) {
#pragma unroll 1
        for (int q = 0; q < ROWS; q += 4) {
            const int row = half * ROWS + q;
            f32x4 v;
#pragma unroll
            for (int s = 0; s < 4; ++s) v[s] = z[(row + s) * ZP + c];
            sum += (v[0] + v[1]) + (v[2] + v[3]);
            if (r0 + row < a.lddzt) dme_store4(dzt + (c0 + c) * a.lddzt + r0 + row, v);
        }
    }
    if (a.dbias) {
        __syncthreads();
        float* other = z;
        if (half) other[c] = sum;
        __syncthreads();
        if (!half && k0 + c < a.K) a.dbias[tr * a.K + k0 + c] = sum + other[c];
    }
}

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
    float* entry_g;
};

// The row's pieces become l, the loss, and what the gradient needs of them.  16 lanes a row, sums in 64 bits.
__global__ __launch_bounds__(256) void row_kernel(RowArgs a) {
    const int sub = threadIdx.x & 15;
    const long long r = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool real = r < a.nb;
    const long long rr = real ? r : a.nb - 1;
    float m = -INFINITY;
    for (int t = sub; t < a.tiles; t += 16) m = fmaxf(m, a.part[t * a.nb + rr][0]);
    m = max16(m);
    const float base = m == -INFINITY ? 0.f : m;
    double s = 0.0, f = 0.0, total = 0.0;
    for (int t = sub; t < a.tiles; t += 16) {
        const f32x2 p = a.part[t * a.nb + rr];
        s += (double)p[1] * (double)__builtin_amdgcn_exp2f((p[0] - base) * LOG2E);
    }
    s = sum16(s);
    const double lse = s == 0.0 ? -INFINITY : (double)base + log(s);
    const float weight = a.weights ? a.weights[rr] : 1.f;
    if (a.kind == DENSE) {
        for (int t = sub; t < a.tiles; t += 16) {
            f += a.part_f[t * a.nb + rr];
            total += a.part_t[t * a.nb + rr];
        }
        f = sum16(f);
        total = sum16(total);
    } else if (a.kind == CSR) {
        total = a.rows.total[rr];
        if (total == total) {  // uniform over the row's lanes: sum16 below is outside
            const long long e1 = row_begin(a.rows, rr + 1);
            for (long long e = row_begin(a.rows, rr) + sub; e < e1; e += 16) {
                const double z = (double)a.entry_z[e], x = (double)a.rows.val[e];
                f += f_of(a.likelihood, z, x);
                if (a.lse2 && real) a.entry_g[e] = weight * (float)g_of(a.likelihood, z, x);
            }
        }
        f = sum16(f);
    } else {
        const long long k = a.rows.labels[rr];
        total = k < 0 ? 0.0 : k < a.K ? 1.0 : __builtin_nan("");
        f = k >= 0 && k < a.K ? (double)a.entry_z[rr] : 0.0;
    }
    if (!real || sub != 0) return;
    a.loss[r] = total == 0.0 ? 0.f : (float)(f_of(a.likelihood, lse, total) - f);
    if (!a.lse2) return;
    // exp(z - l) is taken as exp2(z log2 e - lse2); what lse2's rounding to 32 bits drops goes into the coefficient
    const double exact2 = lse * (double)LOG2E;
    const float l2 = total == 0.0 ? INFINITY : (float)exact2;
    a.lse2[r] = l2;
    a.coef[r] = total == 0.0 ? 0.f : (float)((double)weight * g_of(a.likelihood, lse, total) * exp2((double)l2 - exact2));
    a.weight[r] = weight;
}

struct ProductArgs {
    DmeOperands op;
    long long tiles_r, tiles_c;
    int slices, per_split;
    float* part;        // [split][R][ldpart], or null: the result goes to out in T
    long long ldpart, split_stride;
    int add;            // part holds sums already
    void* out;
    long long ldout;
    int vector;         // out's rows are aligned to four values
};

// out = P Q' (R x C), in T, or as 32-bit pieces where k is split over workgroups or over launches.
template <class T>
__global__ __launch_bounds__(256, 2) void product_kernel(ProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, 128, 128, 2, 2> Tile;
    long long tr, tc;
    dme_tile_of(blockIdx.x, a.tiles_r, a.tiles_c, tr, tc);
    const int s0 = (int)blockIdx.y * a.per_split;
    int s1 = s0 + a.per_split;
    s1 = s1 < a.slices ? s1 : a.slices;
    Tile t;
    t.run(a.op, lds, tr * 128, tc * 128, s0, s1);
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = tr * 128 + Tile::row_of(j);
        if (r >= a.op.R) continue;
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const long long c = tc * 128 + Tile::col_of(i);
            if (c >= a.op.C) continue;
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
                    if (c + q < a.op.C) ((T*)a.out)[r * a.ldout + c + q] = (T)v[q];
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

// dbias [K] (+)= the row tiles' sums, in their order.
__global__ __launch_bounds__(256) void bias_kernel(const float* part, long long tiles, long long K, int add, float* dbias) {
    const long long k = (long long)blockIdx.x * 256 + threadIdx.x;
    if (k >= K) return;
    double v = add ? (double)dbias[k] : 0.0;
    for (long long t = 0; t < tiles; ++t) v += (double)part[t * K + k];
    dbias[k] = (float)v;
}

__global__ void zero_kernel(u32* p, long long words) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (long long)gridDim.x * blockDim.x) p[i] = 0;
}

inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }

// Everything a call decides before its first launch.  The workspace is laid out in the same order by both passes.
struct Plan {
    int size;                 // bytes of a value
    bool pack_h, pack_w;      // the operand is copied with a pitch of whole 16-byte chunks first
    long long dpad;           // k of the first product in a packed operand
    long long nb, tiles, chunk;
    int split_w, split_h;     // pieces of k in dW and dH
    bool part_w, part_h;      // they leave 32-bit pieces
    long long ldt, ldpart;
    long long zeros, h, w, table, total, part, part_f, part_t, entry_z, entry_g, lse2, coef, weight, dbias, ht, wt, dz, dzt, pw, ph, bytes;
};

int splits_for(long long tiles, long long slices) {
    long long s = 1024 / (tiles > 0 ? tiles : 1);  // enough workgroups for 256 CUs with some to spare ...
    if (s > slices / 4) s = slices / 4;            // ... each with four slices of k at least
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

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
    p.tiles = (K + TCOLS - 1) / TCOLS;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    p.zeros = take(256);
    if (p.pack_h) p.h = take(p.nb * p.dpad * p.size);
    if (p.pack_w) p.w = take(K * p.dpad * p.size);
    p.part = take(p.tiles * p.nb * 8);
    if (rows->kind == CSR) {
        p.table = take((p.tiles + 1) * p.nb * 4);
        p.total = take(p.nb * 8);
        p.entry_z = take(rows->nnz * 4);
    } else if (rows->kind == DENSE) {
        p.part_f = take(p.tiles * p.nb * 8);
        p.part_t = take(p.tiles * p.nb * 8);
    } else {
        p.entry_z = take(p.nb * 4);
    }
    if (gradient) {
        if (rows->kind == CSR) p.entry_g = take(rows->nnz * 4);
        p.lse2 = take(p.nb * 4);
        p.coef = take(p.nb * 4);
        p.weight = take(p.nb * 4);
        p.ldt = up(p.nb, 16 / p.size);
        p.dbias = take((p.nb + 127) / 128 * K * 4);
        p.ht = take(D * p.ldt * p.size);
        p.wt = take(D * p.tiles * TCOLS * p.size);
        long long c = PIECE_BYTES / (2 * p.ldt * p.size) / TCOLS;
        if (c < 1) c = 1;
        if (c > p.tiles) c = p.tiles;
        const long long pieces = (p.tiles + c - 1) / c;
        p.chunk = (p.tiles + pieces - 1) / pieces * TCOLS;  // pieces of like width
        p.dz = take(p.nb * p.chunk * p.size);
        p.dzt = take(p.chunk * p.ldt * p.size);
        const long long tiles_d = (D + 127) / 128;
        p.ldpart = up(D, 4);
        p.split_w = splits_for((p.chunk + 127) / 128 * tiles_d, (p.ldt * p.size + DME_SLICE - 1) / DME_SLICE);
        p.split_h = splits_for((p.nb + 127) / 128 * tiles_d, (p.chunk * p.size + DME_SLICE - 1) / DME_SLICE);
        p.part_w = p.split_w > 1 || N > p.nb;
        p.part_h = p.split_h > 1 || p.chunk < p.tiles * TCOLS;
        if (p.part_w) p.pw = take((long long)p.split_w * K * p.ldpart * 4);
        if (p.part_h) p.ph = take((long long)p.split_h * p.nb * p.ldpart * 4);
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

template <class T, int TR, int KIND, bool BACKWARD>
int launch_tile(const TileArgs& a, hipStream_t s) {
    typedef DmeTile<T, TR, TCOLS, (TR == 16 ? 1 : 2), (TR == 16 ? 4 : 2)> Tile;
    constexpr int bytes = 2 * Tile::STAGE > TR * ZP * 4 ? 2 * Tile::STAGE : TR * ZP * 4;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, tile_kernel<T, TR, KIND, BACKWARD>, bytes);
    if (rc) return rc;
    hipLaunchKernelGGL((tile_kernel<T, TR, KIND, BACKWARD>), dim3((unsigned)(a.tiles_r * a.tiles_c)), dim3(256), bytes, s, a);
    return DME_OK;
}

template <class T, bool BACKWARD>
int tiles_of_z(TileArgs a, int kind, hipStream_t s) {
    const bool few = a.nb <= 16;
    a.tiles_r = few ? 1 : (a.nb + 127) / 128;
    if (kind == LABELS) return few ? launch_tile<T, 16, LABELS, BACKWARD>(a, s) : launch_tile<T, 128, LABELS, BACKWARD>(a, s);
    if (kind == CSR) return few ? launch_tile<T, 16, CSR, BACKWARD>(a, s) : launch_tile<T, 128, CSR, BACKWARD>(a, s);
    return few ? launch_tile<T, 16, DENSE, BACKWARD>(a, s) : launch_tile<T, 128, DENSE, BACKWARD>(a, s);
}

template <class T>
int product(ProductArgs a, int splits, hipStream_t s) {
    typedef DmeTile<T, 128, 128, 2, 2> Tile;
    a.tiles_r = (a.op.R + 127) / 128;
    a.tiles_c = (a.op.C + 127) / 128;
    a.slices = (int)((a.op.kbytes + DME_SLICE - 1) / DME_SLICE);
    a.per_split = (a.slices + splits - 1) / splits;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, product_kernel<T>, 2 * Tile::STAGE);
    if (rc) return rc;
    hipLaunchKernelGGL(product_kernel<T>, dim3((unsigned)(a.tiles_r * a.tiles_c), (unsigned)splits), dim3(256), 2 * Tile::STAGE, s, a);
    return DME_OK;
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
    const int size = p.size;
    const long long kpad = p.tiles * TCOLS;
    char* ws = c.ws;
    hipLaunchKernelGGL(zero_kernel, dim3(1), dim3(64), 0, s, (u32*)(ws + p.zeros), 64);
    const char* W = (const char*)c.W;
    long long ldw = c.ldw * size, kbytes = c.D * size;
    if (p.pack_w) {
        hipLaunchKernelGGL(dme_pack_kernel<T>, dim3(dme_blocks(c.K * p.dpad, 1024, 8192)), dim3(256), 0, s, (const T*)c.W, c.ldw, c.K, c.D,
                           (T*)(ws + p.w), p.dpad);
        W = ws + p.w;
        ldw = p.dpad * size;
    }
    if (gradient)
        hipLaunchKernelGGL(dme_transpose_kernel<T>, dim3(dme_blocks(up(c.D, 64) * kpad, 4096, 8192)), dim3(256), 0, s, (const T*)c.W, c.ldw, c.K, c.D,
                           (T*)(ws + p.wt), kpad);
    for (long long n0 = 0; n0 < c.N; n0 += p.nb) {
        const long long nb = c.N - n0 < p.nb ? c.N - n0 : p.nb;
        const char* H = (const char*)c.H + n0 * c.ldh * size;
        long long ldh = c.ldh * size;
        if (p.pack_h) {
            hipLaunchKernelGGL(dme_pack_kernel<T>, dim3(dme_blocks(nb * p.dpad, 1024, 8192)), dim3(256), 0, s, (const T*)H, c.ldh, nb, c.D,
                               (T*)(ws + p.h), p.dpad);
            H = ws + p.h;
            ldh = p.dpad * size;
        }
        if (p.pack_h || p.pack_w) kbytes = p.dpad * size;
        TileArgs a{};
        a.op = DmeOperands{H, W, ldh, ldw, nb, c.K, kbytes, ws + p.zeros};
        a.tiles_c = p.tiles;
        a.slices = (int)((kbytes + DME_SLICE - 1) / DME_SLICE);
        a.bias = c.bias;
        a.nb = nb;
        a.K = c.K;
        a.likelihood = c.likelihood;
        Rows& rows = a.rows;
        if (c.rows->kind == CSR) {
            rows.rowptr = (const long long*)c.rows->rowptr + n0;
            rows.col = (const int*)c.rows->colidx;
            rows.val = (const int*)c.rows->vals;
            rows.nnz = c.rows->nnz;
            rows.table = (const int*)(ws + p.table);
            rows.total = (const double*)(ws + p.total);
            hipLaunchKernelGGL(rows_kernel, dim3((unsigned)((nb + 15) / 16)), dim3(256), 0, s, rows, nb, c.K, (int)p.tiles, (int*)(ws + p.table),
                               (double*)(ws + p.total));
        } else if (c.rows->kind == DENSE) {
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
        int rc = tiles_of_z<T, false>(a, c.rows->kind, s);
        if (rc) return rc;
        RowArgs ra{};
        ra.nb = nb;
        ra.K = c.K;
        ra.tiles = (int)p.tiles;
        ra.kind = c.rows->kind;
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
        }
        hipLaunchKernelGGL(row_kernel, dim3((unsigned)((nb + 15) / 16)), dim3(256), 0, s, ra);
        if (!gradient) continue;
        const long long ldt = up(nb, 16 / size);
        hipLaunchKernelGGL(dme_transpose_kernel<T>, dim3(dme_blocks(up(c.D, 64) * up(ldt, 64), 4096, 8192)), dim3(256), 0, s,
                           (const T*)((const char*)c.H + n0 * c.ldh * size), c.ldh, nb, c.D, (T*)(ws + p.ht), ldt);
        a.lse2 = ra.lse2;
        a.coef = ra.coef;
        a.weight = ra.weight;
        a.entry_g = ra.entry_g;
        a.dz = ws + p.dz;
        a.dzt = ws + p.dzt;
        a.lddzt = ldt;
        a.dbias = c.dbias ? (float*)(ws + p.dbias) : nullptr;
        for (long long k0 = 0; k0 < c.K; k0 += p.chunk) {
            const long long width = c.K - k0 < p.chunk ? c.K - k0 : p.chunk;
            a.column = k0;
            a.op.Q = W + k0 * ldw;
            a.op.C = width;
            a.tiles_c = (width + TCOLS - 1) / TCOLS;
            a.lddz = a.tiles_c * TCOLS;
            rc = tiles_of_z<T, true>(a, c.rows->kind, s);
            if (rc) return rc;
            ProductArgs w{};  // dW of the piece = dz' H
            w.op = DmeOperands{ws + p.dzt, ws + p.ht, ldt * size, ldt * size, width, c.D, ldt * size, ws + p.zeros};
            if (p.part_w) {
                w.part = (float*)(ws + p.pw) + k0 * p.ldpart;
                w.ldpart = p.ldpart;
                w.split_stride = c.K * p.ldpart;
                w.add = n0 > 0;
            } else {
                w.out = (T*)c.dW + k0 * c.D;
                w.ldout = c.D;
                w.vector = c.D % 4 == 0;
            }
            rc = product<T>(w, p.split_w, s);
            if (rc) return rc;
            ProductArgs h{};  // dH (+)= dz W
            h.op = DmeOperands{ws + p.dz, ws + p.wt + k0 * size, a.lddz * size, kpad * size, nb, c.D, a.lddz * size, ws + p.zeros};
            if (p.part_h) {
                h.part = (float*)(ws + p.ph);
                h.ldpart = p.ldpart;
                h.split_stride = p.nb * p.ldpart;
                h.add = k0 > 0;
            } else {
                h.out = (T*)c.dH + n0 * c.D;
                h.ldout = c.D;
                h.vector = c.D % 4 == 0;
            }
            rc = product<T>(h, p.split_h, s);
            if (rc) return rc;
        }
        if (p.part_h)
            hipLaunchKernelGGL(join_kernel<T>, dim3(dme_blocks(nb * c.D, 1024, 8192)), dim3(256), 0, s, (const float*)(ws + p.ph), p.ldpart,
                               p.nb * p.ldpart, p.split_h, nb, c.D, (T*)c.dH + n0 * c.D);
        if (c.dbias)
            hipLaunchKernelGGL(bias_kernel, dim3((unsigned)((c.K + 255) / 256)), dim3(256), 0, s, (const float*)a.dbias,
                               nb <= 16 ? 1 : (nb + 127) / 128, c.K, (int)(n0 > 0), c.dbias);
    }
    if (gradient && p.part_w)
        hipLaunchKernelGGL(join_kernel<T>, dim3(dme_blocks(c.K * c.D, 1024, 8192)), dim3(256), 0, s, (const float*)(ws + p.pw), p.ldpart,
                           c.K * p.ldpart, p.split_w, c.K, c.D, (T*)c.dW);
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
