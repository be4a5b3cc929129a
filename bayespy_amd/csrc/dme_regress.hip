// dme_regress.hip — the log loss of count rows under a linear predictor, and its gradient (include/dme_hip.h,
// dme_log_loss*).  z = H W' + b is never kept: a workgroup makes a tile of it on the matrix cores, reduces it to a
// maximum, a sum of exponentials and what the row's counts need of it, and drops it.  The gradient makes the tiles of a
// piece of the columns again, turns them into d loss / d z, and multiplies that piece with W and H.
//
// With l = log sum_k exp z_k and T the row's total (DirichletEstimation/dirichletMultinomialEstimation.py:16-48 is the
// Dirichlet likelihood with one z for all rows):
//     loss = F(l, T) - sum_k F(z_k, x_k)         d loss / d z_k = exp(z_k - l) G(l, T) - G(z_k, x_k)
//     multinomial  F = x z, G = x;               Dirichlet  F = lgamma(e^z + x) - lgamma(e^z), G = dF/dz
// so both likelihoods share the pass over the columns; F and G are needed at the counts alone.  With m the row's largest z and
// s = sum_k e^(z_k - m) the terms are taken relative to m, so that a row whose z are all far out (masks of the type's lowest value)
// loses nothing:
//     multinomial  loss = T log s - sum_k x_k (z_k - m)
//     Dirichlet    F(z, x) = z + R(z, x):  loss = log s + R(l, T) - sum_{x_k > 0} [(z_k - m) + R(z_k, x_k)] + (1 - J) m, J = #{x_k > 0}
// and e^(z - l) = e^(z - m) / s.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "dme_products.h"

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr long long ROW_BLOCK = 16384;             // rows worked on at a time
constexpr long long LOSS_BLOCK = 65536;            // ... where no gradient is wanted, which keeps 8 to 32 bytes a row and tile
// ... and less of them where K is vast: a launch has fewer than 2^32 threads, and tiles of 64 take a thread for 16 values of z
constexpr long long MOST_CELLS = 1ll << 35;
constexpr long long FEW_ROWS = 128;                // up to here a workgroup a row: too few to fill the card with 16 lanes each
// of d loss / d z held at a time: about the memory-side cache, so that the two products read it from there, and pieces still
// large enough to fill the card (N = 8192, K = 50000, D = 1024: 3508 us with 512 MB, 3400 with 256, 3419 with 128, 3582 with 64;
// N = 4099, D = 128: 707, 653, 724, 790)
constexpr long long PIECE_BYTES = 256ll << 20;

enum { LABELS = DME_ROWS_LABELS, CSR = DME_ROWS_CSR, DENSE = DME_ROWS_DENSE };

// 1 / (12 v) - 1 / (360 v^3) + 1 / (1260 v^5): what Stirling's formula leaves of lgamma (v >= 16: below 3e-12).
__device__ double stirling_rest(double v) {
    const double i = 1.0 / v, q = i * i;
    return i * (1.0 / 12.0 - q * (1.0 / 360.0 - q * (1.0 / 1260.0)));
}

// R(z, x) = sum_{1 <= n < x} log(e^z + n) (F without its first term, z itself).  Up to 15 terms are multiplied out, the rest is a difference
// of two Stirling formulas written without their cancelling parts.
__device__ __attribute__((noinline)) double dirichlet_rest(double z, double x) {
    if (!(x > 1.0)) return 0.0 * x;
    if (z > 60.0) return (x - 1.0) * z;  // e^z + n is e^z in 64 bits
    const double a = exp(z);
    double r = 0.0, prod = 1.0;
    const int head = x < 16.0 ? (int)x : 16;
    for (int n = 1; n < head; ++n) {
        prod *= a + n;
        if (prod > 1e200) {
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

__device__ __forceinline__ double g_of(int likelihood, double z, double x) {
    return likelihood == DME_LIKELIHOOD_DIRICHLET ? dirichlet_g(z, x) : x;
}

// The counts that most cells hold, 1 <= x <= 16, in 32 bits.  With a = e^z the terms a + n, 1 <= n < x, are multiplied out, so that R takes
// one logarithm and G, as sum 1 / (a + n) over the same product, one reciprocal.  For z > 0 they are taken over a: with w = 1 / a
//     R = (x - 1) z + log prod (1 + n w)      G = 1 + sum 1 / (1 + n w)
// and no product leaves 16!, however large |z| is.  Terms n and x - n are taken together, (a + n) (a + x - n) = a (a + x) + n (x - n), which
// halves the loop; an even x leaves the term in the middle.  e^-|z| as 2^(z log2 e) is off as a z rounded once more would be, and z comes out of 32-bit
// sums; the products round 15 times 2^-24 at most.  The loop runs as far as the wave's largest count: no lane has a branch of its own.
__device__ __forceinline__ bool is_small(int x) { return x <= 16; }
struct SmallTerms {
    float x, one, ww, ends, middle;  // one = a, ww = 1, ends = a (a + x), middle = a + x / 2, or those over a, a^2, a^2 and a
    bool far;
    SmallTerms() = default;
    __device__ __forceinline__ SmallTerms(float z, int count) {
        far = z > 0.f;
        const float e = __builtin_amdgcn_exp2f(-fabsf(z) * LOG2E), w = far ? e : 1.f;
        x = (float)count;
        one = far ? 1.f : e;
        ww = w * w;
        ends = one * __builtin_fmaf(x, w, one);
        middle = __builtin_fmaf(0.5f * x, w, one);
    }
    __device__ __forceinline__ float pair(float n, float other) const { return __builtin_fmaf(n * other, ww, ends); }
};
// N cells of a lane at once; 0 < count <= 16 where there is a cell, 0 elsewhere
template <int N>
__device__ __forceinline__ void small_rest(const float (&z)[N], const int (&count)[N], float (&r)[N]) {
    SmallTerms t[N];
    float most = 0.f;
#pragma unroll
    for (int q = 0; q < N; ++q) {
        t[q] = SmallTerms(z[q], count[q]);
        most = fmaxf(most, t[q].x);
        r[q] = count[q] > 0 && !(count[q] & 1) ? t[q].middle : 1.f;
    }
    for (float n = 1.f; __any(n < most - n); n += 1.f)
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const float other = t[q].x - n;
            r[q] *= n < other ? t[q].pair(n, other) : 1.f;
        }
#pragma unroll
    for (int q = 0; q < N; ++q) {
        r[q] = __builtin_amdgcn_logf(r[q]) * 0.69314718f;
        if (t[q].far && count[q] > 1) r[q] = __builtin_fmaf(t[q].x - 1.f, z[q], r[q]);
    }
}
// Two terms of sum 1 / (a + n) make (2 a + x) / ((a + n) (a + x - n)).
template <int N>
__device__ __forceinline__ void small_g(const float (&z)[N], const int (&count)[N], float (&g)[N]) {
    SmallTerms t[N];
    float most = 0.f, num[N], den[N];
#pragma unroll
    for (int q = 0; q < N; ++q) {
        t[q] = SmallTerms(z[q], count[q]);
        most = fmaxf(most, t[q].x);
        num[q] = 0.f;
        den[q] = 1.f;
    }
    for (float n = 1.f; __any(n < most - n); n += 1.f)
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const float other = t[q].x - n, both = t[q].pair(n, other);
            const bool in = n < other;
            num[q] = in ? __builtin_fmaf(num[q], both, den[q]) : num[q];
            den[q] = in ? den[q] * both : den[q];
        }
#pragma unroll
    for (int q = 0; q < N; ++q) {
        float sum = 2.f * t[q].middle * num[q] * __builtin_amdgcn_rcpf(den[q]);
        sum += !(count[q] & 1) ? __builtin_amdgcn_rcpf(t[q].middle) : 0.f;
        g[q] = count[q] > 0 ? __builtin_fmaf(t[q].one, sum, 1.f) : 0.f;
    }
}
__device__ __forceinline__ float small_rest(float z, int count) {
    const float zs[1] = {z};
    const int xs[1] = {count};
    float r[1];
    small_rest(zs, xs, r);
    return r[0];
}
__device__ __forceinline__ float small_g(float z, int count) {
    const float zs[1] = {z};
    const int xs[1] = {count};
    float g[1];
    small_g(zs, xs, g);
    return g[0];
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
__device__ __forceinline__ int sum16(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, DME_DPP_QUAD_XOR1, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, DME_DPP_QUAD_XOR2, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, DME_DPP_HALF_MIRROR, 0xf, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, DME_DPP_MIRROR, 0xf, 0xf, false);
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
    int row_bytes;     // of an operand's row that may be read: whole chunks of 16 where it is packed or lies so
    long long tiles_r, tiles_c;
    int slices;
    const float* bias;
    long long nb;      // rows of the block
    long long K;
    long long column;  // first column of the piece
    Rows rows;
    // forward
    f32x2* part;       // [tile][nb]: largest z, sum of e^(z - that)
    double* part_f;    // DENSE: [tile][nb]: the counts' sum of the loss, relative to the tile's largest z (0 if that is -inf)
    double* part_w;    // DENSE: [tile][nb]: how often that z goes into it: sum x (multinomial), number of counts (Dirichlet)
    double* part_t;    // DENSE: [tile][nb]: sum x, NaN where a count is negative
    float* entry_z;    // CSR: [nnz], LABELS: [nb]: z at the counts
    int likelihood;
    // backward
    const float* largest_z;  // [nb]: m
    const float* coef;     // [nb]: weight * G(l, T) / s
    const float* weight;   // [nb]
    void* dz;              // [nb][lddz]
    long long lddz;
    float* dbias;          // [tiles_r][K] or null
};

// bias of four columns; columns from K on get -inf, which leaves them out of every sum
typedef f32x4 f32x4_u __attribute__((aligned(4)));
__device__ __forceinline__ f32x4 bias_of(const TileArgs& a, long long k) {
    f32x4 b = f32x4{0.f, 0.f, 0.f, 0.f};
    if (k + 4 <= a.K) {
        if (a.bias) b = *(const f32x4_u*)(a.bias + k);
    } else {
#pragma unroll
        for (int q = 0; q < 4; ++q) b[q] = k + q < a.K ? (a.bias ? a.bias[k + q] : 0.f) : -INFINITY;
    }
    return b;
}

// whether one of the wave's columns is out: only then is there anything to choose
__device__ __forceinline__ bool any_out(f32x4 b) {
    return __any(b[0] == -INFINITY || b[1] == -INFINITY || b[2] == -INFINITY || b[3] == -INFINITY);
}

// z = products + bias; a column that is out has z = -inf whatever its weights hold
__device__ __forceinline__ f32x4 with_bias(f32x4 v, f32x4 b, bool out) {
    v += b;
    if (out)
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = b[q] == -INFINITY ? -INFINITY : v[q];
    return v;
}

// e^(z - m).  The difference is taken first: z log2 e may leave 32 bits where a mask is the type's lowest value.
__device__ __forceinline__ float exp_of(float z, float m) { return __builtin_amdgcn_exp2f((z - m) * LOG2E); }

// The same for many z of one m, one operation less: 2^(z log2 e - r) e^rest with r = m log2 e rounded to 32 bits and what that drops.
// Not for |m| > FAR, where r's rounding is no small number: it is below 2^-24 |r|, so up to FAR 2^(z log2 e - r) is within a factor 2^(1/8) of
// e^(z - m); at 1e10 it is hundreds, and of 2^rounding and 2^-rounding one is infinite and the other 0.  m is a tile's largest z here and a row's
// there: a run of masked columns is enough to be beyond.
constexpr float FAR = 1e6f;
struct Reference {
    float r, rest;
    __device__ __forceinline__ explicit Reference(float m) {
        r = m * LOG2E;
        rest = fabsf(m) <= FAR ? __builtin_amdgcn_exp2f(-__builtin_fmaf(m, LOG2E, -r)) : 1.f;
    }
    __device__ __forceinline__ float operator()(float z) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, LOG2E, -r)); }
};

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

// The `full`-th 16 bytes of a row, of which only what is left of `bytes` belongs to it: the others are 0.
template <class T>
__device__ __forceinline__ u32q row_end(const char* row, int bytes) {
    constexpr int VEC = 16 / sizeof(T);
    typedef T tv __attribute__((ext_vector_type(VEC)));
    const int first = bytes / 16 * 16;
    tv v{};
#pragma unroll
    for (int q = 0; q < VEC; ++q)
        if (first + q * (int)sizeof(T) < bytes) v[q] = *(const T*)(row + first + q * sizeof(T));
    return __builtin_bit_cast(u32q, v);
}
// 16 bytes of a row, aligned to its values alone if LOOSE.  16-bit values: words of four bytes (17 to 20 bytes in all, each word with bytes of the row in
// it), shifted together where they are used; 16-byte loads from odd places took twice as long.
template <class T, bool LOOSE>
struct Chunk {
    typedef u32q u32q_4 __attribute__((aligned(4)));
    u32q v;
    u32 more;
    __device__ __forceinline__ void load(const char* at) {
        if constexpr (!LOOSE) {
            v = *(const u32q*)at;
        } else if constexpr (sizeof(T) == 4) {
            v = *(const u32q_4*)at;
        } else {
            const u32 shift = (u32)(uintptr_t)at & 2;
            v = *(const u32q_4*)(at - shift);
            more = *(const u32*)(at - shift + (shift ? 16 : 12));
        }
    }
    __device__ __forceinline__ u32q get(u32 shift) const {  // address & 2
        if constexpr (!LOOSE || sizeof(T) == 4) return v;
        u32q o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o[q] = __builtin_amdgcn_alignbyte(q < 3 ? v[(q + 1) & 3] : more, v[q], shift);
        return o;
    }
};
template <class T, bool LOOSE>
__device__ __forceinline__ u32q chunk_at(const char* at) {
    Chunk<T, LOOSE> c;
    c.load(at);
    return c.get((u32)(uintptr_t)at & 2);
}

// z at a row's counts: a scalar product for each, 16 lanes an entry, 16 entries of a wave in flight.  There are few of them beside
// the N K values of z that the tiles make (and drop), so they are made once more here instead of being looked for in every tile.
// One wave takes batches `first`, `first + step`, ... of 16 entries.
template <class T, int KIND, bool LOOSE = false>
__device__ __forceinline__ void entries_of(const TileArgs& a, long long r, int first, int step) {
    const int lane = threadIdx.x & 63, sub = lane & 15, group = lane >> 4;
    const int full = a.row_bytes / 16;
    const char* h = a.h.at + r * a.h.ld;
    const long long p0 = KIND == CSR ? row_begin(a.rows, r) : r, p1 = KIND == CSR ? row_begin(a.rows, r + 1) : r + 1;
    for (long long e0 = p0 + first * 16; e0 < p1; e0 += step * 16) {
        int col = -1;
        if (e0 + sub < p1) {
            const long long k = KIND == CSR ? (long long)a.rows.col[e0 + sub] : a.rows.labels[r];
            col = k >= 0 && k < a.K ? (int)k : -1;
        }
        constexpr int DEEP = KIND == CSR ? 4 : 1;
        int k[DEEP];
        const char* w[DEEP];
        float s[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            k[u] = __shfl(col, u * 4 + group);
            w[u] = a.w.at + (k[u] < 0 ? 0 : k[u]) * a.w.ld;  // row 0 in place of none: read, not used
            s[u] = 0.f;
        }
        for (int q = sub; q < full; q += 16) {
            const u32q x = chunk_at<T, LOOSE>(h + q * 16);
            u32q y[DEEP];
#pragma unroll
            for (int u = 0; u < DEEP; ++u) y[u] = chunk_at<T, LOOSE>(w[u] + q * 16);
#pragma unroll
            for (int u = 0; u < DEEP; ++u) s[u] = dot_step(x, y[u], s[u], T());
        }
        if (LOOSE && a.row_bytes % 16 && sub == 0) {
            const u32q x = row_end<T>(h, a.row_bytes);
#pragma unroll
            for (int u = 0; u < DEEP; ++u) s[u] = dot_step(x, row_end<T>(w[u], a.row_bytes), s[u], T());
        }
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            s[u] = sum16(s[u]);
            if (sub == 0 && k[u] >= 0) {
                const float b = a.bias ? a.bias[k[u]] : 0.f;
                a.entry_z[e0 + u * 4 + group] = b == -INFINITY ? b : s[u] + b;
            }
        }
    }
}

// What workgroups beyond the tiles do in the forward launch: a wave makes a row's z at its counts.
template <class T, int KIND, int WAVES>
__device__ __forceinline__ void beyond_tiles(const TileArgs& a, u32 block) {
    const long long r = (long long)block * WAVES + (threadIdx.x >> 6);
    if (r < a.nb) entries_of<T, KIND>(a, r, 0, 1);
}

__device__ __forceinline__ f32x2 merge(f32x2 v, f32x2 o) {
    const float m = fmaxf(v[0], o[0]), base = m == -INFINITY ? 0.f : m;
    return f32x2{m, v[1] * exp_of(v[0], base) + o[1] * exp_of(o[0], base)};
}

// The forward pass for up to 16 rows: a read of the weights and little else.  A wave makes 16 columns for all rows; its weights
// go from memory straight into the matrix instructions' registers, WIDE loads of 16 bytes a lane ahead, and the rows wait in LDS.
// Nothing is shared between waves but the rows, so many small workgroups keep ~200 KB a CU in flight.  Workgroups before the
// columns' make the rows' z at their counts, so that a call has two launches.  Bound by memory: 1 x 50000 x 512 in bf16 reads 51 MB in
// 12.6 us (4.1 TB/s, call after call of the same weights, which the memory-side cache holds).  LOOSE: rows that are not whole chunks of 16 bytes are read as they lie.
template <class T, int KIND, bool LOOSE>
__global__ __launch_bounds__(256) void few_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    __shared__ f32x2 seen[4][16];
    if (blockIdx.x < a.nb) {  // first, since they wait the longest
        entries_of<T, KIND, LOOSE>(a, blockIdx.x, threadIdx.x >> 6, 4);
        return;
    }
    const u32 block = blockIdx.x - (u32)a.nb;
    constexpr int WIDE = 8;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int full = a.row_bytes / 16, chunks = (a.row_bytes + 15) / 16, rounds = (chunks + 3) / 4;  // a round: 64 bytes of each row
    const long long k0 = (long long)block * 64 + wave * 16;
    const long long k = k0 + c < a.K ? k0 + c : a.K - 1;
    const char* w = a.w.at + k * a.w.ld;
    const u32q none = u32q{0, 0, 0, 0};
    const u32 shift = (u32)(uintptr_t)w & 2;
    Chunk<T, LOOSE> y[2][WIDE];
    u32q end = none;
    if (LOOSE && full < chunks && g == (full & 3)) end = row_end<T>(w, a.row_bytes);
    auto load = [&](Chunk<T, LOOSE>* to, int round) {
#pragma unroll
        for (int u = 0; u < WIDE; ++u) {
            const int at = (round + u) * 4 + g;
            to[u].v = none;
            to[u].more = 0;
            if (at < full) to[u].load(w + at * 16);
        }
    };
    load(y[0], 0);
    const int pitch = (rounds * 4 + 4) * 16;  // bytes; the four chunks more spread the rows over the banks
    for (int i = tid; i < 16 * rounds * 4; i += 256) {
        const int r = i / (rounds * 4), at = i - r * (rounds * 4);
        const char* from = a.h.at + r * a.h.ld;
        u32q v = none;
        if (r < a.nb && at < full)
            v = chunk_at<T, LOOSE>(from + at * 16);
        else if (LOOSE && r < a.nb && at < chunks)
            v = row_end<T>(from, a.row_bytes);
        *(u32q*)(lds + r * pitch + at * 16) = v;
    }
    __syncthreads();
    f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
    const char* h = lds + c * pitch + g * 16;
    auto multiply = [&](const Chunk<T, LOOSE>* with, int round) {
#pragma unroll
        for (int u = 0; u < WIDE; ++u)
            if (round + u < rounds) {
                u32q v = with[u].get(shift);
                if (LOOSE && (round + u) * 4 + g == full) v = end;
                acc[u & 1] = dme_mma(v, *(const u32q*)(h + (round + u) * 64), acc[u & 1], T());
            }
    };
    for (int round = 0; round < rounds; round += 2 * WIDE) {
        load(y[1], round + WIDE);
        multiply(y[0], round);
        load(y[0], round + 2 * WIDE);
        multiply(y[1], round + WIDE);
    }
    const f32x4 b = bias_of(a, k0 + g * 4), z = with_bias(acc[0] + acc[1], b, any_out(b));
    float m = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float base = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) s += exp_of(z[q], base);
    s += __shfl_xor(s, 16);
    s += __shfl_xor(s, 32);
    if (g == 0) seen[wave][c] = f32x2{m, s};
    __syncthreads();
    if (tid < 16 && tid < a.nb) a.part[block * a.nb + tid] = merge(merge(seen[0][tid], seen[1][tid]), merge(seen[2][tid], seen[3][tid]));
}

// Tiles of z, reduced where the matrix instructions left them: a lane has NJ rows and 4 NI columns of each.
//   forward   the largest z of each row and the sum of e^(z - that)
//   backward  e^(z - m) coef, rounded to T (the gradient's one rounding before its products), and the columns' sums
//             of the unrounded values.  The counts are not looked at: patch_kernel puts them in.
// 256 a side where there is work for every CU: 4096 x 50000 x 512 in bf16 takes 221 us forward (950 TFLOP/s; 128 a side 320), which is
// the matrix instructions' time and a pass over the tile's 65536 exponentials beside it.  At D = 128 the passes count as much as the products:
// 4099 x 50000 forward 139 us, backward 158 us for 410 MB of d loss / d z.  A workgroup that stayed for tile after tile, the next one's first
// slice on its way under the epilogue, was 1% faster forward and 4% slower backward, where it had no registers left.
template <class T, int TR, int TC, int WR, int WC, int KIND, bool BACKWARD, int STAGES = 0>
__global__ __launch_bounds__(WR * WC * 64) void tile_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef DmeTile<T, TR, TC, WR, WC, false, false, STAGES> Tile;
    if (!BACKWARD && blockIdx.x >= (u32)(a.tiles_r * a.tiles_c)) {
        beyond_tiles<T, KIND, WR * WC>(a, blockIdx.x - (u32)(a.tiles_r * a.tiles_c));
        return;
    }
    long long tr, tc;
    dme_tile_of(blockIdx.x, (u32)a.tiles_r, (u32)a.tiles_c, tr, tc);
    const long long r0 = tr * TR, c0 = tc * TC, k0 = a.column + c0;
    Tile t;
    t.clear();
    t.run(a.h, a.w, a.D, lds, r0, c0, 0, a.slices);
    const int tid = threadIdx.x, g = (tid & 63) >> 4, wc = (tid >> 6) % WC, wr = (tid >> 6) / WC;
    bool out = false;
    if (a.bias || k0 + TC > a.K) {
        const bool inside = k0 + TC <= a.K;  // then no lane looks at its columns
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const f32x4 b = inside ? *(const f32x4_u*)(a.bias + k0 + Tile::col_of(i)) : bias_of(a, k0 + Tile::col_of(i));
            out |= b[0] == -INFINITY || b[1] == -INFINITY || b[2] == -INFINITY || b[3] == -INFINITY;
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j) t.acc[i][j] += b;
        }
    }
    if (__any(out)) {  // rare: the bias is read again
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const f32x4 b = bias_of(a, k0 + Tile::col_of(i));
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) t.acc[i][j][q] = b[q] == -INFINITY ? -INFINITY : t.acc[i][j][q];
        }
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
            const float base = m == -INFINITY ? 0.f : m;
            float s = 0.f;
            if (!__any(fabsf(base) > FAR)) {
                const Reference e(base);
#pragma unroll
                for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s += e(t.acc[i][j][q]);
                s *= e.rest;
            } else {
#pragma unroll
                for (int i = 0; i < Tile::NI; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) s += exp_of(t.acc[i][j][q], base);
            }
            s += __shfl_xor(s, 16);
            s += __shfl_xor(s, 32);
            if (g == 0) seen[wc * TR + wr * Tile::WTR + j * 16 + (tid & 15)] = f32x2{m, s};
        }
        __syncthreads();
        if (tid < TR && r0 + tid < a.nb) {
            f32x2 v = seen[tid];
#pragma unroll
            for (int w = 1; w < WC; ++w) v = merge(v, seen[w * TR + tid]);
            a.part[tc * a.nb + r0 + tid] = v;
        }
        return;
    }
    float m[Tile::NJ], cf[Tile::NJ];
    bool far = false;
#pragma unroll
    for (int j = 0; j < Tile::NJ; ++j) {
        const long long r = r0 + Tile::row_of(j);
        m[j] = r < a.nb ? a.largest_z[r] : INFINITY;
        cf[j] = r < a.nb ? a.coef[r] : 0.f;
        far |= fabsf(m[j]) > FAR && fabsf(m[j]) < INFINITY;
    }
    // In 16 bits a wave's part goes through LDS (its own piece of it), so that whole lines of rows are stored: the lanes of a matrix
    // instruction hold 8 bytes each of 16 rows, and such stores took 27 us for a round of tiles where the memory needs 7.
    constexpr bool TURN = sizeof(T) == 2 && TR >= 128;
    constexpr int PITCH = Tile::WTC * (int)sizeof(T) + 16;
    char* mine = lds + (tid >> 6) * Tile::WTR * PITCH;
    f32x4 sum[Tile::NI];
    const auto each = [&](auto exp_j) {  // exp_j(j, z): e^(z - m[j])
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j) {
                f32x4 d;
#pragma unroll
                for (int q = 0; q < 4; ++q) d[q] = exp_j(j, t.acc[i][j][q]) * cf[j];
                const long long r = r0 + Tile::row_of(j);
                sum[i] += d;  // rows beyond the block have coefficient 0 (and the last row's z)
                if constexpr (TURN)
                    dme_store4((T*)(mine + (j * 16 + (tid & 15)) * PITCH) + i * 16 + g * 4, d);
                else if (r < a.nb)
                    dme_store4((T*)a.dz + r * a.lddz + c0 + Tile::col_of(i), d);
            }
        }
    };
    if (!__any(far)) {
        float r[Tile::NJ];
#pragma unroll
        for (int j = 0; j < Tile::NJ; ++j) {
            const Reference e(m[j]);
            r[j] = e.r;
            cf[j] *= e.rest;
        }
        each([&](int j, float z) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, LOG2E, -r[j])); });
    } else {
        each([&](int j, float z) { return exp_of(z, m[j]); });
    }
    if constexpr (TURN) {
        constexpr int PER = Tile::WTC * (int)sizeof(T) / 16;  // lanes that store a row
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int q = 0; q < Tile::WTR * PER / 64; ++q) {
            const int row = q * (64 / PER) + (tid & 63) / PER, at = (tid & 63) % PER;
            const long long r = r0 + wr * Tile::WTR + row;
            const u32q v = *(const u32q*)(mine + row * PITCH + at * 16);
            if (r < a.nb) *(u32q*)((T*)a.dz + r * a.lddz + c0 + wc * Tile::WTC + at * 8) = v;
        }
    }
    if (a.dbias) {
        float* sums = (float*)lds;  // [WR][TC]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
#pragma unroll
            for (int q = 0; q < 4; ++q) sum[i][q] = sum16(sum[i][q]);
            if ((tid & 15) == 0) *(f32x4*)(sums + wr * TC + Tile::col_of(i)) = sum[i];
        }
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

// Eight neighbouring counts of a row, as they lie (16 or 32 bytes); 0 beyond K.
struct Counts {
    u32q lo, hi;
    __device__ __forceinline__ void load(const Rows& rows, long long r, long long k, long long K) {
        const char* at = rows.X + (r * rows.ldx + k) * rows.elem;
        lo = hi = u32q{0, 0, 0, 0};
        if (k + 8 <= K && ((uintptr_t)at & 15) == 0) {
            lo = __builtin_nontemporal_load((const u32q*)at);
            if (rows.elem == 4) hi = __builtin_nontemporal_load((const u32q*)at + 1);
        } else if (rows.elem == 2) {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (k + q < K) lo[q / 2] |= (u32)((const unsigned short*)at)[q] << (q % 2 * 16);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                if (k + q < K) lo[q] = ((const u32*)at)[q];
                if (k + 4 + q < K) hi[q] = ((const u32*)at)[4 + q];
            }
        }
    }
    __device__ __forceinline__ void get(int elem, int (&v)[8]) const {
        if (elem == 2) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (int)(lo[q / 2] >> (q % 2 * 16) & 0xffff);
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (int)(q < 4 ? lo[q & 3] : hi[q & 3]);
        }
    }
};

// Dirichlet terms of a dense matrix: R(z, 1) = 0 and G(z, 1) = 1, and a wave that ran every cell's loop to the largest of its counts would
// work for few lanes.  A wave's cells with counts above 1 are put on a list in LDS instead, their z left where it is, and taken 128 at a time; those
// for the 64-bit functions go on to a second list and are taken 64 at a time or, the workgroup's few together, at the end.  (16384 x 1000
// tiles of D = 128, 45% of the counts above 0, 30% above 1, 0.07% above 16: 91 us a pass with the loops in place, 51 with the lists.)
constexpr int LIST = 512;            // cells that a wave makes at a time
template <int WAVES>
struct Lists {
    unsigned short cell[WAVES][LIST + 64];  // row of the wave 4 b | column 7 b | count 5 b (31: or more); 64 places for what is not listed
    unsigned short far[WAVES][128];
    int others[WAVES];               // how many of those a wave has left
    union {
        double f[128];               // forward: of each row: what its sum has beside the listed cells
        float row[128][3];           // backward: of each row: m, coefficient, weight
    };
};

__device__ __forceinline__ int scan16(int v) {  // over the 16 lanes of a row, this one's included
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr: 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
}

template <class T, int TR>
struct Dense {
    static constexpr int NT = TR == 16 ? 256 : 512, WAVES = NT / 64;
    typedef DmeTile<T, TR, DT, (TR == 16 ? 1 : 4), (TR == 16 ? 4 : 2)> Tile;
    static constexpr int USED = TR * ZP * 4 + (int)sizeof(Lists<WAVES>), LDS = Tile::LDS > USED ? Tile::LDS : USED;
    static_assert(2 * LDS <= 160 * 1024, "two workgroups a CU");
};

// Tiles of z with a dense matrix of counts: every value of z may meet a count, so the tile lies in LDS in 32 bits, where a row's
// 16 lanes read it beside the counts, eight neighbouring columns a lane, the next rows' counts on their way.  Bound by vector
// instructions (five sixths of the time at the size above), which is why two workgroups of eight waves share a CU.
template <class T, int TR, bool BACKWARD>
__global__ __launch_bounds__(TR == 16 ? 256 : 512, TR == 16 ? 2 : 4) void dense_kernel(TileArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef typename Dense<T, TR>::Tile Tile;
    constexpr int NT = Dense<T, TR>::NT, WAVES = Dense<T, TR>::WAVES, STEP = NT / 16;  // rows at a time
    long long tr, tc;
    dme_tile_of(blockIdx.x, (u32)a.tiles_r, (u32)a.tiles_c, tr, tc);
    const long long r0 = tr * TR, c0 = tc * DT, k0 = a.column + c0;
    float* z = (float*)lds;
    Lists<WAVES>& lists = *(Lists<WAVES>*)(lds + TR * ZP * 4);
    const int tid = threadIdx.x, sub = tid & 15, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Counts next;
    if (r0 + (tid >> 4) < a.nb) next.load(a.rows, r0 + (tid >> 4), k0 + sub * 8, a.K);
    float m_row = 0.f, cf_row = 0.f, weight_row = 0.f;  // of row `tid`
    if (BACKWARD && tid < TR && r0 + tid < a.nb) {
        m_row = a.largest_z[r0 + tid];
        cf_row = a.coef[r0 + tid];
        weight_row = a.weight[r0 + tid];
    }
    {
        Tile t;
        t.clear();
        t.run(a.h, a.w, a.D, lds, r0, c0, 0, a.slices);
        const bool inside = k0 + DT <= a.K;  // then no lane looks at its columns
#pragma unroll
        for (int i = 0; i < Tile::NI; ++i) {
            const int c = Tile::col_of(i);
            const f32x4 b = inside && a.bias ? *(const f32x4_u*)(a.bias + k0 + c) : bias_of(a, k0 + c);
            const bool out = any_out(b);
#pragma unroll
            for (int j = 0; j < Tile::NJ; ++j) *(f32x4*)(z + Tile::row_of(j) * ZP + c) = with_bias(t.acc[i][j], b, out);
        }
        if (BACKWARD && tid < TR) {
            lists.row[tid][0] = m_row;
            lists.row[tid][1] = cf_row;
            lists.row[tid][2] = weight_row;
        }
    }
    __syncthreads();
    const bool dirichlet = a.likelihood == DME_LIKELIHOOD_DIRICHLET;
    T* dz = (T*)a.dz;
    unsigned short *cell = lists.cell[wave], *far = lists.far[wave];
    const auto fence = [] { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); };
    const auto row_of = [&](int code, int of) { return (code >> 9 & 3) * STEP + of * 4 + (code >> 7 & 3); };
    // a listed cell's value in place of its z
    const auto put = [&](int code, int row, float v, float value) {
        const float* of = lists.row[row];
        z[row * ZP + (code & 127)] = BACKWARD ? exp_of(v, of[0]) * of[1] - of[2] * value : value;
    };
    int filled = 0, others = 0;
    const auto make_other = [&](bool real, int code, int by) {
        const int row = row_of(code, by);
        int x = code >> 11;
        if (x == 31) x = count_at(a.rows, r0 + row, k0 + (code & 127));
        const float v = z[row * ZP + (code & 127)];
        const float value = (float)(BACKWARD ? dirichlet_g((double)v, (double)x) : dirichlet_rest((double)v, (double)x));
        if (real) put(code, row, v, value);
    };
    const auto make = [&] {
        constexpr int N = 2;
        fence();
        for (int e = 0; e < filled; e += 64 * N) {
            int code[N], x[N];
            float v[N], value[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int at = e + u * 64 + lane;
                code[u] = at < filled ? cell[at] : 0;
                x[u] = code[u] >> 11;
                v[u] = z[row_of(code[u], wave) * ZP + (code[u] & 127)];
                const bool other = !is_small(x[u]);
                const u64 b = __builtin_amdgcn_ballot_w64(other);
                if (b) {
                    if (other) {
                        far[others + (int)__builtin_amdgcn_mbcnt_hi((u32)(b >> 32), __builtin_amdgcn_mbcnt_lo((u32)b, 0))] = (unsigned short)code[u];
                        x[u] = 0;
                    }
                    others += __builtin_popcountll(b);
                    fence();
                    if (others >= 64) {
                        make_other(true, far[lane], wave);
                        others -= 64;
                        const unsigned short rest = far[64 + lane];
                        fence();
                        far[lane] = rest;
                        fence();
                    }
                }
            }
            if (BACKWARD)
                small_g(v, x, value);
            else
                small_rest(v, x, value);
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (x[u] > 0) put(code[u], row_of(code[u], wave), v[u], value[u]);
        }
        filled = 0;
        fence();
    };

#pragma unroll 1
    for (int it = 0; it < TR / STEP; ++it) {
        const int row = it * STEP + (tid >> 4);
        const long long r = r0 + row;
        const bool real = r < a.nb;  // the same for all of a row's lanes
        float* zr = z + row * ZP + sub * 8;
        if (__builtin_amdgcn_ballot_w64(real) == 0) {
            if (!BACKWARD) break;
            *(f32x4*)zr = *(f32x4*)(zr + 4) = f32x4{0.f, 0.f, 0.f, 0.f};
            continue;
        }
        int v[8];
        next.get(a.rows.elem, v);
        if (it + 1 < TR / STEP && r + STEP < a.nb) next.load(a.rows, r + STEP, k0 + sub * 8, a.K);
        const f32x4 left = *(const f32x4*)zr, right = *(const f32x4*)(zr + 4);
        const float u[8] = {left[0], left[1], left[2], left[3], right[0], right[1], right[2], right[3]};
        bool listed[8];
        if (dirichlet) {
            int mine = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                listed[q] = real && v[q] > 1;
                mine += listed[q];
            }
            const int upto = scan16(mine), n0 = __builtin_amdgcn_readlane(upto, 15), n1 = __builtin_amdgcn_readlane(upto, 31),
                      n2 = __builtin_amdgcn_readlane(upto, 47), n3 = __builtin_amdgcn_readlane(upto, 63), all = n0 + n1 + n2 + n3;
            if (filled + all > LIST) make();
            const int g = lane >> 4, code = it << 9 | g << 7 | sub * 8;
            int at = filled + upto - mine + (g > 0 ? n0 : 0) + (g > 1 ? n1 : 0) + (g > 2 ? n2 : 0);
            if (all)
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    cell[listed[q] ? at : LIST + lane] = (unsigned short)(code + q | (v[q] < 31 ? v[q] : 31) << 11);
                    at += listed[q];
                }
            filled += all;
        }
        float d[8];  // what takes the place of z; a listed cell waits as it is
        if (!BACKWARD) {
            const float m = max16(fmaxf(fmaxf(fmaxf(u[0], u[1]), fmaxf(u[2], u[3])), fmaxf(fmaxf(u[4], u[5]), fmaxf(u[6], u[7]))));
            const float base = m == -INFINITY ? 0.f : m;
            float s = 0.f, f = 0.f;
            if (!__any(fabsf(base) > FAR)) {
                const Reference e(base);
#pragma unroll
                for (int q = 0; q < 8; ++q) s += e(u[q]);
                s *= e.rest;
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) s += exp_of(u[q], base);
            }
            int counts = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                counts += v[q] > 0;
                f += v[q] > 0 ? (u[q] - base) * (dirichlet ? 1.f : (float)v[q]) : 0.f;
                d[q] = dirichlet && listed[q] ? u[q] : 0.f;
            }
            s = sum16(s);
            const double all = sum16((double)f);
            double t;
            if (a.rows.elem == 2) {
                int total = 0;
#pragma unroll
                for (int q = 0; q < 8; ++q) total += v[q];
                t = (double)sum16(total);
            } else {
                u64 total = 0;
                int least = 0;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    total += (u32)v[q];
                    least = v[q] < least ? v[q] : least;
                }
                t = sum16(least < 0 ? __builtin_nan("") : (double)total);
            }
            const double w = dirichlet ? (double)sum16(counts) : t;
            if (sub == 0 && real) {
                a.part[tc * a.nb + r] = f32x2{m, s};
                a.part_w[tc * a.nb + r] = w;
                a.part_t[tc * a.nb + r] = t;
                if (dirichlet)
                    lists.f[row] = all;
                else
                    a.part_f[tc * a.nb + r] = all;
            }
        } else {
            const float m = lists.row[row][0], cf = lists.row[row][1], weight = lists.row[row][2];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                float e = exp_of(u[q], m) * cf;
                if (v[q] > 0) e -= weight * (dirichlet ? 1.f : (float)v[q]);
                d[q] = !real ? 0.f : dirichlet && listed[q] ? u[q] : e;
            }
            if (!dirichlet && real) {
                dme_store4(dz + r * a.lddz + c0 + sub * 8, f32x4{d[0], d[1], d[2], d[3]});
                dme_store4(dz + r * a.lddz + c0 + sub * 8 + 4, f32x4{d[4], d[5], d[6], d[7]});
            }
        }
        if (BACKWARD || dirichlet) {
            *(f32x4*)zr = f32x4{d[0], d[1], d[2], d[3]};
            *(f32x4*)(zr + 4) = f32x4{d[4], d[5], d[6], d[7]};
        }
    }
    if (dirichlet) {
        make();
        if (lane == 0) lists.others[wave] = others;
        __syncthreads();
        for (int base = wave * 64;; base += NT) {
            int at = base + lane, by = 0, all = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const int n = lists.others[w];
                if (w < WAVES - 1 && base + lane >= all + n) {
                    at = base + lane - all - n;
                    by = w + 1;
                }
                all += n;
            }
            if (base >= all) break;
            const bool in = base + lane < all;
            make_other(in, in ? lists.far[by][at] : 0, in ? by : 0);
        }
        __syncthreads();
        for (int row = tid >> 4; row < TR; row += STEP) {
            const long long r = r0 + row;
            if (r >= a.nb) break;
            const f32x4 left = *(const f32x4*)(z + row * ZP + sub * 8), right = *(const f32x4*)(z + row * ZP + sub * 8 + 4);
            if (!BACKWARD) {
                const f32x4 both = left + right;
                const double f = sum16((double)((both[0] + both[1]) + (both[2] + both[3])));
                if (sub == 0) a.part_f[tc * a.nb + r] = lists.f[row] + f;
            } else {
                dme_store4(dz + r * a.lddz + c0 + sub * 8, left);
                dme_store4(dz + r * a.lddz + c0 + sub * 8 + 4, right);
            }
        }
    }
    if (!BACKWARD || !a.dbias) return;
    __syncthreads();
    const int c = tid % DT, piece = tid / DT;
    constexpr int PIECES = NT / DT;
    float sum = 0.f;
#pragma unroll 4
    for (int row = piece * (TR / PIECES); row < (piece + 1) * (TR / PIECES); ++row) sum += z[row * ZP + c];
    __syncthreads();
    if (piece) z[piece * ZP + c] = sum;
    __syncthreads();
    if (piece || k0 + c >= a.K) return;
#pragma unroll
    for (int q = 1; q < PIECES; ++q) sum += z[q * ZP + c];
    a.dbias[tr * a.K + k0 + c] = sum;
}

struct RowArgs {
    long long nb, K;
    int tiles, kind, likelihood;
    const f32x2* part;
    const double* part_f;
    const double* part_w;
    const double* part_t;
    const float* entry_z;
    Rows rows;
    const float* weights;  // [nb] or null
    float* loss;           // [nb]
    float* largest_z;      // [nb] or null: no gradient is wanted
    float* coef;
    float* weight;
    float* entry_g;        // CSR: [nnz], LABELS: [nb]: weight * G(z, x)
};

// The row's pieces become l, the loss, and what the gradient needs of them, in 64 bits.  Bound by latency: 4099 rows of 196 pieces and
// 35 entries take 10 us.  CSR rows are checked here: columns
// strictly ascending and below K, no negative count, rowptr in order; a row that breaks this has total NaN.
// A workgroup takes 256 / LANES rows.  The pieces lie row beside row, so neighbouring lanes take neighbouring rows there; the counts lie
// entry beside entry, so neighbouring lanes take a row's neighbouring entries.
template <int LANES>
__global__ __launch_bounds__(256) void row_kernel(RowArgs a) {
    constexpr int ROWS = 256 / LANES;
    __shared__ float m_seen[LANES][ROWS];
    __shared__ double s_seen[LANES][ROWS], sums[3][4];
    const long long first = (long long)blockIdx.x * ROWS;
    {
        const int row = threadIdx.x % ROWS, lane = threadIdx.x / ROWS;
        const long long r = first + row < a.nb ? first + row : a.nb - 1;
        float m = -INFINITY;
        double s = 0.0;
        for (int tile = lane; tile < a.tiles; tile += 4 * LANES) {
            f32x2 p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = tile + u * LANES < a.tiles ? a.part[(tile + u * LANES) * a.nb + r] : f32x2{-INFINITY, 0.f};
            const float top = fmaxf(fmaxf(m, fmaxf(p[0][0], p[1][0])), fmaxf(p[2][0], p[3][0])), base = top == -INFINITY ? 0.f : top;
            s *= (double)exp_of(m, base);
#pragma unroll
            for (int u = 0; u < 4; ++u) s += (double)p[u][1] * (double)exp_of(p[u][0], base);
            m = top;
        }
        m_seen[lane][row] = m;
        s_seen[lane][row] = s;
    }
    __syncthreads();
    const int row = threadIdx.x / LANES, sub = threadIdx.x % LANES;
    const long long r = first + row;
    const bool real = r < a.nb;
    const long long rr = real ? r : a.nb - 1;
    float m;
    double s;
    if constexpr (LANES == 16) {
        m = max16(m_seen[sub][row]);
        const float base = m == -INFINITY ? 0.f : m;
        s = sum16(s_seen[sub][row] * (double)exp_of(m_seen[sub][row], base));
    } else {  // one row: each wave makes the same sums of all
        const int l = threadIdx.x & 63;
        m = fmaxf(fmaxf(m_seen[l][0], m_seen[l + 64][0]), fmaxf(m_seen[l + 128][0], m_seen[l + 192][0]));
        m = max16(m);
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const float base = m == -INFINITY ? 0.f : m;
        s = 0.0;
#pragma unroll
        for (int u = 0; u < 256; u += 64) s += s_seen[l + u][0] * (double)exp_of(m_seen[l + u][0], base);
        s = dme_wave_sum_f64(s);
    }
    // the counts: their part of the loss relative to m, their total, and how often m goes into their part
    const bool dirichlet = a.likelihood == DME_LIKELIHOOD_DIRICHLET;
    const double top = (double)m;
    const float weight = a.weights ? a.weights[rr] : 1.f;
    double f = 0.0, total = 0.0, times = 0.0;
    if (a.kind == DENSE) {
        for (int tile = sub; tile < a.tiles; tile += LANES) {
            const long long at = tile * a.nb + rr;
            const double w = a.part_w[at];
            const float mt = a.part[at][0];
            if (w != 0.0) f += a.part_f[at] + w * ((mt == -INFINITY ? 0.0 : (double)mt) - top);
            total += a.part_t[at];
            times += w;
        }
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
            const float z = a.entry_z[e];
            total += (double)x;
            const bool small = dirichlet && x > 0 && is_small(x);
            if (x > 0) {
                times += dirichlet ? 1.0 : (double)x;
                f += ((double)z - top) * (dirichlet ? 1.0 : (double)x);
                if (dirichlet) f += small ? (double)small_rest(z, x) : dirichlet_rest((double)z, (double)x);
            }
            if (a.largest_z && real) a.entry_g[e] = weight * (small ? small_g(z, x) : (float)g_of(a.likelihood, (double)z, (double)x));
        }
        if (bad) total = __builtin_nan("");
    } else if (sub == 0) {  // F(z, 1) = z, G(z, 1) = 1 in both likelihoods
        const long long k = a.rows.labels[rr];
        const bool in = k >= 0 && k < a.K;
        total = k < 0 ? 0.0 : in ? 1.0 : __builtin_nan("");
        f = in ? (double)a.entry_z[rr] - top : 0.0;
        times = in ? 1.0 : 0.0;
        if (a.largest_z && real) a.entry_g[r] = weight;
    }
    if constexpr (LANES == 16) {
        f = sum16(f);
        total = sum16(total);
        times = sum16(times);
    } else {  // through LDS, in the waves' order
        f = dme_wave_sum_f64(f);
        total = dme_wave_sum_f64(total);
        times = dme_wave_sum_f64(times);
        if ((threadIdx.x & 63) == 0) {
            sums[0][threadIdx.x >> 6] = f;
            sums[1][threadIdx.x >> 6] = total;
            sums[2][threadIdx.x >> 6] = times;
        }
        __syncthreads();
        f = (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]);
        total = (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3]);
        times = (sums[2][0] + sums[2][1]) + (sums[2][2] + sums[2][3]);
    }
    // the row's own terms take a thousand instructions in 64 bits: one wave makes the loss of all rows here, one the gradient's coefficients
    const int part = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (LANES == 16 && sub == 0) {
        s_seen[0][row] = s;
        s_seen[1][row] = f;
        s_seen[2][row] = total;
        s_seen[3][row] = times;
        m_seen[0][row] = m;
    }
    __syncthreads();
    if (lane >= ROWS || first + lane >= a.nb) return;
    if constexpr (LANES == 16) {
        s = s_seen[0][lane];
        f = s_seen[1][lane];
        total = s_seen[2][lane];
        times = s_seen[3][lane];
        m = m_seen[0][lane];
    }
    const long long at = first + lane;
    const double over = log(s), l = (double)m + over;
    if (part == 0) {
        double loss = total == total ? -f : total;
        if (dirichlet) {
            loss += over + dirichlet_rest(l, total);
            if (times != 1.0) loss += (1.0 - times) * (double)m;
        } else {
            loss += total * over;
        }
        // both likelihoods are of a sequence of draws, never above 1: what is below 0 is the rounding of z, which was summed in two orders
        // (the tiles' and entries_of's), or of s
        a.loss[at] = total == 0.0 || loss < 0.0 ? 0.f : (float)loss;
    } else if (part == 1 && a.largest_z) {
        const float w = a.weights ? a.weights[at] : 1.f;
        a.largest_z[at] = total == 0.0 ? INFINITY : m;
        a.coef[at] = total == 0.0 ? 0.f : (float)((double)w * g_of(a.likelihood, l, total) / s);
        a.weight[at] = w;
    }
}

struct PatchArgs {
    long long nb, K, column, width;
    Rows rows;
    const float* entry_z;
    const float* entry_g;
    const float* largest_z;
    const float* coef;
    void* dz;
    long long lddz;
    // the counts' column sums for dbias, in the first piece's launch
    u32 blocks, ranges;  // workgroups for them (0: none), ranges of columns
    int range;           // columns of a range
    long long group;     // rows of a group
    double* sums;        // [group of rows][K]
};

// What dbias needs of the counts, entry_g added up by column: a workgroup takes a group of rows and a range of columns, looks through all
// entries of those rows and adds up the range's in LDS, in fixed point, 64 bits wide: sums of whole numbers do not depend on their order.
// Each column has a point of its own, set by its largest entry of the group, which a first look finds: rows of next to no weight have columns of their own
// beside rows of much, and their entries would be lost behind one point for all.  The largest takes 54 bits, which leaves 8 for a group's sum (a row has a
// column once) and holds the 24 bits of entries down to 2^-30 of it whole.  A column with an entry that has left 32 bits is NaN.
// Word frequencies leave few entries of a column together: with atomics in memory, after a hash table in LDS had joined those of 32 rows, 100 000
// of 144 000 were left, and took 25 us; so it is 10, beside the other workgroups.  A group has up to 256 rows, since each leaves K sums, and as many
// entries as the threads hold in two looks, since every range's workgroup looks through all of them (the launch at 4099 rows, 50 000 columns: 24 us with
// groups of 256, 16 with 128).  Ranges are wide and groups large unless too many CUs would be without a workgroup (1024 rows, 10 007 columns: 9 us in
// 32 workgroups, 6 in 160); labels are looked through at once, whatever the group (4000 rows, 1000 columns: 76 us a gradient with 16, 70 with 256).
constexpr int RANGE = 8192, LEAST_RANGE = 1024;  // columns
constexpr int RANGE_BYTES = 8 + 2;   // of LDS for each: its sum and its point
constexpr int MOST_GROUP = 256;      // rows
constexpr int GROUP_ENTRIES = 8192;  // twice what the threads hold at a time
template <int KIND>
__device__ __forceinline__ void sum_counts(const PatchArgs& a, char* lds) {
    constexpr short LOST = 0x7fff;
    const long long group = blockIdx.x / a.ranges, c0 = (long long)(blockIdx.x % a.ranges) * a.range;
    const int width = (int)(a.K - c0 < a.range ? a.K - c0 : a.range);
    u64* sums = (u64*)lds;
    short* point = (short*)(lds + a.range * 8);
    const long long r0 = group * a.group, r1 = r0 + a.group < a.nb ? r0 + a.group : a.nb;
    const long long p0 = KIND == CSR ? row_begin(a.rows, r0) : r0, p1 = KIND == CSR ? row_begin(a.rows, r1) : r1;
    // DEEP entries of a thread at a time; the first ones stay for the second look
    constexpr int DEEP = KIND == CSR ? 8 : 1;
    const auto load = [&](long long e, int (&k)[DEEP], float (&g)[DEEP]) {
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            k[u] = -1;
            g[u] = 0.f;
            if (e + u * 512 < p1) {
                const u64 c = (u64)(KIND == CSR ? (long long)a.rows.col[e + u * 512] : a.rows.labels[e + u * 512]) - (u64)c0;
                k[u] = c < (u64)width ? (int)c : -1;
                g[u] = a.entry_g[e + u * 512];
            }
        }
    };
    int k0[DEEP];
    float g0[DEEP];
    load(p0 + threadIdx.x, k0, g0);
    const auto each = [&](auto take) {
#pragma unroll
        for (int u = 0; u < DEEP; ++u)
            if (k0[u] >= 0) take(k0[u], g0[u]);
        for (long long e = p0 + threadIdx.x + DEEP * 512; e < p1; e += DEEP * 512) {
            int k[DEEP];
            float g[DEEP];
            load(e, k, g);
#pragma unroll
            for (int u = 0; u < DEEP; ++u)
                if (k[u] >= 0) take(k[u], g[u]);
        }
    };
    for (int i = threadIdx.x; i < width; i += 512) sums[i] = 0;
    __syncthreads();
    each([&](int k, float g) { atomicMax((u32*)(sums + k), __builtin_bit_cast(u32, fabsf(g))); });  // ordered like the values
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 512) {
        const float most = __builtin_bit_cast(float, (u32)sums[i]);
        point[i] = !__builtin_isfinite(most) ? LOST : (short)(most > 0.f ? 53 - ilogbf(most) : 0);
        sums[i] = 0;
    }
    __syncthreads();
    each([&](int k, float g) {
        if (point[k] != LOST) atomicAdd(sums + k, (u64)llrint(ldexp((double)g, point[k])));
    });
    __syncthreads();
    for (int i = threadIdx.x; i < width; i += 512)
        a.sums[group * a.K + c0 + i] = point[i] == LOST ? __builtin_nan("") : ldexp((double)(long long)sums[i], -point[i]);
}

// d loss / d z at the counts: the tiles' value made again, minus G, in its place.  LANES lanes a row.  Bound by latency: 4099 rows with 144 000
// entries take 6 us a piece.
template <class T, int KIND, int LANES>
__global__ __launch_bounds__(512) void patch_kernel(PatchArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if (blockIdx.x < a.blocks) return sum_counts<KIND>(a, lds);
    const int sub = threadIdx.x % LANES;
    const long long r = (long long)(blockIdx.x - a.blocks) * (512 / LANES) + threadIdx.x / LANES;
    if (r >= a.nb) return;
    const float m = a.largest_z[r], cf = a.coef[r];
    const long long p0 = KIND == CSR ? row_begin(a.rows, r) : r, p1 = KIND == CSR ? row_begin(a.rows, r + 1) : r + 1;
    for (long long e = p0 + sub; e < p1; e += LANES) {
        const long long k = KIND == CSR ? (long long)a.rows.col[e] : a.rows.labels[r];
        const long long c = k - a.column;
        if (c < 0 || c >= a.width || k >= a.K) continue;
        ((T*)a.dz)[r * a.lddz + c] = (T)(exp_of(a.entry_z[e], m) * cf - a.entry_g[e]);
    }
}

struct ProductArgs {
    DmeOperand p, q;
    long long k;
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
template <class T, int SIDE, bool PK, int STAGES>
__device__ __forceinline__ void product(const ProductArgs& a, u32 block, char* lds) {
    typedef DmeSquare<T, SIDE, PK, true, STAGES> Tile;
    const u32 tiles = (u32)(a.tiles_r * a.tiles_c), split = block / tiles;
    long long tr, tc;
    dme_tile_of(block - split * tiles, (u32)a.tiles_r, (u32)a.tiles_c, tr, tc);
    const int s0 = (int)split * a.per_split;
    int s1 = s0 + a.per_split;
    s1 = s1 < a.slices ? s1 : a.slices;
    Tile t;
    t.clear();
    t.run(a.p, a.q, a.k, lds, tr * SIDE, tc * SIDE, s0, s1);
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
                f32x4* to = (f32x4*)(a.part + split * a.split_stride + r * a.ldpart + c);
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

// Both products of a piece of d loss / d z: dW = dz' H and dH = dz W, in one launch or (no workgroups for the other) one alone.  Their
// tiles are many and few, short and long; together they leave fewer CUs idle than one after the other.  The longer ones begin.
// At D = 128 both are bound by their reads of dz: 4099 x 50000 takes 161 us for twice 410 MB (5.1 TB/s, most of it from the memory-side
// cache); at D = 1024 by the matrix instructions: 8192 x 50000 takes 1550 us (1080 TFLOP/s).
template <class T, int SIDE, int STAGES>
__global__ __launch_bounds__(SIDE >= 192 ? 512 : 256) void products_kernel(ProductArgs w, ProductArgs h, u32 blocks_w, u32 blocks_h, int h_first) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const u32 block = blockIdx.x;
    const bool is_h = h_first ? block < blocks_h : block >= blocks_w;
    if (is_h)
        product<T, SIDE, false, STAGES>(h, h_first ? block : block - blocks_w, lds);
    else
        product<T, SIDE, true, STAGES>(w, h_first ? block - blocks_h : block, lds);
}

// out [R][C] = the sum of `splits` pieces, in their order.  `lines` lines of `length` values, the pieces' `ldpart` apart (a
// multiple of four); one line where there are no gaps.  A wave takes 256 values of a line.
struct JoinArgs {
    const float* part;
    long long ldpart, split_stride;
    int splits;
    long long lines, length;
    void* out;
    int vector;
    u32 blocks;
};

template <class T>
__device__ __forceinline__ void join(const JoinArgs& a, u32 block) {
    const int lane = threadIdx.x & 63;
    const long long across = (a.length + 255) / 256, all = a.lines * across, waves = (long long)a.blocks * 4;
    for (long long t = (long long)block * 4 + (threadIdx.x >> 6); t < all; t += waves) {
        const long long line = across == 1 ? t : t / across, c = (across == 1 ? 0 : t - line * across) * 256 + lane * 4;
        if (c >= a.length) continue;
        const float* at = a.part + line * a.ldpart + c;
        f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
        const auto four = [&](int s, auto last) {  // loads without branches: all on their way at once
            f32x4 p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = *(const f32x4*)(at + (!last || s + u < a.splits ? s + u : s) * a.split_stride);
#pragma unroll
            for (int u = 0; u < 4; ++u) v += !last || s + u < a.splits ? p[u] : f32x4{0.f, 0.f, 0.f, 0.f};
        };
        int s = 0;
        for (; s + 4 <= a.splits; s += 4) four(s, std::false_type());
        if (s < a.splits) four(s, std::true_type());
        T* o = (T*)a.out + line * a.length + c;
        if (a.vector) {
            dme_store4(o, v);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < a.length) o[q] = (T)v[q];
        }
    }
}

// dbias [K] (+)= the row tiles' sums, minus the counts'.  64 columns a workgroup, a quarter of the
// tiles a wave, the quarters added in their order.
struct BiasArgs {
    const float* part;
    long long tiles, K;
    const double* sums;  // [groups][K], or null: dense rows
    long long groups;
    int add;
    float* dbias;
    u32 blocks;
};

__device__ __forceinline__ void add_bias(const BiasArgs& a, u32 block, double (*sums)[64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long k = (long long)block * 64 + lane;
    double v = 0.0;
    if (k < a.K) {
        for (long long t = wave; t < a.tiles; t += 16) {
            float p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u] = t + u * 4 < a.tiles ? a.part[(t + u * 4) * a.K + k] : 0.f;
#pragma unroll
            for (int u = 0; u < 4; ++u) v += (double)p[u];
        }
        if (a.sums)
            for (long long t = wave; t < a.groups; t += 16) {
                double p[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) p[u] = t + u * 4 < a.groups ? a.sums[(t + u * 4) * a.K + k] : 0.0;
#pragma unroll
                for (int u = 0; u < 4; ++u) v -= p[u];
            }
    }
    sums[wave][lane] = v;
    __syncthreads();
    if (wave != 0 || k >= a.K) return;
    v = (sums[0][lane] + sums[1][lane]) + (sums[2][lane] + sums[3][lane]);
    if (a.add) v += (double)a.dbias[k];
    a.dbias[k] = (float)v;
}

// What is left when the products are through, in one launch (10 us at 4099 x 50000 x 128, 20 MB of pieces): the pieces of dH and dW, and dbias (0 workgroups: not this time).
template <class T>
__global__ __launch_bounds__(256) void finish_kernel(JoinArgs w, JoinArgs h, BiasArgs b) {
    __shared__ double sums[4][64];
    u32 block = blockIdx.x;
    if (block < w.blocks) return join<T>(w, block);
    block -= w.blocks;
    if (block < h.blocks) return join<T>(h, block);
    add_bias(b, block - h.blocks, sums);
}

inline long long up(long long v, long long to) { return (v + to - 1) / to * to; }

// Everything a call decides before its first launch.
struct Plan {
    int size;                 // bytes of a value
    bool pack_h, pack_w;      // the operand is copied with a pitch of whole 16-byte chunks first
    long long dpad;           // k of the first product in a packed operand
    long long nb;             // rows of a block
    int side;                 // of the tiles of z: 256, 128, 64, or 16 rows x 128 columns
    bool few;                 // the forward pass goes by few_kernel
    long long tile_rows, tile_cols;
    long long tiles;          // pieces that the forward pass leaves of a row
    long long chunk;          // columns of a piece of d loss / d z
    bool together;            // the two products of a piece go out in one launch
    DmePair cut_w, cut_h;     // how they are cut: one cut for both, or each its own
    bool pieces_w, pieces_h;  // the products leave 32-bit pieces
    long long ldpart;
    long long group;          // rows of a group of the counts' column sums
    // places in the workspace
    long long sums, h, w, part, part_f, part_w, part_t, entry_z, entry_g, largest_z, coef, weight, dbias, dz, pw, ph, bytes;
};

inline long long few_lds(long long bytes) { return 16 * (up(bytes, 64) + 64); }

Plan make_plan(const void* H, long long ldh, const void* W, long long ldw, int type, long long N, long long K, long long D,
               const dme_count_rows_t* rows, bool gradient) {
    Plan p{};
    p.group = 16;
    p.size = type == DME_TYPE_BF16 ? 2 : 4;
    const auto loose = [&](const void* at, long long ld) {
        return ((uintptr_t)at | (uintptr_t)(ld * p.size) | (uintptr_t)(D * p.size)) % 16 != 0;
    };
    p.dpad = up(D, 16 / p.size);
    p.nb = std::min(std::max(N, 1ll), gradient ? ROW_BLOCK : LOSS_BLOCK);
    while (p.nb * K > MOST_CELLS) p.nb = (p.nb + 1) / 2;
    const long long slices = (D * p.size + DME_SLICE - 1) / DME_SLICE;
    const int cut = dme_cut(p.nb, K, slices, p.size, false, 4.0).side;
    p.side = p.nb <= 16 ? 16 : rows->kind == DENSE ? 128 : cut >= 192 ? 256 : cut;
    p.tile_rows = p.side;
    p.tile_cols = p.side == 16 ? 128 : p.side;
    const long long tiles = (K + p.tile_cols - 1) / p.tile_cols;
    // up to 16 rows, while they fit into the LDS that needs no attribute
    p.few = p.side == 16 && rows->kind != DENSE && few_lds(D * p.size) <= 61440;
    p.tiles = p.few ? (K + 63) / 64 : tiles;
    // few rows' losses read every weight once: from anywhere, where a copy would be two passes more
    // (1 x 50000 x 511 in bf16: 36 us with it, 26 without; 7 x 20011 x 201 in fp32: 23, 17)
    p.pack_h = loose(H, ldh) && (gradient || !p.few);
    p.pack_w = loose(W, ldw) && (gradient || !p.few);
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long here = at;
        at += up(bytes, 256);
        return here;
    };
    if (p.pack_h) p.h = take(p.nb * p.dpad * p.size);
    if (p.pack_w) p.w = take(K * p.dpad * p.size);
    const long long forward = at;
    p.part = take(p.tiles * p.nb * 8);
    if (rows->kind == DENSE) {
        p.part_f = take(p.tiles * p.nb * 8);
        p.part_w = take(p.tiles * p.nb * 8);
        p.part_t = take(p.tiles * p.nb * 8);
    }
    if (gradient) {  // the sums for dbias lie where the forward pass's pieces were: row_kernel, the launch before theirs, is the last to read those
        const long long end = at;
        at = forward;
        if (rows->kind != DENSE) {
            const double entries = rows->kind == CSR ? (double)rows->nnz / (double)std::max(N, 1ll) : 1.0;  // of a row
            const auto workgroups = [&](long long group) { return (p.nb + group - 1) / group * ((K + LEAST_RANGE - 1) / LEAST_RANGE); };
            while (p.group < MOST_GROUP && 2 * p.group * entries <= GROUP_ENTRIES && (rows->kind == LABELS || workgroups(2 * p.group) >= 128)) p.group *= 2;
            p.sums = take((p.nb + p.group - 1) / p.group * K * 8);
        }
        p.dbias = take((p.nb + p.tile_rows - 1) / p.tile_rows * K * 4);
        at = std::max(at, end);
    }
    if (rows->kind != DENSE) p.entry_z = take((rows->kind == CSR ? rows->nnz : p.nb) * 4);
    if (gradient) {
        if (rows->kind != DENSE) p.entry_g = take((rows->kind == CSR ? rows->nnz : p.nb) * 4);
        p.largest_z = take(p.nb * 4);
        p.coef = take(p.nb * 4);
        p.weight = take(p.nb * 4);
        long long c = PIECE_BYTES / (p.nb * p.size) / p.tile_cols;
        if (c < 1) c = 1;
        if (c > tiles) c = tiles;
        const long long pieces = (tiles + c - 1) / c;
        p.chunk = (tiles + pieces - 1) / pieces * p.tile_cols;  // pieces of like width
        p.dz = take(p.nb * p.chunk * p.size);
        p.ldpart = up(D, 4);
        const auto slices_of = [&](long long k) { return (k * p.size + DME_SLICE - 1) / DME_SLICE; };
        const long long width = p.chunk < K ? p.chunk : K;
        // Together they fill the card better; where a piece's rows are long each fills it alone, and side by side they only take the caches
        // from each other (N = 4099, D = 128: 229 us apart, 162 together; N = 8192, D = 1024: 1567 apart, 1690 together; D = 256: alike).
        p.together = D <= 512;
        if (p.together) {
            p.cut_w = p.cut_h = dme_pair(width, slices_of(p.nb), p.nb, slices_of(width), D, p.size, N > p.nb, pieces > 1);
        } else {
            const DmeCut w = dme_cut(width, D, slices_of(p.nb), p.size, true), h = dme_cut(p.nb, D, slices_of(width), p.size, true);
            p.cut_w = DmePair{w.side, w.splits, 1, w.us};
            p.cut_h = DmePair{h.side, 1, h.splits, h.us};
        }
        p.pieces_w = p.cut_w.splits_w > 1 || N > p.nb;
        p.pieces_h = p.cut_h.splits_h > 1 || pieces > 1;
        if (p.pieces_w) p.pw = take((long long)p.cut_w.splits_w * K * p.ldpart * 4);
        if (p.pieces_h) p.ph = take((long long)p.cut_h.splits_h * p.nb * p.ldpart * 4);
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

template <class T, int TR, int TC, int WR, int WC, int KIND, bool BACKWARD, int STAGES = 0>
int launch_tile(const TileArgs& a, hipStream_t s) {
    typedef DmeTile<T, TR, TC, WR, WC, false, false, STAGES> Tile;
    static_assert(Tile::LDS >= WC * TR * 8 && Tile::LDS >= WR * TC * 4, "the reductions use the tiles' LDS");
    static std::atomic<bool> done[64];
    constexpr int turned = BACKWARD && sizeof(T) == 2 && TR >= 128 ? TR * WC * (Tile::WTC * (int)sizeof(T) + 16) : 0;
    constexpr int bytes = turned > Tile::LDS ? turned : Tile::LDS;
    const int rc = set_lds(done, tile_kernel<T, TR, TC, WR, WC, KIND, BACKWARD, STAGES>, bytes);
    if (rc) return rc;
    const long long more = BACKWARD ? 0 : (a.nb + Tile::NW - 1) / Tile::NW;
    hipLaunchKernelGGL((tile_kernel<T, TR, TC, WR, WC, KIND, BACKWARD, STAGES>), dim3((unsigned)(a.tiles_r * a.tiles_c + more)), dim3(Tile::NT), bytes, s, a);
    return DME_OK;
}

template <class T, int KIND, bool BACKWARD>
int launch_side(const TileArgs& a, int side, hipStream_t s) {
    if (side == 256) return launch_tile<T, 256, 256, 4, 2, KIND, BACKWARD>(a, s);
    if (side == 128) return launch_tile<T, 128, 128, 2, 2, KIND, BACKWARD>(a, s);
    if (side == 64) {  // a deep pipeline where a CU has one or two of them, two buffers where it can hold five
        if (a.tiles_r * a.tiles_c > 512) return launch_tile<T, 64, 64, 2, 2, KIND, BACKWARD, 2>(a, s);
        return launch_tile<T, 64, 64, 2, 2, KIND, BACKWARD>(a, s);
    }
    return launch_tile<T, 16, 128, 1, 4, KIND, BACKWARD>(a, s);
}

template <class T, int TR, bool BACKWARD>
int launch_dense(const TileArgs& a, hipStream_t s) {
    typedef Dense<T, TR> D;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, dense_kernel<T, TR, BACKWARD>, D::LDS);
    if (rc) return rc;
    hipLaunchKernelGGL((dense_kernel<T, TR, BACKWARD>), dim3((unsigned)(a.tiles_r * a.tiles_c)), dim3(D::NT), D::LDS, s, a);
    return DME_OK;
}

// The tiles of z, forward with z at the counts.
template <class T, bool BACKWARD>
int tiles_of_z(const TileArgs& a, int kind, int side, hipStream_t s) {
    if (kind == DENSE) return side == 16 ? launch_dense<T, 16, BACKWARD>(a, s) : launch_dense<T, 128, BACKWARD>(a, s);
    if (!BACKWARD && kind == CSR) return launch_side<T, CSR, false>(a, side, s);
    return launch_side<T, LABELS, BACKWARD>(a, side, s);  // backward the kind does not matter
}

template <class T, int SIDE, int STAGES = 0>
int launch_products(ProductArgs w, ProductArgs h, const DmePair& cut, bool do_w, bool do_h, hipStream_t s) {
    typedef DmeSquare<T, SIDE, true, true, STAGES> Tile;
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, products_kernel<T, SIDE, STAGES>, Tile::LDS);
    if (rc) return rc;
    const auto lay = [](ProductArgs& a, int splits) {
        a.tiles_r = (a.p.rows + SIDE - 1) / SIDE;
        a.tiles_c = (a.q.rows + SIDE - 1) / SIDE;
        a.slices = (int)((a.k * (long long)sizeof(T) + DME_SLICE - 1) / DME_SLICE);
        a.per_split = (a.slices + splits - 1) / splits;
        return (u32)(a.tiles_r * a.tiles_c * splits);
    };
    const u32 blocks_w = do_w ? lay(w, cut.splits_w) : 0, blocks_h = do_h ? lay(h, cut.splits_h) : 0;
    hipLaunchKernelGGL((products_kernel<T, SIDE, STAGES>), dim3(blocks_w + blocks_h), dim3(Tile::NT), Tile::LDS, s, w, h, blocks_w, blocks_h,
                       (int)(h.per_split > w.per_split));
    return DME_OK;
}

template <class T>
int products(const ProductArgs& w, const ProductArgs& h, const DmePair& cut, bool do_w, bool do_h, hipStream_t s) {
    if (cut.side == 256) return launch_products<T, 256>(w, h, cut, do_w, do_h, s);
    if (cut.side == 192) return launch_products<T, 192>(w, h, cut, do_w, do_h, s);
    if (cut.side == 128) return launch_products<T, 128>(w, h, cut, do_w, do_h, s);
    const long long along = (w.q.rows + 63) / 64;
    const long long all = ((w.p.rows + 63) / 64 * cut.splits_w * do_w + (h.p.rows + 63) / 64 * cut.splits_h * do_h) * along;
    if (all > 512) return launch_products<T, 64, 2>(w, h, cut, do_w, do_h, s);
    return launch_products<T, 64>(w, h, cut, do_w, do_h, s);
}

template <class T, int KIND, int LANES>
int launch_patch(const PatchArgs& a, unsigned lds, hipStream_t s) {
    static std::atomic<bool> done[64];
    const int rc = set_lds(done, patch_kernel<T, KIND, LANES>, RANGE * RANGE_BYTES);
    if (rc) return rc;
    constexpr int rows = 512 / LANES;
    hipLaunchKernelGGL((patch_kernel<T, KIND, LANES>), dim3(a.blocks + (unsigned)((a.nb + rows - 1) / rows)), dim3(512), lds, s, a);
    return DME_OK;
}

JoinArgs join_args(const void* part, long long ldpart, long long split_stride, int splits, long long R, long long C, void* out) {
    const bool whole = ldpart == C;
    JoinArgs a{(const float*)part, ldpart, split_stride, splits, whole ? 1 : R, whole ? R * C : C, out, (int)(C % 4 == 0), 0};
    a.blocks = (u32)dme_blocks(a.lines * ((a.length + 255) / 256), 4, 8192);
    return a;
}

// both in one launch; either may have no rows
void pack(const DmePack& a, const DmePack& b, hipStream_t s) {
    const dim3 grid(dme_blocks(a.rows + b.rows, 4, 16384)), block(256);
    uintptr_t all = 0;  // widths are multiples of 16
    for (const DmePack* p : {&a, &b})
        if (p->rows > 0) all |= (uintptr_t)p->src | (uintptr_t)(p->rows > 1 ? p->pitch : 0) | (uintptr_t)p->bytes | (uintptr_t)p->width;
    if (all % 8 == 0)
        hipLaunchKernelGGL(dme_pack_kernel<u64>, grid, block, 0, s, a, b);
    else if (all % 4 == 0)
        hipLaunchKernelGGL(dme_pack_kernel<u32>, grid, block, 0, s, a, b);
    else
        hipLaunchKernelGGL(dme_pack_kernel<unsigned short>, grid, block, 0, s, a, b);
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
    DmePack pack_w{};
    if (p.pack_w) {
        pack_w = DmePack{w.at, w.ld, c.K, c.D * size, ws + p.w, p.dpad * size};
        w = DmeOperand{ws + p.w, p.dpad * size, c.K};
    }
    double* sums = gradient && kind != DENSE && c.dbias ? (double*)(ws + p.sums) : nullptr;
    for (long long n0 = 0; n0 < c.N; n0 += p.nb) {
        const long long nb = c.N - n0 < p.nb ? c.N - n0 : p.nb;
        DmeOperand h{(const char*)c.H + n0 * c.ldh * size, c.ldh * size, nb};
        DmePack pack_h{};
        if (p.pack_h) {
            pack_h = DmePack{h.at, h.ld, nb, c.D * size, ws + p.h, p.dpad * size};
            h = DmeOperand{ws + p.h, p.dpad * size, nb};
        }
        if (pack_h.rows + pack_w.rows > 0) pack(pack_h, pack_w, s);
        pack_w.rows = 0;  // once
        TileArgs a{};
        a.h = h;
        a.w = w;
        a.D = c.D;
        a.tiles_r = (nb + p.tile_rows - 1) / p.tile_rows;
        a.tiles_c = p.tiles;
        a.slices = (int)((c.D * size + DME_SLICE - 1) / DME_SLICE);
        a.row_bytes = (int)((p.pack_h ? p.dpad : c.D) * size);  // rows that are not whole chunks: both operands are packed, or neither
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
        a.part_w = (double*)(ws + p.part_w);
        a.part_t = (double*)(ws + p.part_t);
        a.entry_z = (float*)(ws + p.entry_z);
        int rc = DME_OK;
        if (p.few) {
            const unsigned blocks = (unsigned)(p.tiles + nb), bytes = (unsigned)few_lds(c.D * size);
            const bool loose = a.row_bytes % 16 || ((uintptr_t)h.at | (uintptr_t)h.ld | (uintptr_t)w.at | (uintptr_t)w.ld) % 16;
            if (kind == CSR && loose)
                hipLaunchKernelGGL((few_kernel<T, CSR, true>), dim3(blocks), dim3(256), bytes, s, a);
            else if (kind == CSR)
                hipLaunchKernelGGL((few_kernel<T, CSR, false>), dim3(blocks), dim3(256), bytes, s, a);
            else if (loose)
                hipLaunchKernelGGL((few_kernel<T, LABELS, true>), dim3(blocks), dim3(256), bytes, s, a);
            else
                hipLaunchKernelGGL((few_kernel<T, LABELS, false>), dim3(blocks), dim3(256), bytes, s, a);
        } else {
            rc = tiles_of_z<T, false>(a, kind, p.side, s);
        }
        if (rc) return rc;
        RowArgs ra{};
        ra.nb = nb;
        ra.K = c.K;
        ra.tiles = (int)p.tiles;
        ra.kind = kind;
        ra.likelihood = c.likelihood;
        ra.part = a.part;
        ra.part_f = a.part_f;
        ra.part_w = a.part_w;
        ra.part_t = a.part_t;
        ra.entry_z = a.entry_z;
        ra.rows = rows;
        ra.loss = c.loss + n0;
        if (gradient) {
            ra.weights = c.weights ? c.weights + n0 : nullptr;
            ra.largest_z = (float*)(ws + p.largest_z);
            ra.coef = (float*)(ws + p.coef);
            ra.weight = (float*)(ws + p.weight);
            ra.entry_g = (float*)(ws + p.entry_g);
        }
        const unsigned groups = (unsigned)(nb <= FEW_ROWS ? nb : (nb + 15) / 16);
        if (nb <= FEW_ROWS)
            hipLaunchKernelGGL(row_kernel<256>, dim3(groups), dim3(256), 0, s, ra);
        else
            hipLaunchKernelGGL(row_kernel<16>, dim3(groups), dim3(256), 0, s, ra);
        if (!gradient) continue;
        a.largest_z = ra.largest_z;
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
                PatchArgs pa{nb, c.K, k0, width, rows, a.entry_z, ra.entry_g, ra.largest_z, ra.coef, a.dz, a.lddz};
                unsigned lds = 0;
                if (sums && k0 == 0) {
                    const long long row_groups = (nb + p.group - 1) / p.group;
                    pa.range = RANGE;
                    while (pa.range > LEAST_RANGE && row_groups * ((c.K + pa.range - 1) / pa.range) < 256) pa.range /= 2;
                    pa.ranges = (u32)((c.K + pa.range - 1) / pa.range);
                    pa.blocks = (u32)row_groups * pa.ranges;
                    pa.group = p.group;
                    pa.sums = sums;
                    lds = (unsigned)pa.range * RANGE_BYTES;
                }
                rc = kind == CSR ? launch_patch<T, CSR, 16>(pa, lds, s) : launch_patch<T, LABELS, 1>(pa, lds, s);
                if (rc) return rc;
            }
            const char* dz = (const char*)a.dz;
            ProductArgs mw{}, mh{};
            mw.p = DmeOperand{dz, a.lddz * size, width};  // dW of the piece = dz' H
            mw.q = DmeOperand{h.at, h.ld, c.D};
            mw.k = nb;
            if (p.pieces_w) {
                mw.part = (float*)(ws + p.pw) + k0 * p.ldpart;
                mw.ldpart = p.ldpart;
                mw.split_stride = c.K * p.ldpart;
                mw.add = n0 > 0;
            } else {
                mw.out = (T*)c.dW + k0 * c.D;
                mw.ldout = c.D;
                mw.vector = c.D % 4 == 0;
            }
            mh.p = DmeOperand{dz, a.lddz * size, nb};  // dH (+)= dz W
            mh.q = DmeOperand{a.w.at, a.w.ld, c.D};
            mh.k = width;
            if (p.pieces_h) {
                mh.part = (float*)(ws + p.ph);
                mh.ldpart = p.ldpart;
                mh.split_stride = p.nb * p.ldpart;
                mh.add = k0 > 0;
            } else {
                mh.out = (T*)c.dH + n0 * c.D;
                mh.ldout = c.D;
                mh.vector = c.D % 4 == 0;
            }
            if (p.together) {
                rc = products<T>(mw, mh, p.cut_w, true, true, s);
            } else {
                rc = products<T>(mw, mh, p.cut_w, true, false, s);
                if (!rc) rc = products<T>(mw, mh, p.cut_h, false, true, s);
            }
            if (rc) return rc;
        }
        JoinArgs jw{}, jh{};
        BiasArgs bias{};
        if (p.pieces_w && n0 + nb == c.N) jw = join_args(ws + p.pw, p.ldpart, c.K * p.ldpart, p.cut_w.splits_w, c.K, c.D, c.dW);
        if (p.pieces_h) jh = join_args(ws + p.ph, p.ldpart, p.nb * p.ldpart, p.cut_h.splits_h, nb, c.D, (T*)c.dH + n0 * c.D);
        if (c.dbias)
            bias = BiasArgs{a.dbias, a.tiles_r, c.K, sums, (nb + p.group - 1) / p.group, (int)(n0 > 0), c.dbias, (u32)((c.K + 63) / 64)};
        const u32 blocks = jw.blocks + jh.blocks + bias.blocks;
        if (blocks) hipLaunchKernelGGL(finish_kernel<T>, dim3(blocks), dim3(256), 0, s, jw, jh, bias);
    }
    DME_HIP_CHECK(hipGetLastError());
    return DME_OK;
}

int check_call(const void* H, int64_t ldh, const void* W, int64_t ldw, int type, int64_t N, int64_t K, int64_t D, const dme_count_rows_t* rows,
               int likelihood) {
    DME_REQUIRE(type == DME_TYPE_BF16 || type == DME_TYPE_F32, "features and weights are bf16 or fp32");
    DME_REQUIRE(N >= 0 && K >= 1 && D >= 1, "bad shape: N = %lld, K = %lld, D = %lld", (long long)N, (long long)K, (long long)D);
    DME_REQUIRE(K <= (1ll << 29) && D <= (1ll << 20) && N <= (1ll << 40), "shape out of range");
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
        pack(DmePack{nullptr, 0, K, 0, (char*)dW, D * size}, DmePack{nullptr, 0, dbias ? 1 : 0, 0, (char*)dbias, K * 4}, (hipStream_t)stream);
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
