// dme_products.h — the tile product that the regression operators are made of: out[r][c] = sum_k P[r][k] Q[c][k],
// both operands with k contiguous, on the matrix cores, 32-bit sums.
//
// A workgroup of NW = WR x WC waves makes a tile of TR x TC outputs.  k goes by slices of 128 bytes (64 bf16 / fp16,
// 32 fp32 values): a slice of the tile's TR + TC rows is copied from memory straight into LDS (16 bytes a lane, no
// registers in between), two buffers, so that the copies of slice s + 1 fly while slice s is multiplied.  A row's eight
// 16-byte chunks are stored at chunk ^ (row & 7): lanes of a wave that read the same chunk of 8 neighbouring rows then
// touch all banks once.  Q is the matrix instruction's first operand, so a lane ends up with ONE r (lane & 15) and four
// neighbouring c: rows are reduced and stored in vectors.
#pragma once
#include "dme_common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef u32 u32q __attribute__((ext_vector_type(4)));

// 16 bytes of k of one operand row.  For fp32 the four values of a lane go to four instructions of four k each: the
// lanes' k then are 4 * (lane >> 4) + step instead of step * 4 + (lane >> 4), the same set for both operands.
__device__ __forceinline__ f32x4 dme_mma(const u32q& q, const u32q& p, f32x4 acc, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q), __builtin_bit_cast(bf16x8, p), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 dme_mma(const u32q& q, const u32q& p, f32x4 acc, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q), __builtin_bit_cast(f16x8, p), acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 dme_mma(const u32q& q, const u32q& p, f32x4 acc, float) {
    const f32x4 a = __builtin_bit_cast(f32x4, q), b = __builtin_bit_cast(f32x4, p);
#pragma unroll
    for (int s = 0; s < 4; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], acc, 0, 0, 0);
    return acc;
}

template <class T>
__device__ __forceinline__ void dme_store4(T* to, f32x4 v) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
    *(t4*)to = o;
}

// Operands of one product.  Rows are clamped to the last real one (their outputs are not used), k beyond kbytes is read
// from `zeros` (16 zero bytes); base pointers and pitches are multiples of 16 bytes (dme_pack_kernel sees to that).
struct DmeOperands {
    const char* P;
    const char* Q;
    long long ldp, ldq;  // pitches in bytes
    long long R, C;      // rows of P, rows of Q
    long long kbytes;    // bytes of k in a row, a multiple of 16
    const char* zeros;
};

constexpr int DME_SLICE = 128;  // bytes of k in a slice

template <class T, int TR, int TC, int WR, int WC>
struct DmeTile {
    static constexpr int NW = WR * WC, NT = NW * 64;
    static constexpr int WTR = TR / WR, WTC = TC / WC;  // a wave's part
    static constexpr int NJ = WTR / 16, NI = WTC / 16;  // its 16 x 16 blocks
    static constexpr int STAGE = (TR + TC) * DME_SLICE;  // bytes of one buffer
    static constexpr int COPIES = (TR + TC) * 8 / 64;    // wave copies (1 KB) of one slice
    static constexpr int PER_WAVE = (COPIES + NW - 1) / NW;

    f32x4 acc[NI][NJ];

    // acc = the tile at (r0, c0) over the slices [s0, s1).  lds: 2 * STAGE bytes, free for the caller afterwards (a
    // barrier has been passed).  Every thread of the workgroup calls this.
    __device__ __forceinline__ void run(const DmeOperands& o, char* lds, long long r0, long long c0, int s0, int s1) {
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int chunk = (lane & 7) ^ (lane >> 3);  // the chunk of k this lane copies, whatever the row group
        const char* src[PER_WAVE];
#pragma unroll
        for (int t = 0; t < PER_WAVE; ++t) {
            const int row = (t * NW + wave) * 8 + (lane >> 3);
            if (row < TR) {
                long long r = r0 + row;
                r = r < o.R ? r : o.R - 1;
                src[t] = o.P + r * o.ldp + chunk * 16;
            } else {
                long long c = c0 + (row - TR);
                c = c < o.C ? c : o.C - 1;
                src[t] = o.Q + c * o.ldq + chunk * 16;
            }
        }
        auto copy = [&](int s, int buf) {
            const long long k = (long long)s * DME_SLICE;
            const bool in = k + chunk * 16 < o.kbytes;
#pragma unroll
            for (int t = 0; t < PER_WAVE; ++t) {
                const int piece = t * NW + wave;
                if (COPIES % NW == 0 || piece < COPIES) {
                    const char* from = in ? src[t] + k : o.zeros;
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                                     (__attribute__((address_space(3))) void*)(lds + buf * STAGE + piece * 1024), 16, 0, 0);
                }
            }
        };
        const int wr = wave / WC, wc = wave % WC;
        const int swz = lane & 7, g = lane >> 4;
        const int prow = (wr * WTR + (lane & 15)) * DME_SLICE, qrow = (TR + wc * WTC + (lane & 15)) * DME_SLICE;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        copy(s0, 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        for (int s = s0; s < s1; ++s) {
            const int buf = (s - s0) & 1;
            if (s + 1 < s1) copy(s + 1, buf ^ 1);
            const char* at = lds + buf * STAGE;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int off = ((h * 4 + g) ^ swz) * 16;
                u32q p[NJ], q[NI];
#pragma unroll
                for (int j = 0; j < NJ; ++j) p[j] = *(const u32q*)(at + prow + j * 16 * DME_SLICE + off);
#pragma unroll
                for (int i = 0; i < NI; ++i) q[i] = *(const u32q*)(at + qrow + i * 16 * DME_SLICE + off);
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < NJ; ++j) acc[i][j] = dme_mma(q[i], p[j], acc[i][j], T());
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // slice s + 1 is in LDS ...
            __syncthreads();                                  // ... and everybody has read slice s
        }
    }

    // this lane's r and first c of block (i, j), relative to the tile
    __device__ __forceinline__ static int row_of(int j) {
        const int tid = threadIdx.x;
        return (tid >> 6) / WC * WTR + j * 16 + (tid & 15);
    }
    __device__ __forceinline__ static int col_of(int i) {
        const int tid = threadIdx.x;
        return (tid >> 6) % WC * WTC + i * 16 + ((tid & 63) >> 4) * 4;
    }
};

// Which tile a workgroup makes.  Workgroups go round the 8 XCDs one by one, and each XCD has an L2 of its own: XCD x
// takes the x-th eighth of the tiles, in columns of 8 row tiles, so that the operand rows that its 32 CUs read at the
// same time overlap.
__device__ __forceinline__ void dme_tile_of(long long block, long long tiles_r, long long tiles_c, long long& tr, long long& tc) {
    const long long n = tiles_r * tiles_c;
    const long long per = n / 8, more = n % 8, x = block & 7, at = block >> 3;
    long long t = x * per + (x < more ? x : more) + at;
    const long long band = t / (8 * tiles_c), first = band * 8;
    const long long high = tiles_r - first < 8 ? tiles_r - first : 8;
    t -= band * 8 * tiles_c;
    tr = first + t % high;
    tc = t / high;
}

// dst [rows][ldd bytes] = src [rows][cols] (any pitch and alignment), zero beyond cols: a row pitch of whole slices.
template <class T>
__global__ void dme_pack_kernel(const T* src, long long lds_, long long rows, long long cols, T* dst, long long ldd) {
    const long long n = rows * ldd;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const long long r = i / ldd, c = i - r * ldd;
        dst[i] = c < cols ? src[r * lds_ + c] : (T)0.f;
    }
}

// dst [cols][ldd] = transpose of src [rows][cols], zero beyond rows (ldd >= rows, in elements).
template <class T>
__global__ void dme_transpose_kernel(const T* src, long long lds_, long long rows, long long cols, T* dst, long long ldd) {
    __shared__ T tile[64][65];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const long long tiles_c = (cols + 63) / 64, tiles_r = (ldd + 63) / 64;
    for (long long t = blockIdx.x; t < tiles_c * tiles_r; t += gridDim.x) {
        const long long r0 = t / tiles_c * 64, c0 = t % tiles_c * 64;
        for (int y = ty; y < 64; y += 4) {
            const long long r = r0 + y, c = c0 + tx;
            tile[y][tx] = r < rows && c < cols ? src[r * lds_ + c] : (T)0.f;
        }
        __syncthreads();
        for (int y = ty; y < 64; y += 4) {
            const long long c = c0 + y, r = r0 + tx;
            if (c < cols && r < ldd) dst[c * ldd + r] = tile[tx][y];
        }
        __syncthreads();
    }
}

inline int dme_blocks(long long work, long long per, long long most) {
    long long b = (work + per - 1) / per;
    return (int)(b < 1 ? 1 : b > most ? most : b);
}
