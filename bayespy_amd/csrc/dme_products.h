// dme_products.h — the tile product that the regression operators are made of: out[r][c] = sum_k P[r][k] Q[c][k],
// on the matrix cores, 32-bit sums.
//
// A workgroup of NW = WR x WC waves makes a tile of TR x TC outputs.  k goes by slices of 128 bytes (64 bf16 / fp16,
// 32 fp32 values): a slice of the tile's TR + TC rows is copied from memory straight into LDS (16 bytes a lane, no
// registers in between), two buffers (four for small tiles, whose products are short beside the memory's answer), so that the
// copies of later slices fly while slice s is multiplied.  A row's eight
// 16-byte chunks are stored at chunk ^ (row & 7): lanes of a wave that read the same chunk of 8 neighbouring rows then
// touch all banks once.  Both operands may also lie the other way round ("k-major", see DmeTile).  Q is the matrix instruction's first operand, so a lane ends up with ONE r (lane & 15) and four
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

// An operand of a product: `rows` rows of k values, either with k contiguous (ld: bytes from row to row; what follows the
// row's k values up to a multiple of 16 bytes is zero), or "k-major", with the rows contiguous (ld: bytes from one k to the next;
// what follows the rows up to a multiple of 16 bytes may be read and is not used).  Base and ld are multiples of 16 bytes.
struct DmeOperand {
    const char* at;
    long long ld;
    long long rows;
};

constexpr int DME_SLICE = 128;  // bytes of k in a slice

// 16 bytes a lane from memory to LDS at `to` + lane * 16 (`to` uniform).  In assembly because the compiler waits for every copy it knows
// of before a transposing LDS read, whatever buffer that reads; who calls this waits with s_waitcnt vmcnt(0) itself.  No register
// is written.  One wait state belongs between a write of m0 and its use here.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is reserved: that is why its change is said
__device__ __forceinline__ void dme_copy_to_lds(const char* from, u32 to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory", "m0");
}
#pragma clang diagnostic pop

// What products read in place of what lies outside an operand.  Never written.
static __device__ __attribute__((aligned(256))) u32 dme_zeros[64];

// The product of a TR x TC tile.  PK / QK: the operand is k-major.
//
// A k-major slice lies in LDS as it does in memory, one line of TR (TC) values for each k.  16-bit operands are turned by the
// transposing LDS read (16 lanes read 4 lines of 16 values, each lane gets one row's 4 k), 32-bit ones by four reads of a
// word.  The 16 lines that a wave reads at once begin in the same bank, so the 16-value groups of line k are stored at
// group ^ f(k), f spreading them over the banks.
template <class T, int TR, int TC, int WR, int WC, bool PK = false, bool QK = false, int STAGES_ = 0>
struct DmeTile {
    static constexpr int TR_ = TR, TC_ = TC, NW = WR * WC, NT = NW * 64;
    static constexpr int WTR = TR / WR, WTC = TC / WC;  // a wave's part
    static constexpr int NJ = WTR / 16, NI = WTC / 16;  // its 16 x 16 blocks
    static constexpr int STAGE = (TR + TC) * DME_SLICE;  // bytes of one buffer
    static constexpr int STAGES = STAGES_ ? STAGES_ : TR + TC <= 144 ? 4 : 2;
    static constexpr int LDS = STAGES * STAGE;
    static constexpr int COPIES = (TR + TC) / 8;         // wave copies (1 KB) of one slice
    static constexpr int PER_WAVE = (COPIES + NW - 1) / NW;
    static constexpr int SIZE = sizeof(T);
    static constexpr int KS = DME_SLICE / SIZE;  // k of a slice
    static constexpr int KH = KS / 2;            // k of one instruction round (64 bytes)

    f32x4 acc[NI][NJ];

    // where line k of a k-major operand of TM rows keeps its groups of 16 values
    template <int TM>
    __device__ __forceinline__ static int spread(int k) {
        if (SIZE == 4) return (k >> 2) & 3;
        return TM % 128 ? ((k >> 1) & 1) | ((k >> 3) & 1) << 1 : (k & 3) | ((k >> 3) & 1) << 2;
    }

    // source of one lane's 16 bytes of piece `piece` (1 KB) of an operand, and in how many slices from the first on it lies
    // inside the operand
    template <int TM, bool KMAJOR>
    __device__ __forceinline__ static void source(const DmeOperand& o, long long first, long long K, int piece, int lane, const char*& src, int& limit) {
        if (!KMAJOR) {
            const int chunk = (lane & 7) ^ (lane >> 3);  // piece * 8 rows do not change row & 7
            long long r = first + piece * 8 + (lane >> 3);
            r = r < o.rows ? r : o.rows - 1;  // rows beyond the last are not used: any will do
            src = o.at + r * o.ld + chunk * 16;
            const long long bytes = K * SIZE - chunk * 16;
            limit = bytes > 0 ? (int)((bytes + DME_SLICE - 1) / DME_SLICE) : 0;
        } else {
            constexpr int LINE = TM * SIZE / 16;  // 16-byte chunks of a line
            const int at = piece * 64 + lane, k = at / LINE, slot = at % LINE;
            const int chunk = slot ^ (spread<TM>(k) * SIZE);  // a group is SIZE chunks
            const long long r = first + chunk * (16 / SIZE);
            src = o.at + k * o.ld + r * SIZE;
            limit = r < o.rows && k < K ? (int)((K - k + KS - 1) / KS) : 0;
        }
    }

    // block b (16 rows) of an operand's slice in LDS, round h: this lane's 16 bytes of k
    template <int TM, bool KMAJOR>
    __device__ __forceinline__ static u32q fragment(const char* at, int b, int h) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        if (!KMAJOR) return *(const u32q*)(at + (b * 16 + c) * DME_SLICE + ((h * 4 + g) ^ (lane & 7)) * 16);
        constexpr int LINE = TM * SIZE;
        if constexpr (SIZE == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* lds_ptr;
            const int k = h * KH + 8 * g + (c >> 2);  // + 4: the same spread
            const char* p = at + k * LINE + (b ^ spread<TM>(k)) * 32 + (c & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 4 * LINE));
            return __builtin_bit_cast(u32q, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int k = h * KH + 4 * g;
            const char* p = at + k * LINE + (b ^ spread<TM>(k)) * 64 + c * 4;
            u32q v;
#pragma unroll
            for (int s = 0; s < 4; ++s) v[s] = *(const u32*)(p + s * LINE);
            return v;
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // acc += the tile at (r0, c0) over the slices [s0, s1) of k < K.  lds: LDS bytes, free for the caller afterwards (a
    // barrier has been passed).  Every thread of the workgroup calls this.
    __device__ __forceinline__ void run(const DmeOperand& P, const DmeOperand& Q, long long K, char* lds, long long r0, long long c0, int s0, int s1) {
        const char *p[1] = {P.at}, *q[1] = {Q.at};
        run(P, Q, p, q, K, lds, r0, c0, s0, s1);
    }

    // acc += the sum of PARTS products whose operands lie alike, part i at p[i] and q[i] (P.at, Q.at are not used), as one run of slices.
    template <int PARTS>
    __device__ __forceinline__ void run(const DmeOperand& P, const DmeOperand& Q, const char* const (&p)[PARTS], const char* const (&q)[PARTS],
                                        long long K, char* lds, long long r0, long long c0, int s0, int s1) {
        if (s0 >= s1) return;
        const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const char* src[PER_WAVE];
        int limit[PER_WAVE];
        const long long pstep = PK ? KS * P.ld : DME_SLICE, qstep = QK ? KS * Q.ld : DME_SLICE;
#pragma unroll
        for (int t = 0; t < PER_WAVE; ++t) {
            const int piece = t * NW + wave;
            if (piece < TR / 8) {
                source<TR, PK>(DmeOperand{p[0], P.ld, P.rows}, r0, K, piece, lane, src[t], limit[t]);
                src[t] += s0 * pstep;
            } else {
                source<TC, QK>(DmeOperand{q[0], Q.ld, Q.rows}, c0, K, piece - TR / 8, lane, src[t], limit[t]);
                src[t] += s0 * qstep;
            }
        }
        const u32 to = (u32)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
        int slice = s0, part = 0;  // the next one to be copied
        auto copy = [&](int buf) {
#pragma unroll
            for (int t = 0; t < PER_WAVE; ++t) {
                const int piece = t * NW + wave;
                if (COPIES % NW == 0 || piece < COPIES) {
                    const char* from = slice < limit[t] ? src[t] : (const char*)dme_zeros;
                    dme_copy_to_lds(from, to + buf * STAGE + piece * 1024);
                    src[t] += piece < TR / 8 ? pstep : qstep;
                }
            }
            ++slice;
            if (PARTS > 1 && slice == s1 && part + 1 < PARTS) {
                slice = s0;
                long long dp = 0, dq = 0;  // from this part's end to the next one's beginning
#pragma unroll
                for (int i = 0; i + 1 < PARTS; ++i)
                    if (part == i) {
                        dp = p[i + 1] - p[i];
                        dq = q[i + 1] - q[i];
                    }
                dp -= (s1 - s0) * pstep;
                dq -= (s1 - s0) * qstep;
                ++part;
#pragma unroll
                for (int t = 0; t < PER_WAVE; ++t) src[t] += t * NW + wave < TR / 8 ? dp : dq;
            }
        };
        const int wr = wave / WC * NJ, wc = wave % WC * NI;
        auto half = [&](const char* at, int h) {
            u32q x[NJ], y[NI];
#pragma unroll
            for (int j = 0; j < NJ; ++j) x[j] = fragment<TR, PK>(at, wr + j, h);
#pragma unroll
            for (int i = 0; i < NI; ++i) y[i] = fragment<TC, QK>(at + TR * DME_SLICE, wc + i, h);
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = dme_mma(y[i], x[j], acc[i][j], T());
        };
        auto multiply = [&](const char* at) {
            half(at, 0);
            half(at, 1);
        };
        // 32 bits: the last slice by itself, whose second half may lie beyond K (1024 x 10007 x 100: three and a half slices instead of four, 144 ->
        // 141 us).  In 16 bits a half is few instructions, and the longer code costs more (4099 x 50000 x 128: 504 -> 515).
        constexpr bool APART = SIZE == 4;
        const int n = (s1 - s0) * PARTS, body = APART ? n - 1 : n;
        const bool whole = !APART || K * SIZE > (long long)s1 * DME_SLICE - DME_SLICE / 2;
        if constexpr (STAGES == 2) {
            copy(0);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            for (int u = 0; u < body; ++u) {
                if (APART || u + 1 < n) copy((u + 1) & 1);
                multiply(lds + (u & 1) * STAGE);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // slice u + 1 is in LDS ...
                __syncthreads();                                  // ... and everybody has read slice u
            }
        } else {
            // every wave issues COPIES / NW copies of a slice at least, so that many times the slices that may still be on their
            // way are what it may have outstanding (copies come back in their order)
            constexpr int AHEAD = STAGES - 2, OUT = AHEAD * (COPIES / NW);
            static_assert(OUT < 64, "vmcnt has six bits");
#pragma unroll
            for (int u = 0; u < STAGES - 1; ++u)
                if (u < n) copy(u);
            for (int u = 0; u < body; ++u) {
                if (u + AHEAD < n)
                    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OUT) : "memory");
                else
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                __syncthreads();  // slice u is in LDS, and everybody has read slice u - 1
                if (u + STAGES - 1 < n) copy((u + STAGES - 1) % STAGES);
                multiply(lds + u % STAGES * STAGE);
            }
            if (APART) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
        if (APART) {
            half(lds + body % STAGES * STAGE, 0);
            if (whole) half(lds + body % STAGES * STAGE, 1);
            __syncthreads();
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
__device__ __forceinline__ u32 dme_xcd_order(u32 block, u32 n) {
    const u32 per = n / 8, more = n % 8, x = block & 7;
    return x * per + (x < more ? x : more) + (block >> 3);
}
__device__ __forceinline__ void dme_tile_of(u32 block, u32 tiles_r, u32 tiles_c, long long& tr, long long& tc) {
    u32 t = dme_xcd_order(block, tiles_r * tiles_c);  // fits: the launch has as many workgroups
    const u32 band = t / (8 * tiles_c), first = band * 8;
    const u32 high = tiles_r - first < 8 ? tiles_r - first : 8;
    t -= first * tiles_c;
    tr = first + t % high;
    tc = t / high;
}

// dst (rows of `width` bytes) = src (rows of `bytes` bytes, `pitch` apart), zero in what is more.
struct DmePack {
    const char* src;
    long long pitch, rows, bytes;
    char* dst;
    long long width;
};

// Two of them, in values of V (as many bytes as every row's beginning and length allow).  A wave takes a row.
template <class V>
__global__ __launch_bounds__(256) void dme_pack_kernel(DmePack a, DmePack b) {
    constexpr long long SIZE = sizeof(V);
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows + b.rows; r += (long long)gridDim.x * 4) {
        const bool first = r < a.rows;
        const long long line = first ? r : r - a.rows, bytes = first ? a.bytes : b.bytes, width = first ? a.width : b.width;
        const char* src = first ? a.src + line * a.pitch : b.src + line * b.pitch;
        char* dst = first ? a.dst + line * a.width : b.dst + line * b.width;
        for (long long c = (threadIdx.x & 63) * SIZE; c < width; c += 256 * SIZE) {
            V v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = c + u * 64 * SIZE < bytes ? *(const V*)(src + c + u * 64 * SIZE) : V(0);
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (c + u * 64 * SIZE < width) *(V*)(dst + c + u * 64 * SIZE) = v[u];
        }
    }
}

inline int dme_blocks(long long work, long long per, long long most) {
    long long b = (work + per - 1) / per;
    return (int)(b < 1 ? 1 : b > most ? most : b);
}

// The waves of a SIDE x SIDE tile.
template <class T, int SIDE, bool PK = false, bool QK = false, int STAGES = 0>
using DmeSquare = DmeTile<T, SIDE, SIDE, (SIDE == 256 ? 4 : 2), (SIDE == 192 ? 4 : 2), PK, QK, STAGES>;

// How a product of R x C outputs over `slices` slices of k is cut: tiles of 256, 192, 128 or 64 a side, and into how many pieces
// of k.  Measured in bf16 (fp32) at 4096^3 and 8192^3: 256 a side, one workgroup to a CU, 1150-1290 (141) TFLOP/s; 192, one to a CU, 960-1010;
// 128, two to a CU, 910-1110 (138); 64, two to a CU, 600 (105).  Small products are bound by how many CUs have a tile at all, and
// pieces of k cost a pass over their 32-bit sums.
struct DmeCut {
    int side, splits;
    double us;
};
struct DmeKind {
    int side, per_cu;
    double bf16, f32;  // in FLOP / us
};
constexpr DmeKind DME_KINDS[] = {{256, 1, 1200e6, 141e6}, {192, 1, 1000e6, 135e6}, {128, 2, 980e6, 138e6}, {64, 2, 600e6, 105e6}};

// us of one slice of one tile while the CU's other places are taken too
inline double dme_slice_us(const DmeKind& kind, int size) {
    return (double)kind.side * kind.side * (DME_SLICE / size) * 2.0 * 256.0 * kind.per_cu / (size == 4 ? kind.f32 : kind.bf16);
}
// ... and of a piece of k while they are not, in its share.  (Whole products gain less: told the same of those, 2048 x 2048 steps took smaller
// tiles and 500 us instead of 447.)
constexpr double DME_ALONE = 0.75;
// us of writing and adding up pieces of 32-bit sums
inline double dme_join_us(int splits, double values) { return splits > 1 ? 4.0 + splits * values * 8.0 / 4e6 : 0.0; }

// into how many pieces `slices` slices go when they are cut into `splits` of the same length, rounded up: the others would have none
inline int dme_pieces(long long slices, long long splits) {
    const long long each = (slices + splits - 1) / splits;
    return each > 0 ? (int)((slices + each - 1) / each) : 1;
}

// `products`: how many a slice costs (the sum of as many products is made)
inline DmeCut dme_cut(long long R, long long C, long long slices, int size, bool split, double extra_per_tile_us = 0.0, bool symmetric = false,
                      long long batch = 1, int products = 1) {
    DmeCut best{0, 1, 0.0};
    for (const DmeKind& kind : DME_KINDS) {
        const int side = kind.side, per_cu = kind.per_cu;
        const long long along = (R + side - 1) / side, slots = 256ll * per_cu;
        const long long tiles = batch * (symmetric ? along * (along + 1) / 2 : along * ((C + side - 1) / side));
        const double slice = dme_slice_us(kind, size);
        const auto consider = [&](long long s) {
            if (s > 1 && slices * products / s < 2) return;
            s = dme_pieces(slices, s);
            const double rounds = (double)((tiles * s + slots - 1) / slots);
            const double each = s > 1 && tiles * s <= 256 && per_cu > 1 ? DME_ALONE * slice : slice;
            const double us = rounds * ((double)((slices + s - 1) / s * products + 2) * each + extra_per_tile_us * side * side / 65536.0 * per_cu) +
                              dme_join_us((int)s, (double)batch * R * C);
            if (best.side == 0 || us < best.us) best = DmeCut{side, (int)s, us};
        };
        for (int s = 1; s <= (split ? 64 : 1); s *= 2) consider(s);
        if (split && tiles > 0 && tiles < 256) consider(256 / tiles < 64 ? 256 / tiles : 64);  // a tile for every CU
    }
    return best;
}

// The same for two products launched together, Rw x C over sw slices and Rh x C over sh: one side for both, each with its own pieces
// of k.  The workgroups go out as CUs fall free, so what counts is the whole work over the card and, at its end, about half of the
// shorter kind.  `joined_w`, `joined_h`: the product leaves 32-bit sums in any case.
struct DmePair {
    int side, splits_w, splits_h;
    double us;
};
inline DmePair dme_pair(long long Rw, long long sw, long long Rh, long long sh, long long C, int size, bool joined_w, bool joined_h) {
    DmePair best{0, 1, 1, 0.0};
    for (const DmeKind& kind : DME_KINDS) {
        const long long side = kind.side, across = (C + side - 1) / side, tw = (Rw + side - 1) / side * across, th = (Rh + side - 1) / side * across;
        const double slots = 256.0 * kind.per_cu, slice = dme_slice_us(kind, size);
        for (int cuts_w = 1; cuts_w <= 64 && (cuts_w == 1 || sw / cuts_w >= 2); cuts_w *= 2)
            for (int cuts_h = 1; cuts_h <= 64 && (cuts_h == 1 || sh / cuts_h >= 2); cuts_h *= 2) {
                const int a = dme_pieces(sw, cuts_w), b = dme_pieces(sh, cuts_h);
                const double lw = (double)((sw + a - 1) / a + 2), lh = (double)((sh + b - 1) / b + 2);
                const double whole = ((double)tw * a * lw + (double)th * b * lh) / slots, last = lw < lh ? lw : lh, longest = lw < lh ? lh : lw;
                double us = whole + 0.5 * last;
                if (us < longest) us = longest;
                us = us * slice + dme_join_us(joined_w && a == 1 ? 2 : a, (double)Rw * C) + dme_join_us(joined_h && b == 1 ? 2 : b, (double)Rh * C);
                if (best.side == 0 || us < best.us) best = DmePair{(int)side, a, b, us};
            }
    }
    return best;
}
