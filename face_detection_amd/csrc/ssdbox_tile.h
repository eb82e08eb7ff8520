// Matrix product of one tile per workgroup for the classifier losses (gfx950): out[n][m] = sum_k A[m][k] B[n][k],
// m the index that is contiguous in the result.  Both operands go from HBM to LDS without passing registers
// (global_load_lds, 16 bytes a lane), one K tile of 128 bytes a row ahead of the matrix instructions.
//
// An operand lies in memory either with k contiguous (rows of m or n) or with m / n contiguous (rows of k).  The first
// kind is read from LDS as 16 bytes of k per lane; the second is transposed on the way out of LDS (ds_read_b64_tr_b16; plain
// 4-byte reads for float32).  So the gradients read the weight, the hidden rows and the logits' gradient as they are.
//
// LDS holds 16-byte pieces in an order that keeps the reads off each other's banks; since a global_load_lds writes its
// lanes' pieces back to back, the order is made by which piece each lane asks for:
//   rows of k pieces:  piece c of row r at position c ^ (r & 7)              (eight rows of one read on eight positions)
//   rows of k, 16 bit: 32-byte granule at position ^ ((k & 3) | (k >> 3 & 1) << 2), float32: 64-byte granule ^ (k >> 2 & 3)
#pragma once

#include "ssdbox_internal.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int kRowBytes = 128;       // one K tile of an operand whose rows hold k: 64 values of 16 bits, 32 of float32

template <typename T>
struct TileNum;

template <>
struct TileNum<bf16_t> {
    static SSD_DEV void mma(f32x4 &c, u32x4 a, u32x4 b)
    {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

template <>
struct TileNum<f16_t> {
    static SSD_DEV void mma(f32x4 &c, u32x4 a, u32x4 b)
    {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

template <>
struct TileNum<float> {
    // Four values of k a lane: the j-th instruction takes k = 4 * (lane / 16) + j of both operands.
    static SSD_DEV void mma(f32x4 &c, u32x4 a, u32x4 b)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(u2f(a[j]), u2f(b[j]), c, 0, 0, 0);
    }
};

// What lanes ask for that lie beyond the last k: zeros, so that the tile's rest adds nothing.
static __device__ __align__(16) const unsigned kZeroPiece[4] = {0u, 0u, 0u, 0u};

SSD_DEV unsigned lds_address(const void *p)
{
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char *)p;
}

// A value that is the same in all lanes, in scalar registers.
SSD_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
SSD_DEV const char *uniform(const char *p)
{
    const unsigned long long u = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
    return (const char *)((unsigned long long)hi << 32 | lo);
}

// 64 lanes x 16 bytes to LDS at `lds` (wave-uniform, lanes back to back).  No register receives the data and nothing waits
// here: the caller waits on vmcnt before a barrier and reads after it.
SSD_DEV void load_to_lds(unsigned lds, const char *base, unsigned offset)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 :
                 : "s"(uniform((int)lds)), "v"(offset), "s"(uniform(base))
                 : "memory");
}

SSD_DEV void load_to_lds_at(unsigned lds, const char *address)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(uniform((int)lds)), "v"(address)
                 : "memory");
}

// One operand of a tile: E rows (of m or n), BK values of k.
//   KROWS false: memory rows are m / n, k contiguous;  KROWS true: memory rows are k.
template <typename T, int E, bool KROWS, int THREADS>
struct TileOperand {
    static constexpr int kPieces = E * kRowBytes / 16;
    static constexpr int kPer = kPieces / THREADS;
    static constexpr int kBK = kRowBytes / (int)sizeof(T);
    static constexpr int kVec = 16 / (int)sizeof(T);
    static constexpr int kPiecesPerRow = KROWS ? E * (int)sizeof(T) / 16 : kRowBytes / 16;
    static_assert(kPieces % THREADS == 0, "every lane loads in every step");

    const char *base;                // this tile's first row at the K tile to be loaded next
    unsigned offset[kPer];           // this lane's pieces, bytes from base
    unsigned lds;                    // wave's first piece in buffer 0
    long long step;                  // bytes from one K tile to the next

    // row of k (KROWS) or first k (otherwise) that piece i of this lane covers, within the K tile
    static SSD_DEV int piece_k(int i)
    {
        const int c = i * THREADS + (int)threadIdx.x;
        const int row = c / kPiecesPerRow, pos = c % kPiecesPerRow;
        return KROWS ? row : (pos ^ (row & 7)) * kVec;
    }

    // extent: rows of m / n there are from e0 on (at least 1); ld in values
    SSD_DEV void init(const void *p, long long ld, long long e0, int extent, long long k0, const char *smem)
    {
        const long long ldb = ld * (int)sizeof(T);
        base = uniform((const char *)p + (KROWS ? k0 * ldb + e0 * (int)sizeof(T) : e0 * ldb + k0 * (int)sizeof(T)));
        step = KROWS ? kBK * ldb : kRowBytes;
        lds = lds_address(smem) + (unsigned)uniform(threadIdx.x / 64) * 1024u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = i * THREADS + (int)threadIdx.x;
            const int row = c / kPiecesPerRow, pos = c % kPiecesPerRow;
            if (KROWS) {
                int src;
                if (sizeof(T) == 2)
                    src = (((pos >> 1) ^ ((row & 3) | ((row >> 3 & 1) << 2))) << 1) | (pos & 1);
                else
                    src = (((pos >> 2) ^ (row >> 2 & 3)) << 2) | (pos & 3);
                if (src * kVec >= extent) src = 0;       // columns beyond the last are read from the first: never stored
                offset[i] = (unsigned)((long long)row * ldb) + (unsigned)src * 16u;
            } else {
                const int r = row < extent ? row : extent - 1;
                offset[i] = (unsigned)((long long)r * ldb) + (unsigned)((pos ^ (row & 7)) * 16);
            }
        }
    }

    // left: values of k from this K tile on
    SSD_DEV void load(unsigned buffer_bytes, int left)
    {
        if (left >= kBK) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) load_to_lds(lds + buffer_bytes + i * THREADS * 16u, base, offset[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const char *a = piece_k(i) < left ? base + offset[i] : (const char *)kZeroPiece;
                load_to_lds_at(lds + buffer_bytes + i * THREADS * 16u, a);
            }
        }
        base += step;
    }

    // the fragment of rows e .. e + 15 (e a multiple of 16), half ks of the K tile
    static SSD_DEV u32x4 fragment(const char *tile, int e, int ks)
    {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
        if constexpr (!KROWS) {
            return *(const u32x4 *)(tile + (e + i) * kRowBytes + (((ks * 4 + g) ^ (i & 7)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const int r = i >> 2, f = r | (g & 1) << 2;
            const char *p = tile + (ks * 32 + 8 * g + r) * (E * 2) + (((e >> 4) ^ f) << 5) + (i & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * E * 2));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const char *p = tile + (ks * 16 + 4 * g) * (E * 4) + (((e >> 4) ^ g) << 6) + i * 4;
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *(const unsigned *)(p + j * E * 4);
            return v;
        }
    }
};

// acc[mi][nj][i]: m = 16 mi + 4 (lane / 16) + i, n = 16 nj + lane % 16 of the wave's part of the tile.
template <typename T, int BM, int BN, int WM, int WN, bool A_KROWS, bool B_KROWS>
struct TileProduct {
    static constexpr int kThreads = WM * WN * 64;
    static constexpr int MF = BM / WM / 16, NF = BN / WN / 16;
    static constexpr int kBuffer = (BM + BN) * kRowBytes;
    static constexpr int kLds = 2 * kBuffer;
    typedef TileOperand<T, BM, A_KROWS, kThreads> OpA;
    typedef TileOperand<T, BN, B_KROWS, kThreads> OpB;
    static constexpr int kBK = OpA::kBK;

    // k: values of k there are from the K tile `first` on the operands were set to
    static SSD_DEV void run(OpA &a, OpB &b, int k, const char *smem, f32x4 (&acc)[MF][NF])
    {
        const int wave = uniform(threadIdx.x / 64);
        const int em = (wave / WN) * (BM / WM), en = (wave % WN) * (BN / WN);
#pragma unroll
        for (int mi = 0; mi < MF; ++mi)
#pragma unroll
            for (int nj = 0; nj < NF; ++nj) acc[mi][nj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (k <= 0) return;
        // float32: a long chain of additions rounds as often as it has links, so each K tile's 32 values are summed apart
        constexpr bool kTwice = sizeof(T) == 4;
        f32x4 all[kTwice ? MF : 1][kTwice ? NF : 1];
        if constexpr (kTwice)
#pragma unroll
            for (int mi = 0; mi < MF; ++mi)
#pragma unroll
                for (int nj = 0; nj < NF; ++nj) all[mi][nj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        a.load(0, k);
        b.load(0, k);
        unsigned cur = 0;
        for (int left = k; left > 0; left -= kBK) {
            // every wave's pieces of this K tile have landed, and no wave reads the other buffer any more
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            const unsigned next = cur ^ kBuffer;
            if (left > kBK) {
                a.load(next, left - kBK);
                b.load(next, left - kBK);
            }
            const char *ta = smem + cur, *tb = smem + BM * kRowBytes + cur;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                u32x4 fb[NF];
#pragma unroll
                for (int nj = 0; nj < NF; ++nj) fb[nj] = OpB::fragment(tb, en + nj * 16, ks);
#pragma unroll
                for (int mi = 0; mi < MF; ++mi) {
                    const u32x4 fa = OpA::fragment(ta, em + mi * 16, ks);
#pragma unroll
                    for (int nj = 0; nj < NF; ++nj) TileNum<T>::mma(acc[mi][nj], fa, fb[nj]);
                }
            }
            cur = next;
            if constexpr (kTwice)
#pragma unroll
                    for (int mi = 0; mi < MF; ++mi)
#pragma unroll
                        for (int nj = 0; nj < NF; ++nj) {
                            all[mi][nj] += acc[mi][nj];
                            acc[mi][nj] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        }
        }
        if constexpr (kTwice)
#pragma unroll
            for (int mi = 0; mi < MF; ++mi)
#pragma unroll
                for (int nj = 0; nj < NF; ++nj) acc[mi][nj] += all[mi][nj];
    }
};

// Which tile workgroup `id` of `tm * tn` takes: consecutive workgroups run on different XCDs, so each XCD is given
// one run of the tile order, and the order goes through `group` tiles of n before the next m (an XCD's 32 workgroups then
// share operands in its L2).
SSD_DEV void tile_of(int id, int tm, int tn, int group, int &m, int &n)
{
    const int total = tm * tn, q = total / 8, r = total % 8, x = id % 8;
    const int t = x * q + (x < r ? x : r) + id / 8;
    const int per = group * tm, gi = t / per, first = gi * group;
    const int width = tn - first < group ? tn - first : group;
    const int rem = t - gi * per;
    n = first + rem % width;
    m = rem / width;
}
