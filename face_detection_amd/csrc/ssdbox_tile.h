// Matrix products of the classifier losses (gfx950): out[n][m] = sum_k A[m][k] B[n][k], m the index that is contiguous in
// the result, computed as a stream of tiles per workgroup.
//
// A workgroup walks through its tiles, and each tile through stages of 64 bytes of k (32 values of 16
// bits, 16 of float32).  Both operands of a stage go from HBM to LDS without passing registers (global_load_lds, 16
// bytes a lane) into one of four buffers, three stages and more ahead of their use and across the tiles' borders, so
// that a tile's first stages arrive while the epilogue of the tile before runs.  Of a stage, the fragments of one half of k
// are read from LDS while the matrix instructions of the other half run.  One barrier a stage, between its halves:
//
//   first half:  MFMA on half 0 (in registers), read half 1 from buffer s
//   barrier:     every wave has read buffer s; stage s + 1 has landed (all but the two youngest stages' loads are back)
//   second half: load stage s + 4 into buffer s, read half 0 of stage s + 1, MFMA on half 1
//
// An operand lies in memory either with k contiguous (rows of m or n) or with m / n contiguous (rows of k).  The first
// kind is read from LDS as 16 bytes of k per lane; the second is transposed on the way out of LDS (ds_read_b64_tr_b16; plain
// 4-byte reads for float32).  So the gradients read the weight, the hidden rows and the logits' gradient as they are.
//
// LDS holds 16-byte pieces in an order that keeps the lanes that are read in one clock (256 bytes, 64 banks) off each
// other's banks; since a global_load_lds writes its lanes' pieces back to back, the order is made by which piece each lane
// asks for:
//   k contiguous:   piece c (of 4) of row r at c ^ (r >> 2 & 3): sixteen rows' pieces cover 256 bytes
//   rows of k, 16 bit: 32-byte granule at its index ^ (k & 3) << 1: of four rows two granules each
//   rows of k, float32: 128-byte block at its index ^ (k >> 2 & 1): of two rows one block each
#pragma once

#include "ssdbox_internal.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStageBytes = 64;      // of k, per row of m or n
constexpr int kStages = 4;           // buffers in LDS

template <typename T>
struct TileNum;

template <>
struct TileNum<bf16_t> {
    static SSD_DEV void mma(f32x16 &c, u32x4 a, u32x4 b)
    {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

template <>
struct TileNum<f16_t> {
    static SSD_DEV void mma(f32x16 &c, u32x4 a, u32x4 b)
    {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

template <>
struct TileNum<float> {
    // Four values of k a lane: the j-th instruction takes k = 4 * (lane / 32) + j of both operands.
    static SSD_DEV void mma(f32x16 &c, u32x4 a, u32x4 b)
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(u2f(a[j]), u2f(b[j]), c, 0, 0, 0);
    }
};

// What lanes ask for that lie beyond the last k: zeros, so that the stage's rest adds nothing.
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
// here: the stream waits on vmcnt before a barrier and reads after it.
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

// One operand of a stage: E rows (of m or n).  KROWS false: memory rows are m / n, k contiguous;  true: memory rows are k.
template <typename T, int E, bool KROWS, int THREADS>
struct TileOperand {
    static constexpr int kPer = E * kStageBytes / 16 / THREADS;          // 16-byte pieces a lane
    static constexpr int kBK = kStageBytes / (int)sizeof(T);
    static constexpr int kVec = 16 / (int)sizeof(T);
    static constexpr int kPiecesPerRow = KROWS ? E * (int)sizeof(T) / 16 : kStageBytes / 16;
    static_assert(kPer >= 1 && (!KROWS || E >= 128), "every lane loads, and a row of k has eight granules");

    const char *base;                // first row of the tile at the next stage's k
    unsigned offset[kPer];           // this lane's pieces, bytes from base
    long long step;                  // bytes from one stage to the next

    static SSD_DEV int granule(int k) { return (k & 3) << 1; }

    // row of k (KROWS) or first k (otherwise) that piece i of this lane covers, within the stage
    static SSD_DEV int piece_k(int i)
    {
        const int c = i * THREADS + (int)threadIdx.x;
        const int row = c / kPiecesPerRow, pos = c % kPiecesPerRow;
        return KROWS ? row : (pos ^ (row >> 2 & 3)) * kVec;
    }

    // extent: rows of m / n there are from e0 on (at least 1; with KROWS a multiple of a piece); ld in values
    SSD_DEV void init(const void *p, long long ld, long long e0, int extent, long long k0)
    {
        const long long ldb = ld * (int)sizeof(T);
        base = uniform((const char *)p + (KROWS ? k0 * ldb + e0 * (int)sizeof(T) : e0 * ldb + k0 * (int)sizeof(T)));
        step = KROWS ? kBK * ldb : kStageBytes;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int c = i * THREADS + (int)threadIdx.x;
            const int row = c / kPiecesPerRow, pos = c % kPiecesPerRow;
            if (KROWS) {
                int src = sizeof(T) == 2 ? (((pos >> 1) ^ granule(row)) << 1) | (pos & 1) : pos ^ (row >> 2 & 1) << 3;
                if (src * kVec >= extent) src = 0;       // columns beyond the last are read from the first: never stored
                offset[i] = (unsigned)((long long)row * ldb) + (unsigned)src * 16u;
            } else {
                const int r = row < extent ? row : extent - 1;
                offset[i] = (unsigned)((long long)r * ldb) + (unsigned)((pos ^ (row >> 2 & 3)) * 16);
            }
        }
    }

    // piece i of a whole stage to `lds` (the wave's first piece's place)
    SSD_DEV void load_whole(unsigned lds, int i) const { load_to_lds(lds + i * THREADS * 16u, base, offset[i]); }

    // left: values of k from this stage on; none: the stage is not wanted, zeros keep the count of loads in flight
    SSD_DEV void load(unsigned lds, int left) const
    {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const char *a = piece_k(i) < left ? base + offset[i] : (const char *)kZeroPiece;
            load_to_lds_at(lds + i * THREADS * 16u, a);
        }
    }

    // the fragment of rows e .. e + 31 (e a multiple of 32), half ks of the stage: 16 bytes of k a lane
    static SSD_DEV u32x4 fragment(const char *tile, int e, int ks)
    {
        const int lane = threadIdx.x & 63;
        if constexpr (!KROWS) {
            const int row = e + (lane & 31);
            return *(const u32x4 *)(tile + row * kStageBytes + (((ks * 2 + (lane >> 5)) ^ (row >> 2 & 3)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds4;
            const int i = lane & 15, g = lane >> 4, r = i >> 2;
            const int k = ks * 16 + 8 * (g >> 1) + r;
            const char *p = tile + k * (E * 2) + ((((e >> 4) + (g & 1)) ^ r << 1) << 5) + (i & 3) * 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * E * 2));
            return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const char *p = tile + (ks * 8 + 4 * (lane >> 5)) * (E * 4) + ((e ^ (lane >> 5) << 5) + (lane & 31)) * 4;
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *(const unsigned *)(p + j * E * 4);
            return v;
        }
    }
};

struct TileUnit {                    // a tile (or a part of its k)
    int m0, n0, k0, k;               // first m, n and k, and how many values of k
    int part;
};

// Which of `total` units a workgroup, the `block`-th of `blocks`, takes, in turn.  Consecutive workgroups run on different XCDs,
// so each XCD is given one run of the order and its workgroups go through it side by side: they share operands in its L2.
struct TileTurns {
    int at, end, step;
    SSD_DEV void init(int total, int block, int blocks)
    {
        const int x = block % 8, q = total / 8, r = total % 8;
        const int lo = x * q + (x < r ? x : r);
        end = lo + q + (x < r ? 1 : 0);
        step = (blocks - x + 7) / 8;
        at = lo + block / 8;
    }
};

// The order of tiles: through `group` tiles of n before the next m.
SSD_DEV void tile_of(int t, int tm, int tn, int group, int &m, int &n)
{
    const int per = group * tm, gi = t / per, first = gi * group;
    const int width = tn - first < group ? tn - first : group;
    const int rem = t - gi * per;
    n = first + rem % width;
    m = rem / width;
}

// acc[mi][nj][e]: m = 32 mi + 8 (e / 4) + 4 (lane / 32) + e % 4, n = 32 nj + lane % 32 of the wave's part of the tile.
template <typename T, int BM, int BN, int WM, int WN, bool A_KROWS, bool B_KROWS>
struct TileStream {
    static constexpr int kThreads = WM * WN * 64;
    static constexpr int MF = BM / WM / 32, NF = BN / WN / 32;
    static constexpr int kBuffer = (BM + BN) * kStageBytes;
    static constexpr int kLds = kStages * kBuffer;
    typedef TileOperand<T, BM, A_KROWS, kThreads> OpA;
    typedef TileOperand<T, BN, B_KROWS, kThreads> OpB;
    static constexpr int kBK = OpA::kBK;
    static constexpr int kLoads = OpA::kPer + OpB::kPer;                 // a stage's, per lane

    // unit(i, TileUnit &): the i-th unit;  set(OpA &, OpB &, unit, slot): its operands, and what its epilogue wants in LDS (one
    // of kSlots places; loaded with load_to_lds, it has landed, in all waves, when the epilogue runs: it is older than the
    // unit's first stage);  use(acc, unit, em, en, slot): its epilogue.
    // An epilogue does better without global loads of its own: their wait would be one for every load in flight.
    static constexpr int kSlots = kStages + 1;   // as many units may be on their way, of a stage each
    template <typename Unit, typename Set, typename Use>
    static SSD_DEV void run(int total, int block, int blocks, const char *smem, Unit unit, Set set, Use use)
    {
        TileTurns turn;
        turn.init(total, block, blocks);
        if (turn.at >= turn.end) return;
        const int wave = uniform(threadIdx.x / 64);
        const int em = (wave / WN) * (BM / WM), en = (wave % WN) * (BN / WN);

        // ---- what is loaded: runs ahead
        OpA a;
        OpB b;
        TileTurns ahead = turn;
        int left = 0;                            // values of k of the unit being loaded
        int slot_put = 0, slot_get = 0;
        const unsigned first = (unsigned)uniform((int)(lds_address(smem) + threadIdx.x / 64 * 1024u));
        unsigned put = first;                    // where the wave's pieces of the next stage go
        const auto next_put = [&]() {
            a.base += a.step;
            b.base += b.step;
            left -= kBK;
            put = put == first + (kStages - 1) * kBuffer ? first : put + kBuffer;
        };
        // any stage: the last of a unit, the first of the next, or none
        const auto load = [&]() {
            while (left <= 0 && ahead.at < ahead.end) {
                TileUnit u;
                unit(ahead.at, u);
                ahead.at += ahead.step;
                left = u.k;
                if (left > 0) {
                    set(a, b, u, slot_put);
                    slot_put = slot_put == kSlots - 1 ? 0 : slot_put + 1;
                }
            }
            a.load(put, left);
            b.load(put + BM * kStageBytes, left);
            next_put();
        };
        const auto load_whole = [&](int i) {     // piece i of a whole stage of the same unit
            if (i < OpA::kPer) a.load_whole(put, i);
            else b.load_whole(put + BM * kStageBytes, i - OpA::kPer);
        };

        f32x16 acc[MF][NF];
        // float32: a long chain of additions rounds as often as it has links, so stages are summed up apart
        constexpr bool kTwice = sizeof(T) == 4;
        f32x16 all[kTwice ? MF : 1][kTwice ? NF : 1];
        u32x4 a0[MF], b0[NF], a1[MF], b1[NF];
        constexpr int kMma = MF * NF, kReads = MF + NF;
        constexpr int kReadsEach = (kReads + kMma / 2 - 1) / (kMma / 2), kLoadsEach = (kLoads + (kMma + 1) / 2 - 1) / ((kMma + 1) / 2);

        for (int i = 0; i < kStages; ++i) load();
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"((kStages - 1) * kLoads) : "memory");
#pragma unroll
        for (int mi = 0; mi < MF; ++mi) a0[mi] = OpA::fragment(smem, em + mi * 32, 0);
#pragma unroll
        for (int nj = 0; nj < NF; ++nj) b0[nj] = OpB::fragment(smem + BM * kStageBytes, en + nj * 32, 0);

        unsigned get = 0;
        for (; turn.at < turn.end; turn.at += turn.step) {
            TileUnit u;
            unit(turn.at, u);
#pragma unroll
            for (int mi = 0; mi < MF; ++mi)
#pragma unroll
                for (int nj = 0; nj < NF; ++nj) {
                    acc[mi][nj] = f32x16{};
                    if constexpr (kTwice) all[mi][nj] = f32x16{};
                }
            for (int k = u.k; k > 0; k -= kBK) {
                const char *ta = smem + get, *tb = smem + BM * kStageBytes + get;
                get = get == (kStages - 1) * kBuffer ? 0 : get + kBuffer;
                // reads between the first half of the matrix instructions (they are waited for behind the last), loads between
                // the others
#pragma unroll
                for (int i = 0; i < kMma; ++i) {
                    TileNum<T>::mma(acc[i / NF][i % NF], a0[i / NF], b0[i % NF]);
#pragma unroll
                    for (int r = i * kReadsEach; r < (i + 1) * kReadsEach && r < kReads; ++r) {
                        if (r < NF) b1[r] = OpB::fragment(tb, en + r * 32, 1);
                        else a1[r - NF] = OpA::fragment(ta, em + (r - NF) * 32, 1);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(2 * kLoads) : "memory");
                ta = smem + get;
                tb = smem + BM * kStageBytes + get;
                const bool plain = left >= kBK;
                if (!plain) load();
#pragma unroll
                for (int i = 0; i < kMma; ++i) {
                    TileNum<T>::mma(acc[i / NF][i % NF], a1[i / NF], b1[i % NF]);
#pragma unroll
                    for (int r = i * kReadsEach; r < (i + 1) * kReadsEach && r < kReads; ++r) {
                        if (r < NF) b0[r] = OpB::fragment(tb, en + r * 32, 0);
                        else a0[r - NF] = OpA::fragment(ta, em + (r - NF) * 32, 0);
                    }
                    if (i >= kMma / 2 && plain)
#pragma unroll
                        for (int l = (i - kMma / 2) * kLoadsEach; l < (i - kMma / 2 + 1) * kLoadsEach && l < kLoads; ++l)
                            load_whole(l);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (plain) next_put();
                if constexpr (kTwice)
#pragma unroll
                    for (int mi = 0; mi < MF; ++mi)
#pragma unroll
                        for (int nj = 0; nj < NF; ++nj) {
                            all[mi][nj] += acc[mi][nj];
                            acc[mi][nj] = f32x16{};
                        }
            }
            if constexpr (kTwice) use(all, u, em, en, slot_get);
            else use(acc, u, em, en, slot_get);
            if (u.k > 0) slot_get = slot_get == kSlots - 1 ? 0 : slot_get + 1;
        }
        // LDS may be another workgroup's once this one has ended: no load may be on its way to it
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
};
