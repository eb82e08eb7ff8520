// Cross entropy of a linear head over many classes, with its gradients; of the logits and of d no more than about 2 GiB each is
// stored at a time.
//
//   z = s H W^T (rows x classes), l = label, eps = label smoothing, V = classes
//   nll = log sum_v exp z_v - z_l,   loss = (1 - eps) nll + eps (log sum_v exp z_v - mean_v z_v)
//   d_nv = g_n s (p_nv - eps / V - (1 - eps) [v = l]),   dH = d W,   dW = d^T H
//
// Rows without a class (label < 0) leave the batch first: the counted rows are copied together, so a padded batch costs
// what its counted rows cost and nothing of a padded row (a NaN, say) reaches a sum over rows.  Then
//   1  logits, a tile of classes x rows per workgroup; of each tile only (max, sum of exp) per row leave the chip
//   2  per row: log-sum-exp, loss, and what the gradient needs (four floats a row)
//   3  per piece of the classes (a d of 2 GiB: all of them, as a rule), and per chunk of the rows where 256 classes of all are more:
//      the logits again, turned into d in the epilogue and written in the operands' type; dH += d W_piece, dW_piece = d^T H.
// Recomputing the logits is 2 of the gradient's 8 rows * classes * dim operations.  The last piece need not be: while step 1
// runs, what d can be made of waits for a pass that turns it into d.  float32: the products, in d's own place.  bfloat16: the
// exponentials in 16 bits, relative to their tile's maximum, there too (float16's 11 bits round them finer than d's 8).
// float16, whose d has 11 bits too and would be rounded twice: the products, in a place of their own.
// Few logits are written as products, too, and a row of them goes through statistics and d in one launch.
//
// The label's own class stays out of the sum of exponentials: with S = sum over the others of exp(z_v - M), a sure row's
// nll is log1p(S exp(M - z_l)) and p_l - 1 is expm1(-nll), both without the cancellation that 1 - p_l has.
// Exponentials are taken to base 2: exp(z_v - M) = 2^(a L - m) with a the product as summed, L = s log2(e) and m the row's
// largest a L rounded once; m itself is what the rows' kernel adds back, so its rounding cancels.
// Sums over k stay in float32 accumulators; over tiles and rows of partial results they are added in a fixed order, in
// float64 for the exponentials.  d is rounded to the operands' type, which is what the matrix instructions read: once, but for
// bfloat16's kept exponentials, whose first rounding to 11 bits is an eighth of the second one to 8.
#include <math.h>

#include <type_traits>

#include "ssdbox_tile.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;
constexpr int kRowThreads = 256;
constexpr long long kMostLd = 1 << 21;        // from one row of an operand to the next: a tile's rows in 32 bits of bytes
constexpr long long kMostRows = (1 << 24) - 1;  // of workgroups of 256: a launch takes fewer than 2^32 threads
constexpr int kRowsEach = 4;          // rows a workgroup places and copies
constexpr int kCountRows = 1024;      // rows a workgroup counts, where there are many
constexpr int kShiftFrom = 10, kMostShift = 10;   // of a row of float16's d, beyond the scale that all have (see row_finish)
constexpr int kCountFrom = 4096;      // rows from which counting has a launch of its own: below, reading all labels before
                                      // a workgroup's rows again costs less than the launch

struct HeadScale {                    // what the gradient's rows are multiplied by before d, and the results after
    float down, up;
};

struct alignas(16) HeadRow {          // a counted row: p_v = 2^(a L - m) * c / Z with c = g_n s folded in
    float m, pz, label, smooth;       // pz = c / Z, label = c (p_l - (1 - eps) - eps / V), smooth = c eps / V
};

// ------------------------------------------------------------------------------ rows
struct PrepArgs {
    const void *labels;
    int label_bytes, rows;
    long long classes;
    const float *grad_loss;
    float logit_scale, smoothing;
    int scaled;                       // 16-bit gradients: bring the largest c (1 - eps) to just under 2^15
    const void *hidden;
    long long ld;
    int dim, pitch;
    int *block_count;                 // counted rows and largest |grad_loss| of every kCountRows rows, or NULL
    float *block_max;
    int *place_count;                 // the number of counted rows; behind it, of more than one chunk, each chunk's
    int chunks, chunk_rows;
    int *row, *label;                 // per counted row: the row it was, its class
    HeadScale *scale;
    float *loss;
    void *out, *grad_hidden;
    bool stay;                        // every row keeps its place, and is copied whatever its label
    int prep_blocks;                  // workgroups of rows; the launch's others lay out the weight
    const void *weight;
    long long weight_ld;
    void *weight_out;
};

SSD_DEV long long label_at(const void *p, int bytes, int n)
{
    return bytes == 8 ? ((const long long *)p)[n] : (long long)((const int *)p)[n];
}

SSD_DEV bool counted_at(const PrepArgs &p, int n)
{
    const long long lab = label_at(p.labels, p.label_bytes, n);
    return lab >= 0 && lab < p.classes;
}

// Sum and maximum over the workgroup's waves, in all lanes.
template <int WAVES>
SSD_DEV int block_total(int x, int *lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) x += lds[w];
    return x;
}
template <int WAVES>
SSD_DEV float block_max(float x, float *lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) x = fmaxf(x, lds[w]);
    return x;
}

// What d is scaled by: called by the whole workgroup.
template <int WAVES>
SSD_DEV HeadScale scale_of(const PrepArgs &p, float *lds)
{
    HeadScale s = {1.0f, 1.0f};
    if (!p.scaled) return s;
    float g = 0.0f;
    if (!p.grad_loss) {
        g = 1.0f / (float)p.rows;
    } else {
        if (p.block_count) {
            for (int i = threadIdx.x; i < (p.rows + kCountRows - 1) / kCountRows; i += WAVES * 64) g = fmaxf(g, p.block_max[i]);
        } else {
            for (int n = threadIdx.x; n < p.rows; n += WAVES * 64)
                if (counted_at(p, n)) g = fmaxf(g, fabsf(p.grad_loss[n]));
        }
        g = block_max<WAVES>(g, lds);
    }
    // Of float16 this uses the range; and an unsure row's d at its label, -c (1 - eps - p), which weighs most in the
    // gradients, is a value that both types have, just under a power of two, where their rounding is finest.
    const float c = g * p.logit_scale * (1.0f - fminf(p.smoothing, 0.5f));
    if (c > 1e-30f && c < 1e30f) {
        s.down = 32768.0f * (1.0f - 1.0f / 128.0f) / c;
        s.up = 1.0f / s.down;
    }
    return s;
}

// Labels of kCountRows rows a workgroup; latency (5 us at 8192 rows).
__global__ __launch_bounds__(kRowThreads) void head_count_kernel(const PrepArgs p)
{
    __shared__ int s_count[4];
    __shared__ float s_max[4];
    int c = 0;
    float g = 0.0f;
    const int end = min(p.rows, ((int)blockIdx.x + 1) * kCountRows);
    for (int n = blockIdx.x * kCountRows + threadIdx.x; n < end; n += kRowThreads)
        if (counted_at(p, n)) {
            ++c;
            if (p.grad_loss) g = fmaxf(g, fabsf(p.grad_loss[n]));
        }
    c = block_total<kRowThreads / 64>(c, s_count);
    g = block_max<kRowThreads / 64>(g, s_max);
    if (threadIdx.x == 0) {
        p.block_count[blockIdx.x] = c;
        p.block_max[blockIdx.x] = g;
    }
}

// Rows of a weight whose rows do not start at 16-byte boundaries, laid out so that they do: 16 bytes a lane, which the
// loads take from any value's boundary.
template <typename T>
SSD_DEV void pitch_weight(const T *weight, long long ld, long long classes, int dim, int pitch, T *out, int block, int blocks)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
    const int pieces = pitch / kVec;
    const long long all = classes * pieces, step = (long long)blocks * kRowThreads;
    for (long long i = (long long)block * kRowThreads + threadIdx.x; i < all; i += step) {
        const long long v = i / pieces;
        const int d = (int)(i - v * pieces) * kVec;
        const T *from = weight + v * ld + d;
        u32x4 x;
        if (d + kVec <= dim) {
            const Raw r = *(const Raw *)from;
            x = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
        } else {
            union { T v[kVec]; u32x4 w; } y;
#pragma unroll
            for (int j = 0; j < kVec; ++j) y.v[j] = d + j < dim ? from[j] : (T)0.0f;
            x = y.w;
        }
        *(u32x4 *)(out + v * pitch + d) = x;
    }
}

// Each workgroup takes kRowsEach rows: counts the rows before them (the order of the counted rows is that of the batch, so that
// sums over rows are the same every time), copies the counted ones to their places, with zeros behind their last value, and
// settles the others.  A copy, bound by HBM (8192 x 2048 bfloat16: 67 MB in 15.6 us) or, short, by its own labels' latency (5 us).
template <typename T>
__global__ __launch_bounds__(kRowThreads) void head_prep_kernel(const PrepArgs p)
{
    __shared__ int s_count[4];
    __shared__ float s_max[4];
    __shared__ int s_place[kRowsEach];
    if ((int)blockIdx.x >= p.prep_blocks) {
        pitch_weight<T>((const T *)p.weight, p.weight_ld, p.classes, p.dim, p.pitch, (T *)p.weight_out,
                        blockIdx.x - p.prep_blocks, gridDim.x - p.prep_blocks);
        return;
    }
    const int t = threadIdx.x, first = blockIdx.x * kRowsEach;
    if (p.stay) {
        if (t < kRowsEach) s_place[t] = first + t;
    } else {
        const int blocks = p.block_count ? first / kCountRows : 0;
        int before = 0;
        for (int i = t; i < blocks; i += kRowThreads) before += p.block_count[i];
        for (int n = blocks * kCountRows + t; n < first; n += kRowThreads) before += counted_at(p, n) ? 1 : 0;
        before = block_total<kRowThreads / 64>(before, s_count);
        if (t < 64) {
            const int n = first + t;
            const bool mine = t < kRowsEach && n < p.rows;
            const long long lab = mine ? label_at(p.labels, p.label_bytes, n) : -1;
            const bool counted = lab >= 0 && lab < p.classes;
            const unsigned long long bal = __ballot(counted);
            const int at = before + __popcll(bal & ((1ull << t) - 1ull));
            if (counted) {
                p.row[at] = n;
                p.label[at] = (int)lab;
            } else if (mine) {
                p.loss[n] = lab < 0 ? 0.0f : u2f(0x7FC00000u);
            }
            if (t < kRowsEach) s_place[t] = counted ? at : -1;
            if (t == 0 && first + kRowsEach >= p.rows) {
                const int all = before + __popcll(bal);
                *p.place_count = all;
                if (p.chunks > 1)
                    for (int i = 0; i < p.chunks; ++i) p.place_count[1 + i] = min(max(all - i * p.chunk_rows, 0), p.chunk_rows);
            }
        }
    }
    __syncthreads();
    const T *hidden = (const T *)p.hidden;
    constexpr int kVec = 16 / (int)sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
    for (int i = t >> 6; i < kRowsEach && first + i < p.rows; i += kRowThreads / 64) {
        const long long n = first + i, at = s_place[i];
        const int lane = t & 63;
        if (at >= 0) {
            const T *from = hidden + n * p.ld;
            T *o = (T *)p.out + at * p.pitch;
            for (int d = lane * kVec; d < p.pitch; d += 64 * kVec) {
                if (d + kVec <= p.dim) {
                    const Raw r = *(const Raw *)(from + d);
                    *(u32x4 *)(o + d) = u32x4{r.w[0], r.w[1], r.w[2], r.w[3]};
                } else {
#pragma unroll
                    for (int j = 0; j < kVec; ++j) o[d + j] = d + j < p.dim ? from[d + j] : (T)0.0f;
                }
            }
        } else if (p.grad_hidden) {
            T *o = (T *)p.grad_hidden + n * p.dim;
            for (int d = lane; d < p.dim; d += 64) o[d] = (T)0.0f;
        }
    }
    if (p.stay || blockIdx.x != 0) return;
    const HeadScale s = scale_of<kRowThreads / 64>(p, s_max);
    if (t == 0) *p.scale = s;
}

// --------------------------------------------------------------------------- products
struct LogitArgs {
    const void *weight, *rows;        // classes x dim from the piece's first class on; counted rows x dim
    long long ldw, ldh;
    int dim, classes, tiles;          // classes and tiles of classes in this piece
    int first;                        // the piece's first class
    float l2;                         // logit_scale * log2(e)
    const int *count, *label;
    float2 *stat;                     // [row][slots]: (max, sum of exponentials) of one wave's part of a tile
    float *sum_z;                     // [row][slots], or NULL without smoothing
    long long slots;
    float *z_label;                   // [row]: the label's product, before the scale
    const HeadRow *row;
    void *delta;                      // [row][ld_delta]: d, or from class kept_from on what is kept
    long long ld_delta;
    int kept_from;
};

// What a tile of logits leaves: statistics, d, or statistics and what d can be made of later.
enum { kStat = 0, kDelta = 1, kStatKeep = 2 };

// That is for bfloat16 exponentials times 2^15 as float16, otherwise the products as float32; for float32 and bfloat16 it lies
// where d will.
template <typename T>
using Kept = typename std::conditional<__is_same(T, bf16_t), f16_t, float>::type;

// Sixteen neighbouring values of one row of the result, half of them in the lane 32 further: lo at m + 4 h .. + 3 and hi
// at m + 8 + 4 h .. + 3 (h = lane / 32).  16-bit types trade halves, so that each lane stores 16 bytes (from any value's
// boundary: rows of an odd length start there).  Called by both lanes alike; left: values there are from m on.
template <typename T>
SSD_DEV void store_pair(T *row, int m, const float (&lo)[4], const float (&hi)[4], int left, bool in)
{
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
    const int h = (int)(threadIdx.x >> 5 & 1);
    if (left >= 16) {
        Raw a, b;
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a.w[i] = f2u(lo[i]);
                b.w[i] = f2u(hi[i]);
            }
            if (!in) return;
            *(Raw *)(row + m + 4 * h) = a;
            *(Raw *)(row + m + 8 + 4 * h) = b;
        } else {
            union { T v[8]; unsigned w[4]; } x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x.v[i] = (T)lo[i];
                x.v[4 + i] = (T)hi[i];
            }
            const auto p = __builtin_amdgcn_permlane32_swap(x.w[0], x.w[2], false, false);
            const auto q = __builtin_amdgcn_permlane32_swap(x.w[1], x.w[3], false, false);
            a.w[0] = p[0];
            a.w[1] = q[0];
            a.w[2] = p[1];
            a.w[3] = q[1];
            if (in) *(Raw *)(row + m + 8 * h) = a;
        }
        return;
    }
    if (!in) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (4 * h + i < left) row[m + 4 * h + i] = (T)lo[i];
        if (8 + 4 * h + i < left) row[m + 8 + 4 * h + i] = (T)hi[i];
    }
}

// The logits by tiles: matrix instructions, and behind each tile its exponentials (one v_exp_f32 a logit, which the
// stream's loads for the next tile run under).  Long dim: bound by the matrix instructions at the clock that the power limit leaves
// (3891 x 32000 x 4096 bfloat16, value: 907 us, 1.12 PFLOP/s of 1.36 that the library's product alone reaches, matrix cores busy 74 %
// of the time; 7782 x 131072 x 2048 with the exponentials stored: 4.06 ms, 1.03, 62 %); short dim: by the epilogue (1694 x 104936 x
// 16: 102 us, 1.7e12 exponentials a second).
template <typename T, int BM, int BN, int WM, int WN, int BLOCKS, int WHAT>
__global__ __launch_bounds__(WM * WN * 64, BLOCKS * WM * WN / 4) void head_logit_kernel(const LogitArgs p)
{
    typedef TileStream<T, BM, BN, WM, WN, false, false> S;
    // what the epilogue wants of its rows: labels (a wave's load of 1024 bytes, of which BN / 256 are wanted), and for d HeadRow
    constexpr int kSlot = 1024 + (WHAT == kDelta ? BN * 16 : 0);
    __shared__ __align__(1024) char smem[S::kLds + S::kSlots * kSlot];
    const int count = uniform(*p.count);
    const int tn = (count + BN - 1) / BN;
    const auto unit = [&](int i, TileUnit &u) {
        int m, n;
        tile_of(i, p.tiles, tn, 8, m, n);
        u = TileUnit{m * BM, n * BN, 0, p.dim, 0};
    };
    const auto set = [&](typename S::OpA &a, typename S::OpB &b, const TileUnit &u, int slot) {
        a.init(p.weight, p.ldw, u.m0, p.classes - u.m0, 0);
        b.init(p.rows, p.ldh, u.n0, count - u.n0, 0);
        const int wave = uniform(threadIdx.x / 64), lane = threadIdx.x & 63, last = (count - 1 - u.n0);
        const unsigned to = lds_address(smem) + S::kLds + slot * kSlot;
        if (wave == 0) load_to_lds_at(to, (const char *)(p.label + u.n0) + (lane * 4 <= last ? lane : last / 4) * 16);
        if constexpr (WHAT == kDelta)
            for (int i = wave; i < BN / 64; i += WM * WN) {
                const int n = i * 64 + lane;
                load_to_lds_at(to + 1024 + i * 1024, (const char *)(p.row + u.n0 + (n <= last ? n : last)));
            }
    };
    const auto use = [&](f32x16 (&acc)[S::MF][S::NF], const TileUnit &u, int em, int en, int slot) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
        const char *kept = smem + S::kLds + slot * kSlot;
        const int v0 = u.m0 + em + 4 * h;                        // within the piece
        const bool edge = u.m0 + em + 32 * S::MF > p.classes;    // the wave's part has classes that do not exist
#pragma unroll
        for (int nj = 0; nj < S::NF; ++nj) {
            const int at = en + nj * 32 + (lane & 31), n = u.n0 + at;
            const bool in = n < count;
            const int lab = in ? ((const int *)kept)[at] - p.first : -1;
            const int rel = lab - (u.m0 + em);
            // the tests of single values only where one of the wave's labels lies here, or the last class
            const bool plain = !edge && !__any(rel >= 0 && rel < 32 * S::MF);
            if constexpr (WHAT != kDelta) {
                float mx = -INFINITY, sz = 0.0f, s = 0.0f;
                if (plain) {
#pragma unroll
                    for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                        for (int e = 0; e < 16; ++e) mx = fmaxf(mx, acc[mi][nj][e]);
                    if (p.sum_z)
#pragma unroll
                        for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                            for (int e = 0; e < 16; ++e) sz += acc[mi][nj][e];
                } else {
#pragma unroll
                    for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int v = v0 + mi * 32 + (e >> 2) * 8 + (e & 3);
                            const float z = acc[mi][nj][e];
                            if (v < p.classes) {
                                sz += z;
                                if (v != lab) mx = fmaxf(mx, z);
                                else p.z_label[n] = z;
                            }
                        }
                }
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float m = mx * p.l2;
                // times 2^15, for what is kept in float16; the loss is to the bit the same whether something is kept or not
                const float ref = (mx == -INFINITY ? 0.0f : m) - 15.0f;
                const bool keep = WHAT == kStatKeep && u.m0 >= p.kept_from;
                Kept<T> *kept_row = (Kept<T> *)p.delta + (long long)n * p.ld_delta - p.kept_from;
#pragma unroll
                for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        float x[2][4];
                        const int at8 = u.m0 + em + mi * 32 + e * 2;
                        if constexpr (WHAT == kStatKeep && __is_same(Kept<T>, float)) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) x[i >> 2][i & 3] = acc[mi][nj][e + i];
                            if (keep) store_pair<float>(kept_row, at8, x[0], x[1], 16, in);
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            x[i >> 2][i & 3] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mi][nj][e + i], p.l2, -ref));
                        if (plain) {
#pragma unroll
                            for (int i = 0; i < 8; ++i) s += x[i >> 2][i & 3];
                        } else {
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int v = at8 + 4 * h + (i >> 2) * 8 + (i & 3);
                                if (v >= p.classes) x[i >> 2][i & 3] = 0.0f;
                                if (v != lab) s += x[i >> 2][i & 3];
                            }
                        }
                        if constexpr (WHAT == kStatKeep && !__is_same(Kept<T>, float))
                            if (keep) store_pair<f16_t>(kept_row, at8, x[0], x[1], 16, in);
                    }
                s *= 0x1p-15f;
                s += __shfl_xor(s, 32);
                const long long slot = (long long)n * p.slots + (u.m0 + em) / (32 * S::MF);
                if (in && h == 0) p.stat[slot] = make_float2(m, s);
                if (p.sum_z) {
                    sz += __shfl_xor(sz, 32);
                    if (in && h == 0) p.sum_z[slot] = sz;
                }
            } else {
                const HeadRow r = ((const HeadRow *)(kept + 1024))[at];
                T *out = (T *)p.delta + (long long)n * p.ld_delta;
#pragma unroll
                for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        float d[2][4];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            d[i >> 2][i & 3] = __builtin_fmaf(
                                __builtin_amdgcn_exp2f(__builtin_fmaf(acc[mi][nj][e + i], p.l2, -r.m)), r.pz, -r.smooth);
                        const int m = u.m0 + em + mi * 32 + e * 2;
                        if (!plain)
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const int v = m + 4 * h + (i >> 2) * 8 + (i & 3);
                                if (v == lab) d[i >> 2][i & 3] = r.label;
                                if (v >= p.classes) d[i >> 2][i & 3] = 0.0f;
                            }
                        store_pair<T>(out, m, d[0], d[1], 16, in);
                    }
            }
        }
    };
    S::run(p.tiles * tn, blockIdx.x, gridDim.x, smem, unit, set, use);
}

// ------------------------------------------------------------------------ row statistics
struct RowArgs {
    const int *count, *row, *label;
    const float2 *stat;
    const float *sum_z;
    long long slots;
    const float *z_label;
    float l2, logit_scale, smoothing;
    long long classes;
    int rows;
    const float *grad_loss;
    const HeadScale *scale;
    float *loss;
    HeadRow *out;
    float *row_up;                    // float16 with rows' weights: 2^-shift of each counted row, and its values times that for
    const void *values;               // dW (in their place, or not)
    void *scaled;
    int pitch;
};

// A counted row's values times 2^-shift, by a workgroup.
template <typename T, int THREADS>
SSD_DEV void scale_row(const T *from, T *to, int pitch, int shift)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    if (from == to && shift == 0) return;
    const float f = u2f((uint32_t)(127 - shift) << 23);
    for (int d = threadIdx.x * kVec; d < pitch; d += THREADS * kVec) {
        union { u32x4 w; T v[kVec]; } x;
        x.w = *(const u32x4 *)(from + d);
#pragma unroll
        for (int i = 0; i < kVec; ++i) x.v[i] = (T)((float)x.v[i] * f);
        *(u32x4 *)(to + d) = x.w;
    }
}

// A row's loss and its gradient's terms: the others' exponentials sum to s * 2^m, the label's is 2^(z l2) with its product z.
// Float16 has few exponents: with one scale for all, p of a row whose weight is 10^6 times smaller than the largest would lie among
// the subnormals.  The d of rows below 2^-10 of the largest is raised by 2^shift, so that it keeps 2^-28 of the row's weight, which
// its dH gives back, and its values in dW's product.  Those lose what falls below 2^-24 there, in terms 2^-10 to 2^-20 of others':
// rows of larger weights stay as they are, since their d needs nothing and hidden values may be small.
SSD_DEV HeadRow row_finish(const RowArgs &p, int n_in, float down, float m, double s, double sz, float z, int &shift)
{
    shift = 0;
    const double zl = (double)z * (double)p.l2;
    double nll = 0.0;
    if (s != 0.0) {
        const double d = (double)m - zl;
        nll = d > 500.0 ? d * kLn2 + log(s) : log1p(s * exp2(d));
    }
    double loss = nll;
    if (p.smoothing != 0.0f) {
        const double mean = sz * (double)p.logit_scale / (double)p.classes;
        loss = (1.0 - (double)p.smoothing) * nll + (double)p.smoothing * (nll + (double)z * (double)p.logit_scale - mean);
    }
    p.loss[n_in] = (float)loss;
    HeadRow r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (!p.out) return r;
    const double g = p.grad_loss ? (double)p.grad_loss[n_in] : 1.0 / (double)p.rows;
    double c = g * (double)p.logit_scale * (double)down;
    if (p.row_up) {
        const double v = fabs(c) * (1.0 - fmin((double)p.smoothing, 0.5));     // at most 32768 (1 - 1 / 128)
        while (shift < kMostShift && v * (double)(2 << (kShiftFrom + shift)) <= 32512.0) ++shift;
        c *= (double)(1 << shift);
    }
    const float top = fmaxf(m, (float)zl);
    const double whole = (s != 0.0 ? s * exp2((double)m - (double)top) : 0.0) + exp2(zl - (double)top);
    const double share = (double)p.smoothing / (double)p.classes;
    r.m = top;
    r.pz = (float)(c / whole);
    r.label = (float)(c * (expm1(-nll) + (double)p.smoothing - share));
    r.smooth = (float)(c * share);
    return r;
}

// A row a workgroup: its tiles' statistics together, then its loss.  Latency: two dependent loads and float64 logarithms (9 us
// for 1529 rows of 784 slots, 30 for 7782 of 1024).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void head_row_kernel(const RowArgs p)
{
    __shared__ float s_m[THREADS / 64];
    __shared__ double s_s[THREADS / 64], s_z[THREADS / 64];
    __shared__ int s_shift;
    const int n = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    if (n >= *p.count) return;
    const float2 *st = p.stat + (long long)n * p.slots;
    float m = -INFINITY;
    double s = 0.0, sz = 0.0;
    for (long long i = t; i < p.slots; i += THREADS) {
        const float2 x = st[i];
        const float nm = fmaxf(m, x.x);
        if (nm != -INFINITY) {
            s = s * (double)__builtin_amdgcn_exp2f(m - nm) + (double)x.y * (double)__builtin_amdgcn_exp2f(x.x - nm);
        } else {
            s += (double)x.y;                   // nothing finite so far: zero, or a NaN
        }
        m = nm;
        if (p.sum_z) sz += (double)p.sum_z[(long long)n * p.slots + i];
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float om = __shfl_xor(m, o);
        const double os = __shfl_xor(s, o);
        const float nm = fmaxf(m, om);
        if (nm != -INFINITY)
            s = s * (double)__builtin_amdgcn_exp2f(m - nm) + os * (double)__builtin_amdgcn_exp2f(om - nm);
        else
            s += os;
        m = nm;
        sz += __shfl_xor(sz, o);
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_s[wave] = s;
        s_z[wave] = sz;
    }
    __syncthreads();
    if (t == 0) {
        m = -INFINITY;
        for (int w = 0; w < THREADS / 64; ++w) m = fmaxf(m, s_m[w]);
        s = 0.0;
        sz = 0.0;
        for (int w = 0; w < THREADS / 64; ++w) {
            s += m != -INFINITY ? s_s[w] * (double)__builtin_amdgcn_exp2f(s_m[w] - m) : s_s[w];
            sz += s_z[w];
        }
        const HeadRow r = row_finish(p, p.row[n], p.out ? p.scale->down : 1.0f, m, s, sz, p.z_label[n], s_shift);
        if (p.out) p.out[n] = r;
        if (p.row_up) p.row_up[n] = u2f((uint32_t)(127 - s_shift) << 23);
    }
    if (!p.scaled) return;
    __syncthreads();
    scale_row<f16_t, THREADS>((const f16_t *)p.values + (long long)n * p.pitch, (f16_t *)p.scaled + (long long)n * p.pitch,
                              p.pitch, s_shift);
}

// Few logits: their products (in parts, where k was cut) are joined in the parts' order a row at a time, with the row's
// statistics and its d.  DIRECT: of the batch's own rows, which nothing has placed before; what prep does then happens here,
// but that the rows without a class stay where they are, with d and values of zero (row_of -1: their gradient is written here).
// Three passes over a row that stays in the caches; latency (4 us for 1000 classes, 11 for 10007).
template <typename T, int THREADS, bool DIRECT>
__global__ __launch_bounds__(THREADS) void head_few_kernel(const RowArgs p, const PrepArgs b, float *part, long long ld_part,
                                                           long long part_stride, int parts, T *delta, long long ld_delta)
{
    __shared__ float s_m[THREADS / 64], s_g[THREADS / 64], s_label;
    __shared__ double s_s[THREADS / 64], s_z[THREADS / 64];
    __shared__ HeadRow s_row;
    __shared__ int s_shift;
    const int n = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6, classes = (int)p.classes;
    int lab, n_in;
    float down = 1.0f;
    if constexpr (DIRECT) {
        if (p.out) {
            const HeadScale s = scale_of<THREADS / 64>(b, s_g);
            down = s.down;
            if (n == 0 && t == 0) *b.scale = s;
        }
        const long long given = label_at(b.labels, b.label_bytes, n);
        const bool counted = given >= 0 && given < p.classes;
        lab = (int)given;
        n_in = n;
        if (p.out) {
            if (t == 0) b.row[n] = counted ? n : -1;
            constexpr int kVec = 16 / (int)sizeof(T);
            for (int d = t * kVec; d < b.pitch; d += THREADS * kVec)
                *(u32x4 *)((T *)b.out + (long long)n * b.pitch + d) =
                    counted ? *(const u32x4 *)((const T *)b.hidden + n * b.ld + d) : u32x4{0u, 0u, 0u, 0u};
        }
        if (!counted) {
            if (t == 0) p.loss[n] = given < 0 ? 0.0f : u2f(0x7FC00000u);
            if (!p.out) return;
            for (int v = t; v < (classes + 63) / 64 * 64; v += THREADS) delta[n * ld_delta + v] = (T)0.0f;
            if (b.grad_hidden)
                for (int d = t; d < b.dim; d += THREADS) ((T *)b.grad_hidden)[(long long)n * b.dim + d] = (T)0.0f;
            return;
        }
    } else {
        if (n >= *p.count) return;
        lab = p.label[n];
        n_in = p.row[n];
        if (p.out) down = p.scale->down;
    }
    float *z = part + (long long)n * ld_part;
    float mx = -INFINITY;
    double sz = 0.0;
    for (int v = t * 4; v < classes; v += THREADS * 4) {     // rows are padded to whole fours
        f32x4 x = *(const f32x4 *)(z + v);
        for (int i = 1; i < parts; ++i) x += *(const f32x4 *)(z + v + i * part_stride);
        if (parts > 1) *(f32x4 *)(z + v) = x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (v + j >= classes) continue;
            sz += (double)x[j];
            if (v + j == lab) s_label = x[j];
            else mx = fmaxf(mx, x[j]);
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        mx = fmaxf(mx, __shfl_xor(mx, o));
        sz += __shfl_xor(sz, o);
    }
    if (lane == 0) {
        s_m[wave] = mx;
        s_z[wave] = sz;
    }
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) mx = fmaxf(mx, s_m[w]);
    const float m = mx * p.l2, ref = mx == -INFINITY ? 0.0f : m;
    double s = 0.0;
    for (int v = t * 4; v < classes; v += THREADS * 4) {
        const f32x4 x = *(const f32x4 *)(z + v);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (v + j < classes && v + j != lab) s += (double)__builtin_amdgcn_exp2f(__builtin_fmaf(x[j], p.l2, -ref));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) s_s[wave] = s;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < THREADS / 64; ++w) {
            s_s[0] += s_s[w];
            s_z[0] += s_z[w];
        }
        s_row = row_finish(p, n_in, down, m, s_s[0], s_z[0], s_label, s_shift);
        if (p.row_up) p.row_up[n] = u2f((uint32_t)(127 - s_shift) << 23);
    }
    if (!p.out) return;
    __syncthreads();
    const HeadRow r = s_row;
    if constexpr (__is_same(T, f16_t))
        if (p.scaled)                 // (each lane what it has copied, if it has)
            scale_row<T, THREADS>((const T *)p.values + (long long)n * p.pitch, (T *)p.scaled + (long long)n * p.pitch,
                                  p.pitch, s_shift);
    T *d = delta + (long long)n * ld_delta;
    for (int v = t * 4; v < (classes + 63) / 64 * 64; v += THREADS * 4) {    // d has zeros behind the last class
        struct __align__(4 * sizeof(T)) { T v[4]; } o;
        const f32x4 x = v < classes ? *(const f32x4 *)(z + v) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float y = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x[j], p.l2, -r.m)), r.pz, -r.smooth);
            if (v + j == lab) y = r.label;
            o.v[j] = (T)(v + j < classes ? y : 0.0f);
        }
        *(decltype(o) *)(d + v) = o;
    }
}

struct KeptArgs {
    const int *count, *label;
    const HeadRow *row;
    const float2 *stat;
    long long slots;
    int each, first, classes;         // classes a slot; the piece's first class and how many
    float l2;
    const void *kept;                 // kept and delta may be one
    long long ld_kept;
    void *delta;
    long long ld_delta, piece;
    int blocks;                       // workgroups a row
};

// What was kept to d, 16 bytes of d a lane.  Of exponentials: 2^(a L - m_tile + 15) * 2^(m_tile - 15 - m) * c / Z - c eps / V.
// Of products: as the logits' epilogue does it.  HBM: bfloat16 in place 4 bytes a logit (7782 x 131072: 697 us, 5.9 TB/s), float16
// 6 (1529 x 50021: 90 us, 5.1 TB/s).
template <typename T>
__global__ __launch_bounds__(kRowThreads) void head_kept_kernel(const KeptArgs p)
{
    constexpr int kVec = 16 / (int)sizeof(T);
    const int n = blockIdx.x / p.blocks;
    if (n >= *p.count) return;
    const int v = ((int)(blockIdx.x % p.blocks) * kRowThreads + (int)threadIdx.x) * kVec;
    if (v >= p.piece) return;
    const HeadRow r = p.row[n];
    constexpr int kWords = kVec * (int)sizeof(Kept<T>) / 16;
    union { u32x4 w[kWords]; Kept<T> e[kVec]; } x;
    union { u32x4 w; T d[kVec]; } o;
    const u32x4 *from = (const u32x4 *)((const Kept<T> *)p.kept + n * p.ld_kept + v);
#pragma unroll
    for (int i = 0; i < kWords; ++i) x.w[i] = from[i];
    float f = 0.0f;
    if constexpr (!__is_same(Kept<T>, float)) {
        const long long slot = (p.first + v) / p.each;
        const float m = slot < p.slots ? p.stat[n * p.slots + slot].x : -INFINITY;
        f = __builtin_amdgcn_exp2f(m - 15.0f - r.m) * r.pz;
    }
    const int lab = p.label[n] - p.first;
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        float d;
        if constexpr (__is_same(Kept<T>, float))
            d = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(x.e[i], p.l2, -r.m)), r.pz, -r.smooth);
        else
            d = __builtin_fmaf((float)x.e[i], f, -r.smooth);
        if (v + i == lab) d = r.label;
        o.d[i] = (T)(v + i < p.classes ? d : 0.0f);
    }
    *(u32x4 *)((T *)p.delta + n * p.ld_delta + v) = o.w;
}

// ----------------------------------------------------------------------- gradient products
struct GradArgs {
    const void *a, *b;                // logits: [m][k], [n][k];  dH: [k][m], [n][k];  dW: [k][m], [k][n]
    long long lda, ldb;
    int m, a_extent, n, k;            // a_extent: rows or columns of A that may be read
    const int *n_count, *k_count;     // device-side n or k, or NULL
    int tm;
    int parts;                        // k is cut into
    const HeadScale *scale;
    void *out;                        // [n][ldo], through row_of when given
    long long ldo;
    const int *row_of;
    const float *row_up;              // what row n is multiplied by besides, or NULL
    float *part;                      // [part][n][ld_part] instead of out, or NULL
    long long ld_part, part_stride;
    int add;                          // to what part holds
};

// A product whose result is written, or its parts: dH = d W, dW = d^T H, and few logits.  Matrix instructions at long k (7782 x
// 131072 x 2048 bfloat16: dH 3.29 ms, 1.27 PFLOP/s, the library's 1.35; dW 3.35, 1.25 PFLOP/s, the library's 1.10); at short k HBM
// (256 x 1000003 x 512: dW 484 us, 3.3 TB/s read and written).
template <typename T, int BM, int BN, int WM, int WN, bool A_KROWS, bool B_KROWS>
SSD_DEV void product(const GradArgs &p, int block, int blocks, char *smem)
{
    typedef TileStream<T, BM, BN, WM, WN, A_KROWS, B_KROWS> S;
    const int nn = uniform(p.n_count ? *p.n_count : p.n);
    const int kk = uniform(p.k_count ? *p.k_count : p.k);
    const int tn = (nn + BN - 1) / BN;
    const int each = ((kk + S::kBK - 1) / S::kBK + p.parts - 1) / p.parts * S::kBK;   // values of k a part, whole stages
    const auto unit = [&](int i, TileUnit &u) {
        const int part = i / (p.tm * tn);
        int m, n;
        tile_of(i - part * p.tm * tn, p.tm, tn, 8, m, n);
        const int k0 = part * each, left = kk - k0;
        u = TileUnit{m * BM, n * BN, k0, left < each ? left : each, part};
    };
    const auto set = [&](typename S::OpA &a, typename S::OpB &b, const TileUnit &u, int) {
        a.init(p.a, p.lda, u.m0, p.a_extent - u.m0, u.k0);
        b.init(p.b, p.ldb, u.n0, nn - u.n0, u.k0);
    };
    const float up = p.scale->up;
    const auto use = [&](f32x16 (&acc)[S::MF][S::NF], const TileUnit &u, int em, int en, int) {
        const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma unroll
        for (int nj = 0; nj < S::NF; ++nj) {
            const int n = u.n0 + en + nj * 32 + (lane & 31);
            bool in = n < nn;
            if (p.part) {
                float *o = p.part + u.part * p.part_stride + (long long)n * p.ld_part;
#pragma unroll
                for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const int m = u.m0 + em + mi * 32 + e * 2 + 4 * h;
                        if (in && m < p.m) {      // ld_part is a multiple of 4: the last group may pass m, not the row
                            f32x4 v = {acc[mi][nj][e], acc[mi][nj][e + 1], acc[mi][nj][e + 2], acc[mi][nj][e + 3]};
                            if (p.add) v += *(const f32x4 *)(o + m);
                            *(f32x4 *)(o + m) = v;
                        }
                    }
            } else {
                const int to = in ? (p.row_of ? p.row_of[n] : n) : -1;
                in = to >= 0;
                float up_n = up;
                if constexpr (__is_same(T, f16_t))
                    if (p.row_up && in) up_n *= p.row_up[n];
                T *o = (T *)p.out + (in ? (long long)to : 0) * p.ldo;
#pragma unroll
                for (int mi = 0; mi < S::MF; ++mi)
#pragma unroll
                    for (int e = 0; e < 16; e += 8) {
                        const int m = u.m0 + em + mi * 32 + e * 2;
                        float d[2][4];
#pragma unroll
                        for (int i = 0; i < 8; ++i) d[i >> 2][i & 3] = acc[mi][nj][e + i] * up_n;
                        store_pair<T>(o, m, d[0], d[1], p.m - m, in);
                    }
            }
        }
    };
    S::run(p.parts * p.tm * tn, block, blocks, smem, unit, set, use);
}

template <typename T, int BM, int BN, int WM, int WN, int BLOCKS, bool A_KROWS, bool B_KROWS>
__global__ __launch_bounds__(WM * WN * 64, BLOCKS * WM * WN / 4) void head_grad_kernel(const GradArgs p)
{
    __shared__ __align__(1024) char smem[TileStream<T, BM, BN, WM, WN, A_KROWS, B_KROWS>::kLds];
    product<T, BM, BN, WM, WN, A_KROWS, B_KROWS>(p, blockIdx.x, gridDim.x, smem);
}

// Both gradients of d in one launch, where neither fills the chip with its largest tiles: dH by the first h_blocks workgroups.
template <typename T, int HN, int HWM, int HWN>
__global__ __launch_bounds__(256, 2) void head_both_kernel(const GradArgs h, const GradArgs w, int h_blocks)
{
    __shared__ __align__(1024) char smem[TileStream<T, 128, 128, 2, 2, true, true>::kLds];
    if ((int)blockIdx.x < h_blocks)
        product<T, 128, HN, HWM, HWN, true, false>(h, blockIdx.x, h_blocks, smem);
    else
        product<T, 128, 128, 2, 2, true, true>(w, blockIdx.x - h_blocks, gridDim.x - h_blocks, smem);
}

struct JoinArgs {
    const float *part;
    long long ld_part, part_stride;
    int parts, m, n;
    int waves;                        // that share a piece's parts: with it goes the order of the sum, which is a product's own
    const int *n_count;
    const HeadScale *scale;
    void *out;
    long long ldo;
    const int *row_of;
    const float *row_up;
    long long first;                  // the launch's first workgroup of the product's
};

// The parts of a product over a long k, added in a fixed order: reads from the caches (128 parts of 256 x 512: 67 MB
// in 13 us).  Four values a lane, eight parts on their way at a time; up to WAVES waves share the parts of 256 values.
template <typename T, int WAVES>
SSD_DEV void join(const JoinArgs &p, long long block, f32x4 (&s_sum)[WAVES > 1 ? WAVES : 1][64])
{
    constexpr int kPieces = WAVES < 4 ? 4 / WAVES : 1;
    const int across = (p.m + 255) / 256, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long id = (block + p.first) * kPieces + (WAVES > 1 ? 0 : wave);
    const int n = (int)(id / across), m = ((int)(id % across) * 64 + lane) * 4;
    const bool in = n < (p.n_count ? *p.n_count : p.n) && m < p.m;
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) {
        const float *x = p.part + (long long)n * p.ld_part + m;
        const int each = (p.parts + p.waves - 1) / p.waves;
        int i = WAVES > 1 ? wave * each : 0;
        const int end = min(p.parts, i + each);
        for (; i + 8 <= end; i += 8) {
            f32x4 v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = *(const f32x4 *)(x + (i + j) * p.part_stride);
#pragma unroll
            for (int j = 0; j < 8; ++j) s += v[j];
        }
        for (; i < end; ++i) s += *(const f32x4 *)(x + i * p.part_stride);
    }
    if constexpr (WAVES > 1) {
        s_sum[wave][lane] = s;
        __syncthreads();
        if (wave != 0) return;
        for (int w = 1; w < p.waves; ++w) s += s_sum[w][lane];
    }
    if (!in) return;
    const int to = p.row_of ? p.row_of[n] : n;
    if (to < 0) return;
    const float up = p.row_up ? p.scale->up * p.row_up[n] : p.scale->up;
    T *o = (T *)p.out + to * p.ldo + m;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (m + j < p.m) o[j] = (T)(s[j] * up);
}

// One product's parts, or in one launch two products'.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void head_join_kernel(const JoinArgs a, const JoinArgs b, int a_blocks)
{
    __shared__ f32x4 s_sum[WAVES > 1 ? WAVES : 1][64];
    if ((int)blockIdx.x < a_blocks) join<T, WAVES>(a, blockIdx.x, s_sum);
    else join<T, WAVES>(b, blockIdx.x - a_blocks, s_sum);
}

// -------------------------------------------------------------------------------- plan
// Few logits are written (float32, they stay in the caches) and joined a row a workgroup, which a row of more than
// kFewClasses keeps too busy; and where they are little work too, the rows stay where they are: one launch less, while padded
// rows cost what the others cost.  A call of so little work is as long as its launches are many: a gradient takes three
// (products, rows, both gradients) instead of six.  Measured (rows x classes x dim, bfloat16, with gradients; before, now):
//   1000 x 1000 x 256 50 32 us,  4000 x 200 x 256 52 36,  1000 x 4000 x 256 62 51,  250 x 4000 x 1500 71 63,
//   4000 x 2000 x 64 63 54;  float32: 138 x 882 x 248 67 36,  1000 x 4000 x 128 81 75
constexpr long long kFewLogits = 1 << 23, kFewClasses = 1 << 14;
constexpr double kDirectWork = 1ll << 31, kDirectWorkF32 = 1 << 29;   // rows * classes * dim

// Everything that follows from sizes: which tile, how many parts, and the workspace.
struct HeadPlan {
    int es, vec;                      // bytes and 16-byte values of a type
    int tile, dh_tile, dw_tile;       // tiles of the three products (kTileM, kTileN)
    int bm, bn, each;                 // of the logits; each: classes of one wave's part of a tile
    int few_parts;                    // few tiles of logits: parts of their k, or 0
    long long few_ld;
    int pitch;                        // dim rounded up to 16 bytes
    bool copy_weight, keep;           // keep: of the last piece what d can be made of
    bool direct;                      // few logits and little work: the rows stay where they are
    long long class_tiles, slots;
    long long piece, ld_delta;        // classes a piece, and from one row of its d to the next
    int pieces;
    int chunks;                       // of counted rows, whose d of a piece is there at a time
    long long chunk_rows;
    int dh_parts, dw_parts;
    bool scale_in_place;              // float16's rows times 2^-shift: nothing reads them as they were after their statistics
    size_t o_few, o_blocks, o_rows, o_row_up, o_scaled, o_weight, o_row, o_label, o_count, o_scale, o_stat, o_sumz, o_zl, o_out;
    size_t o_delta, o_kept, o_dh, o_dw;
    size_t bytes;
};

constexpr size_t kDeltaBytes = (size_t)1 << 31;    // of one piece's d (256 bytes a row, half as much again at most, come on top)
constexpr long long kChunkRow = 8192;              // bytes of a row of d at most, where rows are cut

// From which dim on something is kept.  Measured (rows x classes x dim, taken again, kept; us):
//   bfloat16  1000 x 30000 x 128 140 141,  60 x 200000 x 256 116 107,  256 x 1000003 x 512 1710 1540,  8192 x 131072 x 768 6360 5560
//   float16   1000 x 30000 x 256 145 149,  300 x 100000 x 512 293 268,  4096 x 50000 x 2048 3127 2689
//   float32   500 x 20000 x 64 138 130,  2000 x 30000 x 512 2029 1608: always
constexpr int kKeepAboveBf16 = 192, kKeepAboveF16 = 384;

size_t put(size_t &at, size_t bytes)
{
    const size_t o = at;
    at = (at + bytes + 255) / 256 * 256;
    return o;
}

constexpr int kTileM[3] = {128, 128, 256}, kTileN[3] = {64, 128, 256};

long long tiles(int tile, long long m, long long n)
{
    return (m + kTileM[tile] - 1) / kTileM[tile] * ((n + kTileN[tile] - 1) / kTileN[tile]);
}

// The tile of a product whose k cannot be cut.  The largest does most per value read, but keeps one workgroup a compute
// unit busy for long; measured (rows x classes x dim, bfloat16, value alone; tiles of 128x64, 128x128, 256x256):
//   512 x 32768 x 1024 - 61 55 us,  256 x 8192 x 1024 25 26 43,  1024 x 1024 x 1024 24 29 45,  8192 x 4096 x 2048 - 201 170
// float32, whose instructions take sixteen times as long: 61 x 10007 x 512 34 53,  2048 x 8192 x 512 167 162.
int whole_tile(long long m, long long n, int es)
{
    if (es == 2 && n > 128 && tiles(2, m, n) >= 256) return 2;
    if (n > 64 && tiles(1, m, n) >= (es == 2 ? 256 : 1024)) return 1;
    return 0;
}

constexpr int kPartBytes = 128 << 20;  // of a product's parts together
constexpr long long kJoinBlocks = 1 << 20;    // workgroups of one join

// The tile of a product whose k may be cut, and into how many parts: so that the chip is filled, at least eight stages each.
// The largest tile does what it computes about 1.45 times as fast as the next one, so it may not compute more than that many
// times as much: 4000 x 30000 x 64 bfloat16 282 us, 313 with it;  6287 x 30000 x 384 843, 777 with it.
// (rows_of_k: both operands' rows are of k, which the smallest tile does not take.)
void cut_tile(long long m, long long n, long long k_stages, int es, bool rows_of_k, int &tile, int &parts)
{
    const bool wide = 4 * tiles(2, m, n) * 20 <= 29 * tiles(1, m, n);
    if (es == 2 && n > 128 && wide && tiles(2, m, n) * k_stages >= 256 * 16) tile = 2;
    else if (rows_of_k || (n > 64 && tiles(1, m, n) * k_stages >= 512 * 12)) tile = 1;
    else tile = 0;
    const long long units = n > 0 ? tiles(tile, m, n) : 1, fill = tile == 2 ? 256 : (tile == 1 ? 512 : 768);
    long long p = fill / units;
    if (p > k_stages / 8) p = k_stages / 8;
    const long long most = ((long long)kPartBytes / 4) / (m * (n > 0 ? n : 1) + 1);
    if (p > most) p = most;
    parts = p < 1 ? 1 : (int)p;
}

HeadPlan make_plan(long long rows, long long classes, long long dim, long long weight_ld, int dtype, float smoothing,
                   bool grad_hidden, bool grad_weight)
{
    HeadPlan q = {};
    q.es = dtype == SSDBOX_DTYPE_F32 ? 4 : 2;
    q.vec = 16 / q.es;
    q.pitch = (int)((dim + q.vec - 1) / q.vec * q.vec);
    q.copy_weight = dim % q.vec != 0 || weight_ld % q.vec != 0;
    const int bk = kStageBytes / q.es;
    q.tile = whole_tile(classes, rows, q.es);
    q.bm = kTileM[q.tile];
    q.bn = kTileN[q.tile];
    q.each = q.tile == 2 ? 128 : (q.tile == 1 ? 64 : 32);
    // Much of the chip idle over a long k: the logits are cut along it, and few enough to be written.  Measured (cut, whole;
    // value and gradients): 25 x 17213 x 1701 float32 233 301 us, 1024 x 2048 x 2048 bfloat16 102 110, 64 x 20000 x 1024 96 72.
    const long long n_tiles = tiles(q.tile, classes, rows);
    const bool few = rows > 0 && rows * classes <= kFewLogits && classes <= kFewClasses;
    q.direct = few && rows <= kCountFrom &&
               (double)rows * (double)classes * (double)dim <= (q.es == 4 ? kDirectWorkF32 : kDirectWork);
    if (few || (rows > 0 && q.pitch >= 16 * bk && (n_tiles < 128 || (n_tiles < 384 && (q.es == 4 || rows >= 512))))) {
        int tile = 0;
        cut_tile(classes, rows, (q.pitch + bk - 1) / bk, q.es, false, tile, q.few_parts);
        q.tile = tile;
        q.few_ld = (classes + 3) / 4 * 4;
    }
    q.class_tiles = (classes + q.bm - 1) / q.bm;
    q.slots = q.class_tiles * (q.bm / q.each);
    const bool grad = grad_hidden || grad_weight;
    q.chunks = 1;
    q.chunk_rows = rows;
    if (grad) {
        const long long row_bytes = rows * q.es > 0 ? rows * q.es : 1;
        long long most = (long long)kDeltaBytes / row_bytes / 256 * 256;
        if (most < 256) most = 256;
        if (most > (1 << 21)) most = 1 << 21;
        const long long whole = (classes + 255) / 256 * 256;
        q.pieces = (int)((whole + most - 1) / most);
        q.piece = ((whole + q.pieces - 1) / q.pieces + 255) / 256 * 256;
        q.pieces = (int)((whole + q.piece - 1) / q.piece);
        // 256 bytes more than the piece, often a power of two: the rows that one store or load touches would otherwise all
        // lie in one channel of the L2 (d of 8192 x 65536: 2.2 -> 1.9 ms)
        q.ld_delta = q.piece + 256 / q.es;
        if (q.few_parts) {
            if ((size_t)(rows * q.ld_delta) * q.es > kDeltaBytes) q.ld_delta = (classes + 63) / 64 * 64;
        } else if (rows * q.es * 256 > (long long)kDeltaBytes) {
            // So many rows that a piece of any width is too much: they are cut, too.  dW is added over the chunks, which costs
            // less than dH over pieces, so pieces are wide again (ms, pieces of 256 classes of all rows, of 1024, 2048, 4096 of
            // chunks:  2000000 x 4000 x 64 float32 70.2 67.4 67.8 77.6,  3000000 x 4000 x 64 bfloat16 43.9 37.5 35.7 33.6).
            const long long widest = kChunkRow / q.es;
            q.pieces = (int)((whole + widest - 1) / widest);
            q.piece = ((whole + q.pieces - 1) / q.pieces + 255) / 256 * 256;
            q.pieces = (int)((whole + q.piece - 1) / q.piece);
            q.ld_delta = q.piece + 256 / q.es;
            q.chunk_rows = (long long)kDeltaBytes / (q.ld_delta * q.es) / 256 * 256;
            q.chunks = (int)((rows + q.chunk_rows - 1) / q.chunk_rows);
        }
        // The pass over what is kept and its stores move bytes, the products it spares take 2 dim operations a logit.  Of chunks
        // only float32 of one piece keeps them (kept, taken again, ms: 3000000 x 200 x 512 float32 28.6 33.8; 4500000 x 200 x 512
        // bfloat16 18.1 17.0).
        if (q.few_parts) q.keep = false;
        else if (dtype == SSDBOX_DTYPE_F32) q.keep = q.chunks == 1 || q.pieces == 1;
        else if (q.chunks > 1) q.keep = false;
        else if (dtype == SSDBOX_DTYPE_BF16) q.keep = dim > kKeepAboveBf16;
        else q.keep = dim > kKeepAboveF16 && q.pieces == 1 && (size_t)(rows * q.ld_delta) * 4 <= kDeltaBytes;
    }
    size_t at = 0;
    q.o_few = put(at, (size_t)q.few_parts * rows * q.few_ld * 4);
    q.o_count = put(at, (1 + (q.chunks > 1 ? q.chunks : 0)) * 4);
    q.o_scale = put(at, 256);
    q.o_blocks = put(at, rows > kCountFrom ? (rows + kCountRows - 1) / kCountRows * 8 : 0);
    q.o_row = put(at, rows * 4);
    q.o_label = put(at, rows * 4);
    q.o_zl = put(at, rows * 4);
    q.o_out = put(at, rows * sizeof(HeadRow));
    q.o_rows = put(at, (size_t)rows * q.pitch * q.es);
    q.scale_in_place = q.few_parts || (q.keep && q.pieces == 1);
    const bool half = dtype == SSDBOX_DTYPE_F16 && grad;
    q.o_row_up = put(at, half ? rows * 4 : 0);
    q.o_scaled = put(at, half && grad_weight && !q.scale_in_place ? (size_t)rows * q.pitch * q.es : 0);
    q.o_stat = put(at, q.few_parts ? 0 : (size_t)rows * q.slots * sizeof(float2));
    q.o_sumz = put(at, smoothing != 0.0f && !q.few_parts ? (size_t)rows * q.slots * 4 : 0);
    q.o_weight = put(at, q.copy_weight ? (size_t)classes * q.pitch * q.es : 0);
    q.o_delta = put(at, grad ? (size_t)q.chunk_rows * q.ld_delta * q.es : 0);
    q.o_kept = put(at, q.keep && dtype == SSDBOX_DTYPE_F16 ? (size_t)rows * q.ld_delta * 4 : 0);
    const long long wide = (dim + 3) / 4 * 4, piece_classes = classes < q.piece ? classes : q.piece;
    if (grad) {
        cut_tile(dim, q.chunk_rows, (q.piece + bk - 1) / bk, q.es, false, q.dh_tile, q.dh_parts);
        cut_tile(dim, piece_classes, (q.chunk_rows + bk - 1) / bk, q.es, true, q.dw_tile, q.dw_parts);
        const long long h = rows > 0 ? tiles(q.dh_tile, dim, q.chunk_rows) : 1, w = tiles(1, dim, piece_classes);
        if (q.dh_tile < 2 && q.dw_tile < 2 && w < 512) {
            // one launch for both, at two workgroups a compute unit: dW takes half, or its tiles, dH what is left (each cut as
            // if alone, 1000 x 1000 x 2048 bfloat16 takes 70 us and not 55, 61 x 10007 x 512 float32 64 and not 59)
            const long long most = w < 256 ? 256 / w : 1;
            if (q.dw_parts > most) q.dw_parts = (int)most;
            long long left = 512 - w * q.dw_parts;
            if (left < 128) left += 512;
            if (q.dh_parts > left / h) q.dh_parts = left > h ? (int)(left / h) : 1;
        }
        if (!grad_hidden) q.dh_parts = 0;
        if (!grad_weight) q.dw_parts = 0;
        q.o_dh = put(at, grad_hidden && (q.dh_parts > 1 || q.pieces > 1) ? (size_t)q.dh_parts * rows * wide * 4 : 0);
        q.o_dw = put(at, q.dw_parts > 1 || (q.dw_parts && q.chunks > 1) ? (size_t)q.dw_parts * q.piece * wide * 4 : 0);
    }
    q.bytes = at;
    return q;
}

struct HeadCall {
    ssdbox_ctx *ctx;
    const void *hidden, *weight, *labels;
    long long hidden_ld, weight_ld;
    int label_bytes;
    long long rows, classes, dim;
    float logit_scale, smoothing;
    const float *grad_loss;
    float *loss;
    void *grad_hidden, *grad_weight;
    char *ws;
};

// Workgroups that stay for the whole launch, as many as run at once.
unsigned stay(const HeadCall &c, long long units, int each)
{
    const long long most = (long long)c.ctx->num_cus * each;
    return (unsigned)(units < most ? (units > 0 ? units : 1) : most);
}

template <typename T, int BM, int BN, int WM, int WN, int BLOCKS, int WHAT>
void launch_tiles(const HeadCall &c, const LogitArgs &a)
{
    const unsigned grid = stay(c, (long long)a.tiles * ((c.rows + BN - 1) / BN), BLOCKS);
    launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_logit_kernel<T, BM, BN, WM, WN, BLOCKS, WHAT>, dim3(grid),
                 dim3(WM * WN * 64), a);
}

template <typename T, int WHAT>
void launch_logits(const HeadCall &c, int tile, const LogitArgs &a)
{
    if (tile == 0) return launch_tiles<T, 128, 64, 4, 1, 2, WHAT>(c, a);
    if (tile == 1) return launch_tiles<T, 128, 128, 2, 2, 2, WHAT>(c, a);
    if constexpr (sizeof(T) == 2) launch_tiles<T, 256, 256, 2, 4, 1, WHAT>(c, a);
}

template <typename T, int BM, int BN, int WM, int WN, int BLOCKS, bool A_KROWS, bool B_KROWS>
void launch_product(const HeadCall &c, GradArgs a)
{
    a.tm = (a.m + BM - 1) / BM;
    const dim3 grid(stay(c, (long long)a.parts * a.tm * ((a.n + BN - 1) / BN), BLOCKS)), block(WM * WN * 64);
    launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_grad_kernel<T, BM, BN, WM, WN, BLOCKS, A_KROWS, B_KROWS>, grid, block, a);
}

template <typename T, bool A_KROWS, bool B_KROWS>
void launch_product(const HeadCall &c, int tile, const GradArgs &a)
{
    if constexpr (!B_KROWS)
        if (tile == 0) return launch_product<T, 128, 64, 4, 1, 3, A_KROWS, B_KROWS>(c, a);
    if constexpr (sizeof(T) == 2)
        if (tile == 2) return launch_product<T, 256, 256, 2, 4, 1, A_KROWS, B_KROWS>(c, a);
    launch_product<T, 128, 128, 2, 2, 2, A_KROWS, B_KROWS>(c, a);
}

JoinArgs join_args(const GradArgs &a)
{
    JoinArgs j = {};
    j.part = a.part;
    j.ld_part = a.ld_part;
    j.part_stride = a.part_stride;
    j.parts = a.parts;
    j.waves = a.parts < 32 ? 1 : (a.parts < 256 ? 4 : 16);
    j.m = a.m;
    j.n = a.n;
    j.n_count = a.n_count;
    j.scale = a.scale;
    j.out = a.out;
    j.ldo = a.ldo;
    j.row_of = a.row_of;
    j.row_up = a.row_up;
    return j;
}

// Workgroups of the whole join of a product by WAVES waves.
template <int WAVES>
long long join_blocks(const JoinArgs &j)
{
    const long long pieces = (long long)j.n * ((j.m + 255) / 256), each = WAVES < 4 ? 4 / WAVES : 1;
    return (pieces + each - 1) / each;
}

template <typename T, int WAVES>
void launch_join(const HeadCall &c, const JoinArgs &a, const JoinArgs &b)
{
    const unsigned blocks = (unsigned)join_blocks<WAVES>(a);
    launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_join_kernel<T, WAVES>, dim3(blocks + (unsigned)join_blocks<WAVES>(b)),
                 dim3(WAVES < 4 ? 256 : WAVES * 64), a, b, (int)blocks);
}

// One product's parts by themselves, so many workgroups a launch that it stays far below 2^32 threads.
template <typename T, int WAVES>
void launch_join(const HeadCall &c, JoinArgs a)
{
    const long long all = join_blocks<WAVES>(a);
    for (; a.first < all; a.first += kJoinBlocks) {
        const unsigned blocks = (unsigned)(all - a.first < kJoinBlocks ? all - a.first : kJoinBlocks);
        launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_join_kernel<T, WAVES>, dim3(blocks), dim3(WAVES < 4 ? 256 : WAVES * 64), a,
                     JoinArgs{}, (int)blocks);
    }
}

template <typename T>
void launch_join(const HeadCall &c, const GradArgs &a)
{
    const JoinArgs x = join_args(a);
    if (x.waves == 1) launch_join<T, 1>(c, x);
    else if (x.waves == 4) launch_join<T, 4>(c, x);
    else launch_join<T, 16>(c, x);
}

// Two products' parts, in one launch where it is no long one.
template <typename T>
void launch_join(const HeadCall &c, const GradArgs &a, const GradArgs &b)
{
    const JoinArgs x = join_args(a), y = join_args(b);
    const int waves = x.waves > y.waves ? x.waves : y.waves;
    if (join_blocks<4>(x) + join_blocks<4>(y) > kJoinBlocks) {    // (a piece each: the most that any number of waves takes)
        launch_join<T>(c, a);
        launch_join<T>(c, b);
    }
    else if (waves == 1) launch_join<T, 1>(c, x, y);
    else if (waves == 4) launch_join<T, 4>(c, x, y);
    else launch_join<T, 16>(c, x, y);
}

// dH and dW of one piece, each if it is wanted, and their parts joined if they are whole: two launches for both where the
// tiles are the smaller ones.  Otherwise dH's parts are joined at once, from the caches (256 x 1000003 x 512: 12 us, and 22
// after dW has gone through them).
template <typename T>
void launch_gradients(const HeadCall &c, const HeadPlan &q, GradArgs h, GradArgs w, bool want_h, bool want_w, bool join_h,
                      bool join_w)
{
    if (want_h && want_w && q.dh_tile < 2 && q.dw_tile < 2) {
        h.tm = (h.m + 127) / 128;
        w.tm = (w.m + 127) / 128;
        const unsigned hb = stay(c, (long long)h.parts * h.tm * ((h.n + kTileN[q.dh_tile] - 1) / kTileN[q.dh_tile]), 2);
        const unsigned wb = stay(c, (long long)w.parts * w.tm * ((w.n + 127) / 128), 2);
        if (q.dh_tile == 0)
            launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_both_kernel<T, 64, 4, 1>, dim3(hb + wb), dim3(256), h, w, (int)hb);
        else
            launch_stage(c.ctx, SSDBOX_STAGE_LOSS, head_both_kernel<T, 128, 2, 2>, dim3(hb + wb), dim3(256), h, w, (int)hb);
        if (join_h && join_w) launch_join<T>(c, h, w);
        else if (join_h) launch_join<T>(c, h);
        else if (join_w) launch_join<T>(c, w);
        return;
    }
    if (want_h) launch_product<T, true, false>(c, q.dh_tile, h);
    if (join_h) launch_join<T>(c, h);
    if (want_w) launch_product<T, true, true>(c, q.dw_tile, w);
    if (join_w) launch_join<T>(c, w);
}

template <typename T>
int run_head(const HeadCall &c, const HeadPlan &q, int dtype)
{
    ssdbox_ctx *ctx = c.ctx;
    const bool grad = c.grad_hidden || c.grad_weight;
    int *count = (int *)(c.ws + q.o_count), *row = (int *)(c.ws + q.o_row), *label = (int *)(c.ws + q.o_label);
    HeadScale *scale = (HeadScale *)(c.ws + q.o_scale);
    T *rows = (T *)(c.ws + q.o_rows);
    float *row_up = dtype == SSDBOX_DTYPE_F16 && grad && c.grad_loss ? (float *)(c.ws + q.o_row_up) : nullptr;
    T *scaled = row_up && !q.scale_in_place ? (T *)(c.ws + q.o_scaled) : rows;
    void *kept = c.ws + (dtype == SSDBOX_DTYPE_F16 ? q.o_kept : q.o_delta);

    PrepArgs s = {};
    s.labels = c.labels;
    s.label_bytes = c.label_bytes;
    s.rows = (int)c.rows;
    s.classes = c.classes;
    s.grad_loss = grad ? c.grad_loss : nullptr;
    s.logit_scale = c.logit_scale;
    s.smoothing = c.smoothing;
    s.scaled = dtype != SSDBOX_DTYPE_F32;
    s.hidden = c.hidden;
    s.ld = c.hidden_ld;
    s.dim = (int)c.dim;
    s.pitch = q.pitch;
    s.place_count = count;
    s.chunks = q.chunks;
    s.chunk_rows = (int)q.chunk_rows;
    s.row = row;
    s.label = label;
    s.scale = scale;
    s.loss = c.loss;
    s.out = rows;
    s.grad_hidden = c.grad_hidden;
    const int n_blocks = (int)((c.rows + kCountRows - 1) / kCountRows);
    if (c.rows > kCountFrom) {
        s.block_count = (int *)(c.ws + q.o_blocks);
        s.block_max = (float *)(c.ws + q.o_blocks) + n_blocks;
        launch_stage(ctx, SSDBOX_STAGE_LOSS, head_count_kernel, dim3((unsigned)n_blocks), dim3(kRowThreads), s);
    }
    const unsigned n_prep = c.rows > 0 ? (unsigned)((c.rows + kRowsEach - 1) / kRowsEach) : 1;
    unsigned n_pitch = 0;
    const T *weight = (const T *)c.weight;
    long long ldw = c.weight_ld;
    if (q.copy_weight && c.rows > 0) {
        n_pitch = stay(c, (c.classes * (q.pitch / q.vec) + kRowThreads - 1) / kRowThreads, 16);
        s.weight = weight;
        s.weight_ld = ldw;
        s.weight_out = c.ws + q.o_weight;
        weight = (const T *)(c.ws + q.o_weight);
        ldw = q.pitch;
    }
    s.prep_blocks = (int)n_prep;
    s.stay = q.direct;
    // (rows as they are: 16-byte pieces, and a tile's rows within the 32 bits of its offsets)
    if (!q.direct || q.copy_weight || c.hidden_ld % q.vec != 0 || (uintptr_t)c.hidden % 16 != 0 || c.hidden_ld > kMostLd) {
        launch_stage(ctx, SSDBOX_STAGE_LOSS, head_prep_kernel<T>, dim3(n_prep + n_pitch), dim3(kRowThreads), s);
        s.hidden = rows;
        s.ld = q.pitch;
    }

    LogitArgs l = {};
    l.weight = weight;
    l.rows = rows;
    l.ldw = ldw;
    l.ldh = q.pitch;
    l.dim = q.pitch;
    l.classes = (int)c.classes;
    l.tiles = (int)q.class_tiles;
    l.l2 = c.logit_scale * kLog2e;
    l.count = count;
    l.label = label;
    l.stat = (float2 *)(c.ws + q.o_stat);
    l.sum_z = c.smoothing != 0.0f ? (float *)(c.ws + q.o_sumz) : nullptr;
    l.slots = q.slots;
    l.z_label = (float *)(c.ws + q.o_zl);
    l.row = (const HeadRow *)(c.ws + q.o_out);
    RowArgs r = {};
    // Logits and rows of one chunk, or of all.
    const auto logits_and_rows = [&](long long row0, long long n_rows, const int *counted) {
        LogitArgs a = l;
        a.rows = rows + row0 * q.pitch;
        a.count = counted;
        a.label = label + row0;
        a.stat = l.stat + row0 * q.slots;
        if (a.sum_z) a.sum_z += row0 * q.slots;
        a.z_label = l.z_label + row0;
        if (q.keep) {
            a.kept_from = (int)((q.pieces - 1) * q.piece);
            a.delta = kept;
            a.ld_delta = q.ld_delta;
            launch_logits<T, kStatKeep>(c, q.tile, a);
        } else {
            launch_logits<T, kStat>(c, q.tile, a);
        }
        RowArgs b = r;
        b.count = counted;
        b.row = row + row0;
        b.label = a.label;
        b.stat = a.stat;
        b.sum_z = a.sum_z;
        b.z_label = a.z_label;
        if (b.out) b.out += row0;
        if (b.row_up) b.row_up += row0;
        b.values = a.rows;
        if (b.scaled) b.scaled = scaled + row0 * q.pitch;
        if (q.slots < 2048 || n_rows > kMostRows / 4)
            launch_stage(ctx, SSDBOX_STAGE_LOSS, head_row_kernel<256>, dim3((unsigned)n_rows), dim3(256), b);
        else
            launch_stage(ctx, SSDBOX_STAGE_LOSS, head_row_kernel<1024>, dim3((unsigned)n_rows), dim3(1024), b);
    };
    const bool keep_chunks = q.keep && q.chunks > 1;             // of one piece: what is kept of a chunk becomes its d at once
    if (c.rows > 0) {
        r.count = count;
        r.row = row;
        r.label = label;
        r.stat = l.stat;
        r.sum_z = l.sum_z;
        r.slots = q.slots;
        r.z_label = l.z_label;
        r.l2 = l.l2;
        r.logit_scale = c.logit_scale;
        r.smoothing = c.smoothing;
        r.classes = c.classes;
        r.rows = (int)c.rows;
        r.grad_loss = c.grad_loss;
        r.scale = scale;
        r.loss = c.loss;
        r.out = grad ? (HeadRow *)(c.ws + q.o_out) : nullptr;
        r.row_up = row_up;
        r.values = rows;
        r.scaled = row_up && c.grad_weight ? scaled : nullptr;
        r.pitch = q.pitch;
        if (q.few_parts) {
            GradArgs f = {};
            f.a = weight;
            f.lda = ldw;
            f.b = q.direct ? s.hidden : rows;
            f.ldb = q.direct ? s.ld : q.pitch;
            f.m = f.a_extent = (int)c.classes;
            f.n = (int)c.rows;
            f.n_count = q.direct ? nullptr : count;
            f.k = q.pitch;
            f.parts = q.few_parts;
            f.scale = scale;
            f.part = (float *)(c.ws + q.o_few);
            f.ld_part = q.few_ld;
            f.part_stride = c.rows * q.few_ld;
            launch_product<T, false, false>(c, q.tile, f);
            T *d = (T *)(c.ws + q.o_delta);
            const auto few = [&](auto kernel, int threads) {
                launch_stage(ctx, SSDBOX_STAGE_LOSS, kernel, dim3((unsigned)c.rows), dim3(threads), r, s, f.part, f.ld_part,
                             f.part_stride, f.parts, d, q.ld_delta);
            };
            if (c.classes < 4096) few(q.direct ? head_few_kernel<T, 256, true> : head_few_kernel<T, 256, false>, 256);
            else few(q.direct ? head_few_kernel<T, 1024, true> : head_few_kernel<T, 1024, false>, 1024);
        } else if (!keep_chunks) {
            logits_and_rows(0, c.rows, count);
        }
    }
    if (!grad) return SSDBOX_OK;

    const long long wide = (c.dim + 3) / 4 * 4;
    for (int turn = 0; turn < q.pieces * q.chunks; ++turn) {
        const int piece = turn / q.chunks, chunk = turn % q.chunks;
        const int i = q.keep ? q.pieces - 1 - piece : piece;     // what is kept has to be used before its place is
        const long long first = i * q.piece, row0 = chunk * q.chunk_rows;
        const int n_class = (int)(c.classes - first < q.piece ? c.classes - first : q.piece);
        const int n_rows = (int)(c.rows - row0 < q.chunk_rows ? c.rows - row0 : q.chunk_rows);
        const int *counted = q.chunks > 1 ? count + 1 + chunk : count;
        T *delta = (T *)(c.ws + q.o_delta);
        if (q.few_parts) {
            // d is there: few tiles are one piece
        } else if (c.rows > 0 && q.keep && (turn == 0 || keep_chunks)) {
            if (keep_chunks) logits_and_rows(row0, n_rows, counted);
            KeptArgs k = {};
            k.count = counted;
            k.label = label + row0;
            k.row = l.row + row0;
            k.stat = l.stat + row0 * q.slots;
            k.slots = q.slots;
            k.each = q.each;
            k.first = (int)first;
            k.classes = n_class;
            k.l2 = l.l2;
            k.kept = kept;
            k.ld_kept = q.ld_delta;
            k.delta = delta;
            k.ld_delta = q.ld_delta;
            k.piece = q.piece;
            k.blocks = (int)((q.piece + kRowThreads * q.vec - 1) / (kRowThreads * q.vec));
            launch_stage(ctx, SSDBOX_STAGE_LOSS, head_kept_kernel<T>, dim3((unsigned)((long long)n_rows * k.blocks)),
                         dim3(kRowThreads), k);
        } else if (c.rows > 0) {
            LogitArgs d = l;
            d.weight = weight + first * ldw;
            d.rows = rows + row0 * q.pitch;
            d.count = counted;
            d.label = label + row0;
            d.row = l.row + row0;
            d.classes = n_class;
            d.first = (int)first;
            d.tiles = (n_class + q.bm - 1) / q.bm;
            d.delta = delta;
            d.ld_delta = q.ld_delta;
            launch_logits<T, kDelta>(c, q.tile, d);
        }
        GradArgs h = {}, w = {};
        h.m = w.m = (int)c.dim;
        h.a_extent = w.a_extent = q.pitch;
        h.scale = w.scale = scale;
        h.ldo = w.ldo = c.dim;
        h.ldb = w.ldb = q.ld_delta;
        h.b = w.b = delta;
        const bool want_h = c.grad_hidden && c.rows > 0;
        bool join_h = false, join_w = false;
        if (want_h) {
            h.a = weight + first * ldw;
            h.lda = ldw;
            h.n = n_rows;
            h.n_count = q.direct ? nullptr : counted;
            h.k = n_class;
            h.parts = q.dh_parts;
            h.out = c.grad_hidden;
            h.row_of = row + row0;
            h.row_up = row_up ? row_up + row0 : nullptr;
            if (q.dh_parts > 1 || q.pieces > 1) {
                h.part = (float *)(c.ws + q.o_dh) + row0 * wide;
                h.ld_part = wide;
                h.part_stride = c.rows * wide;
                h.add = piece > 0;
                join_h = piece == q.pieces - 1;
            }
        }
        if (c.grad_weight) {
            w.a = scaled + row0 * q.pitch;
            w.lda = q.pitch;
            w.n = n_class;
            w.k = n_rows;
            w.k_count = q.direct ? nullptr : counted;
            w.parts = q.dw_parts;
            w.out = (T *)c.grad_weight + first * c.dim;
            if (q.dw_parts > 1 || q.chunks > 1) {
                w.part = (float *)(c.ws + q.o_dw);
                w.ld_part = wide;
                w.part_stride = q.piece * wide;
                w.add = chunk > 0;
                join_w = chunk == q.chunks - 1;
            }
        }
        launch_gradients<T>(c, q, h, w, want_h, c.grad_weight != nullptr, join_h, join_w);
    }
    return SSDBOX_OK;
}

int check_sizes(int64_t rows, int64_t classes, int64_t dim, int64_t weight_ld, int dtype, float smoothing)
{
    SSD_REQUIRE(dtype == SSDBOX_DTYPE_F32 || dtype == SSDBOX_DTYPE_F16 || dtype == SSDBOX_DTYPE_BF16,
                "linear_cross_entropy: dtype %d", dtype);
    SSD_REQUIRE(rows >= 0 && rows <= kMostRows, "linear_cross_entropy: %lld rows outside [0, 2^24)", (long long)rows);
    SSD_REQUIRE(classes >= 1 && classes <= (1 << 28), "linear_cross_entropy: %lld classes outside [1, 2^28]",
                (long long)classes);
    SSD_REQUIRE(dim >= 1 && dim <= (1 << 20), "linear_cross_entropy: dim %lld outside [1, 2^20]", (long long)dim);
    SSD_REQUIRE(weight_ld >= dim && weight_ld <= kMostLd, "linear_cross_entropy: weight row stride %lld outside [%lld, 2^21]",
                (long long)weight_ld, (long long)dim);
    SSD_REQUIRE(smoothing >= 0.0f && smoothing < 1.0f, "linear_cross_entropy: label_smoothing %g outside [0, 1)", smoothing);
    return SSDBOX_OK;
}

}  // namespace

extern "C" int ssdbox_linear_cross_entropy_workspace(int64_t rows, int64_t classes, int64_t dim, int64_t weight_ld,
                                                     int dtype, float label_smoothing, int grad_hidden, int grad_weight,
                                                     size_t *bytes)
{
    SSD_REQUIRE(bytes != nullptr, "linear_cross_entropy_workspace: bytes is NULL");
    int rc = check_sizes(rows, classes, dim, weight_ld, dtype, label_smoothing);
    if (rc != SSDBOX_OK) return rc;
    *bytes = make_plan(rows, classes, dim, weight_ld, dtype, label_smoothing, grad_hidden != 0, grad_weight != 0).bytes;
    return SSDBOX_OK;
}

extern "C" int ssdbox_linear_cross_entropy(ssdbox_ctx *ctx, const void *d_hidden, int64_t hidden_ld, const void *d_weight,
                                           int64_t weight_ld, const void *d_labels, int label_bytes, int64_t rows,
                                           int64_t classes, int64_t dim, int dtype, float logit_scale,
                                           float label_smoothing, const float *d_grad_loss, float *d_loss,
                                           void *d_grad_hidden, void *d_grad_weight, void *d_workspace,
                                           size_t workspace_bytes)
{
    SSD_REQUIRE(ctx != nullptr, "linear_cross_entropy: ctx is NULL");
    int rc = check_sizes(rows, classes, dim, weight_ld, dtype, label_smoothing);
    if (rc != SSDBOX_OK) return rc;
    SSD_REQUIRE(label_bytes == 4 || label_bytes == 8, "linear_cross_entropy: labels of %d bytes", label_bytes);
    SSD_REQUIRE(hidden_ld >= dim, "linear_cross_entropy: hidden row stride %lld below dim %lld", (long long)hidden_ld,
                (long long)dim);
    SSD_REQUIRE(logit_scale > 0.0f && logit_scale <= 1e6f, "linear_cross_entropy: logit_scale %g outside (0, 1e6]",
                logit_scale);
    SSD_REQUIRE(d_weight && d_workspace && (rows == 0 || (d_hidden && d_labels && d_loss)),
                "linear_cross_entropy: NULL buffer");
    const HeadPlan q = make_plan(rows, classes, dim, weight_ld, dtype, label_smoothing, d_grad_hidden != nullptr,
                                 d_grad_weight != nullptr);
    SSD_REQUIRE(workspace_bytes >= q.bytes, "linear_cross_entropy: workspace of %zu bytes, %zu needed", workspace_bytes,
                q.bytes);
    SSD_REQUIRE(((uintptr_t)d_workspace % 256) == 0 && ((uintptr_t)d_weight % 16) == 0 &&
                    ((uintptr_t)d_grad_hidden % 16) == 0 && ((uintptr_t)d_grad_weight % 16) == 0,
                "linear_cross_entropy: weight and gradients have to start at 16 bytes, the workspace at 256");
    SSD_REQUIRE(q.class_tiles * ((rows + q.bn - 1) / q.bn) < (1ll << 31) &&
                    (q.pieces == 0 || (dim + 127) / 128 * ((rows + 63) / 64) * q.dh_parts < (1ll << 31)),
                "linear_cross_entropy: %lld rows x %lld classes", (long long)rows, (long long)classes);

    DeviceGuard guard(ctx->device);
    HeadCall c = {ctx, d_hidden, d_weight, d_labels, hidden_ld, weight_ld, label_bytes, rows, classes, dim, logit_scale,
                  label_smoothing, d_grad_loss, d_loss, d_grad_hidden, d_grad_weight, (char *)d_workspace};
    if (dtype == SSDBOX_DTYPE_F32) rc = run_head<float>(c, q, dtype);
    else if (dtype == SSDBOX_DTYPE_F16) rc = run_head<f16_t>(c, q, dtype);
    else rc = run_head<bf16_t>(c, q, dtype);
    if (rc != SSDBOX_OK) return rc;
    SSD_CHECK_HIP(hipGetLastError());
    return SSDBOX_OK;
}
