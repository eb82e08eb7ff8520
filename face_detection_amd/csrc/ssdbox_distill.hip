// Distillation from a teacher's top logits, with the gradient with respect to the student's logits.
//
// u = z / tau, p = softmax(u) over all classes; the teacher gives K (class, logit) pairs a row, S their classes:
//   without its log-sum-exp: q = softmax over the K of t / tau, no rest
//   with it (at tau):        q = exp(t / tau - lse), q_r = 1 - sum q; the classes outside S are one bucket, p_r of p
//   loss = tau^2 (sum_k q_k (log q_k - log p_k) + q_r (log q_r - log p_r))
//   grad_j = g tau (p_j (Q + q_r) - q_j)  in S,   g tau p_j (Q + q_r - q_r / p_r)  outside (0 where p_r is 0),   Q = sum q
//
// A row is read once, stays in registers for its maximum, its sum and its gradient, and is written once: 2 * V values a row
// is all the HBM traffic there is, which bounds the kernel.  Rows of up to 64 classes: a few lanes a row, each with its
// values in registers; up to 128 pieces of 16 bytes with few entries: sixteen lanes a row; up to 1024 pieces: a wave a row;
// longer: a workgroup a row.  Rows longer than the registers of a workgroup are cut into segments with a launch for the sums
// before the one that writes.
//
// The outside bucket keeps a maximum and a sum of its own (mo, so), so that p_r and its logarithm hold where the top classes
// have everything.  Per-row sums are joined in float64 and logarithms taken of mantissa and exponent apart: the loss is a
// difference of logarithms that are far larger than itself.
#include <math.h>

#include "ssdbox_internal.h"

namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr double kLog2eD = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

struct DistArgs {
    const void *logits;
    long long ld;
    int rows, classes;
    int row0, row_count;              // the launch's rows
    const float *values;
    const void *index;
    int index_bytes, top;
    const float *teacher_lse;
    float tau;
    const float *grad_loss;
    float *loss;
    void *grad;
    int segments, seg_pieces;         // cut rows: segments of a row, 16-byte pieces of a segment
    struct DistPart *part;            // [row][segment]
};

struct DistPart {
    float m, mo;
    double s, so;
    int outside, pad;
};

// Sixteen bytes of a row, which starts at any value's boundary.
template <typename T>
struct Piece {
    static constexpr int N = 16 / (int)sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
    union { unsigned w[4]; T v[N]; };
    SSD_DEV void load(const T *p, int left)       // left: values there are from p on; what is missing is -inf
    {
        if (left >= N) {
            const Raw r = *(const Raw *)p;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = r.w[i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < left ? p[i] : (T)-INFINITY;
        }
    }
    SSD_DEV void store(T *p, int left) const
    {
        if (left >= N) {
            Raw r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r.w[i] = w[i];
            *(Raw *)p = r;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) p[i] = v[i];
        }
    }
};

// The logarithm of a positive float64 of ordinary size, to about 1e-11 of max(1, |ln x|): x = 2^e m with m in [0.707, 1.414],
// ln m = 2 artanh((m - 1) / (m + 1)) by its series.  (The library's would hold its many constants in registers over the rows.)
SSD_DEV double ln_of(double x)
{
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    if (!(x >= 0x1p-1000 && x <= 0x1p1000)) return x == 0.0 ? -INFINITY : (x > 0.0 ? INFINITY : x - x + NAN);
    int e = (int)(u >> 52) - 1023;
    double m = __builtin_bit_cast(double, (u & 0x000FFFFFFFFFFFFFull) | 0x3FF0000000000000ull);
    if (m > 1.41421356) {
        m *= 0.5;
        e += 1;
    }
    const double z = (m - 1.0) / (m + 1.0), w = z * z;
    double c = 1.0 / 13.0;
    c = __builtin_fma(c, w, 1.0 / 11.0);
    c = __builtin_fma(c, w, 1.0 / 9.0);
    c = __builtin_fma(c, w, 1.0 / 7.0);
    c = __builtin_fma(c, w, 0.2);
    c = __builtin_fma(c, w, 1.0 / 3.0);
    c = __builtin_fma(c, w, 1.0);
    return __builtin_fma((double)e, kLn2, 2.0 * z * c);
}

struct Entry {
    int at;                           // class, or -1: not an entry
    float t;
};

SSD_DEV Entry entry_of(const DistArgs &p, long long row, int k)
{
    const long long i = row * p.top + k;
    const long long c = p.index_bytes == 8 ? ((const long long *)p.index)[i] : (long long)((const int *)p.index)[i];
    Entry e = {-1, p.values[i]};
    if (c >= 0 && c < p.classes && e.t != -INFINITY) e.at = (int)c;
    return e;
}

// ---- reductions.  Within a wave by DPP: rows of 16 shift by 1, 2, 4, 8, two broadcasts join the rows, lane 63 has it all.
template <int CTRL, int ROWS>
SSD_DEV float dpp(float x, float none)
{
    return u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(none), (int)f2u(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
SSD_DEV double dpp(double x)
{
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, ROWS, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
SSD_DEV float wave_max(float x)
{
    const float none = -INFINITY;
    x = fmaxf(x, dpp<0x111, 0xf>(x, none));
    x = fmaxf(x, dpp<0x112, 0xf>(x, none));
    x = fmaxf(x, dpp<0x114, 0xf>(x, none));
    x = fmaxf(x, dpp<0x118, 0xf>(x, none));
    x = fmaxf(x, dpp<0x142, 0xa>(x, none));
    x = fmaxf(x, dpp<0x143, 0xc>(x, none));
    return u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(x), 63));
}
SSD_DEV double wave_sum(double x)
{
    x += dpp<0x111, 0xf>(x);
    x += dpp<0x112, 0xf>(x);
    x += dpp<0x114, 0xf>(x);
    x += dpp<0x118, 0xf>(x);
    x += dpp<0x142, 0xa>(x);
    x += dpp<0x143, 0xc>(x);
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)u, 63);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(u >> 32), 63);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// Within sixteen lanes, by rotations: all of them get the same bits, as both sides of every addition are the same two.
SSD_DEV float row_max(float x)
{
    x = fmaxf(x, dpp<0x128, 0xf>(x, x));
    x = fmaxf(x, dpp<0x124, 0xf>(x, x));
    x = fmaxf(x, dpp<0x122, 0xf>(x, x));
    return fmaxf(x, dpp<0x121, 0xf>(x, x));
}
SSD_DEV double row_sum(double x)
{
    x += dpp<0x128, 0xf>(x);
    x += dpp<0x124, 0xf>(x);
    x += dpp<0x122, 0xf>(x);
    return x + dpp<0x121, 0xf>(x);
}

// The waves' values, one in each lane of every eight (or four), joined in all of them.
template <int WAVES>
SSD_DEV float waves_max(float x)
{
    x = fmaxf(x, dpp<0xB1, 0xf>(x, x));
    x = fmaxf(x, dpp<0x4E, 0xf>(x, x));
    if constexpr (WAVES == 8) x = fmaxf(x, dpp<0x141, 0xf>(x, x));
    return u2f((uint32_t)__builtin_amdgcn_readfirstlane((int)f2u(x)));
}
template <int WAVES>
SSD_DEV double waves_sum(double x)
{
    x += dpp<0xB1, 0xf>(x);
    x += dpp<0x4E, 0xf>(x);
    if constexpr (WAVES == 8) x += dpp<0x141, 0xf>(x);
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)u);
    const unsigned hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(u >> 32));
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// THREADS lanes (sixteen, or whole waves) that work on one row.  Each reduction of a row has a place of its own in LDS, so that one
// barrier each is enough.
template <int THREADS>
struct Team {
    static constexpr int kWaves = THREADS < 64 ? 1 : THREADS / 64;    // 1, 4 or 8
    static constexpr int kPlace = kWaves * 4;      // float64 of one reduction
    double *lds;

    static SSD_DEV void sync()
    {
        if constexpr (THREADS > 64) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");    // one wave's LDS accesses run in order
    }
    template <int N>
    SSD_DEV void maxima(int place, float (&x)[N]) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = THREADS == 16 ? row_max(x[i]) : wave_max(x[i]);
        if constexpr (THREADS > 64) {
            float *p = (float *)(lds + place * kPlace);
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) p[(threadIdx.x >> 6) * N + i] = x[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = waves_max<kWaves>(p[(threadIdx.x & (kWaves - 1)) * N + i]);
        }
    }
    template <int N>
    SSD_DEV void sums(int place, double (&x)[N]) const
    {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = THREADS == 16 ? row_sum(x[i]) : wave_sum(x[i]);
        if constexpr (THREADS > 64) {
            double *p = lds + place * kPlace;
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < N; ++i) p[(threadIdx.x >> 6) * N + i] = x[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = waves_sum<kWaves>(p[(threadIdx.x & (kWaves - 1)) * N + i]);
        }
    }
};

// What a row's statistics make of an entry and of the classes outside.  All exponentials of a row are 2^((z - sub) l2 - off)
// with the same float32 l2, and its logarithms take that l2 too: what l2 and off lack in their last place then cancels,
// however far from 0 the logits lie.
struct RowTerms {
    float sub, off, l2;
    double ln_s, inv_s;
    double t_top, ln_t;               // log q = (t - t_top) / tau - ln_t
    double inv_tau;
    double whole;                     // Q + q_r
    float osub;
    double out;                       // outside: grad = 2^((z - osub) l2 - off) out
    float c;                          // g tau

    SSD_DEV double log_q(float t) const { return ((double)t - t_top) * inv_tau - ln_t; }
    SSD_DEV double log_p(float z) const { return (((double)z - (double)sub) * (double)l2 - (double)off) * kLn2 - ln_s; }
    // (in float32, as p is, and as good as the gradient that it goes into; the loss's sums and logarithms are in 64 bits)
    SSD_DEV float q(float t) const { return __builtin_amdgcn_exp2f((float)(log_q(t) * kLog2eD)); }
    SSD_DEV float power(float z) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(z - sub, l2, -off)); }
    SSD_DEV float share(float z) const { return (float)((double)power(z) * inv_s); }
};

// Whether the k-th entry is its class's first.  dup: some class is given twice in this row.
SSD_DEV bool first_of(const DistArgs &p, long long row, int k, const Entry &e, bool dup)
{
    if (dup)
        for (int j = 0; j < k; ++j)
            if (entry_of(p, row, j).at == e.at) return false;
    return true;
}

// The k-th entry's terms: (q, loss, p where it is the class's first).
SSD_DEV void add_entry(double (&sum)[3], const RowTerms &r, const DistArgs &p, long long row, int k, const Entry &e, float z,
                       bool dup)
{
    const float q = r.q(e.t);
    sum[0] += (double)q;
    if (q != 0.0f) sum[1] += (double)q * (r.log_q(e.t) - r.log_p(z));
    if (p.teacher_lse && first_of(p, row, k, e, dup)) sum[2] += (double)r.share(z);
}

// What the teacher gives a class: of all its entries, in their order.
SSD_DEV double teacher_of(const RowTerms &r, const DistArgs &p, long long row, const Entry &e, bool dup)
{
    if (!dup) return (double)r.q(e.t);
    double q = 0.0;
    for (int j = 0; j < p.top; ++j) {
        const Entry o = entry_of(p, row, j);
        if (o.at == e.at) q += (double)r.q(o.t);
    }
    return q;
}

SSD_DEV void terms_teacher(RowTerms &r, const DistArgs &p, long long row, float t_top, double sum_t)
{
    r.inv_tau = 1.0 / (double)p.tau;
    if (p.teacher_lse) {
        r.t_top = 0.0;
        r.ln_t = (double)p.teacher_lse[row];
    } else {
        r.t_top = (double)t_top;
        r.ln_t = ln_of(sum_t);
    }
}

// The row's loss from the sums over its entries (sum_p: of p over the classes they name), and the outside's factor.
// so: of the classes outside, relative to osub.
SSD_DEV double terms_finish(RowTerms &r, const DistArgs &p, long long row, double sum_q, double sum_loss, double sum_p,
                            float osub, double so, bool outside)
{
    r.osub = r.sub;
    const double g = p.grad_loss ? (double)p.grad_loss[row] : 1.0 / (double)p.rows;
    const double c = g * (double)p.tau;
    r.c = (float)c;
    r.whole = sum_q;
    double loss = sum_loss, out = r.whole * r.inv_s;
    if (p.teacher_lse && outside) {
        double q_r = 1.0 - sum_q;
        if (q_r < 0.0) q_r = 0.0;
        // near 1 a bucket is what the entries leave of it, to their own relative error
        const double ln_pr = sum_p < 0.5 ? ln_of(1.0 - sum_p)
                                         : ((double)osub - (double)r.sub) * (double)r.l2 * kLn2 + ln_of(so) - r.ln_s;
        // Where the student has nothing of the bucket that float32 holds (masked classes), a rest that is no more than the
        // rounding of a float32 log-sum-exp is nothing too: times ln p_r, it would be all of the loss.  A larger one counts as
        // defined: +inf where every class outside is -inf, whose shares of the bucket are then none.
        if (!(ln_pr < -104.0 && q_r <= 0x1p-20 * (1.0 + fabs(r.ln_t)))) {
            r.whole = sum_q + q_r;
            if (q_r > 0.0) loss += q_r * (ln_of(q_r) - ln_pr);
            out = 0.0;
            if (so != 0.0) {
                r.osub = osub;
                const double down = (double)__builtin_amdgcn_exp2f((osub - r.sub) * r.l2);
                out = r.whole * r.inv_s * down - q_r / so;
            }
        }
    }
    r.out = out * c;
    return loss * (double)p.tau * (double)p.tau;
}

// ------------------------------------------------------------------- a team of lanes a row
// TEAM lanes a row: R pieces of 16 bytes a lane, TEAM apart, and of what is left beyond the last whole piece a value a lane.
// Each team takes rows a grid apart and asks for the next row's pieces as the gradient of this one leaves their registers (the
// longest rows fill the registers: one row a workgroup).
//
// Any reference near the row's maximum serves its exponentials: float32 holds 2^126 both ways.  The largest of the
// teacher's classes' logits is at hand before the row has arrived, so the row's maximum is taken, from memory again, only where
// the sum says that the reference was far off (or a mask's lowest value overflowed the product).
//
// HBM bounds it: 8192 x 131072 bfloat16 with the rest bucket 931 us, 4.6 TB/s read and written; 3001 x 100003 float32 500 us, 4.8;
// 2048 x 32000 the value alone 31 us, 4.3; one row of 32000 8 us, latency.  (A large copy: 4.96.)
//
// The registers are only ever loaded and read: a piece that holds one of the teacher's classes is summed without them where
// they are not part of the outside bucket, and their gradients are written after the others'.
constexpr int kRegMost = 50;          // pieces a lane that the registers of a workgroup of 512 hold

template <typename T, int TEAM, int R>
struct RowPieces {
    static constexpr int N = 16 / (int)sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Raw { unsigned w[4]; };
    struct X { unsigned w[4]; };
    X x[R];
    float rest;
    int whole, more, t;               // whole pieces, values beyond them, this lane

    // limit: pieces to be read; the lanes beyond read the first piece (a load without a branch leaves the registers in place)
    SSD_DEV void load(int r, const T *z, int limit)
    {
        const int i = r * TEAM + t;
        const Raw q = *(const Raw *)((const char *)z + (unsigned)(i < limit ? i : 0) * 16u);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[r].w[j] = q.w[j];
    }
    SSD_DEV void load_rest(const T *z) { rest = t < more ? (float)z[whole * N + t] : -INFINITY; }
    SSD_DEV float value(int r, int i) const { return value(x[r].w, i); }
    static SSD_DEV float value(const unsigned (&of)[4], int i)
    {
        if constexpr (sizeof(T) == 4) return u2f(of[i]);
        const unsigned w = of[i >> 1];
        if constexpr (__is_same(T, bf16_t)) return u2f(i & 1 ? w & 0xFFFF0000u : w << 16);
        return (float)__builtin_bit_cast(f16_t, (unsigned short)(i & 1 ? w >> 16 : w & 0xFFFFu));
    }
    // Before each use of a piece: keeps the compiler from holding the float32 values of one pass for the next (twice the
    // registers of 16-bit rows) and from working on many pieces at once.
    SSD_DEV void forget(int r)
    {
        asm volatile("" : "+v"(x[r].w[0]), "+v"(x[r].w[1]), "+v"(x[r].w[2]), "+v"(x[r].w[3]), "+v"(t));
        __builtin_amdgcn_sched_barrier(0);
    }
};

// Entries of a lane in registers: 64 entries of sixteen lanes, 256 of the larger teams.
template <int TEAM>
constexpr int kEntries = TEAM <= 64 ? 4 : 1;

template <typename T, int TEAM, int R>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void distill_row_kernel(const DistArgs p)
{
    typedef RowPieces<T, TEAM, R> V;
    constexpr int N = V::N;
    constexpr int kBlockThreads = TEAM < 256 ? 256 : TEAM;
    constexpr int kRows = kBlockThreads / TEAM;
    constexpr bool kBeyond = R == kRegMost;               // rows longer than the registers as well
    constexpr int kWords = (TEAM * R * (kBeyond ? 2 : 1) + 1) * N / 32 + 1;
    __shared__ unsigned s_bits[kRows * kWords];
    __shared__ double s_red[4 * Team<TEAM>::kPlace];
    const int t = threadIdx.x % TEAM;
    const int mine = TEAM == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / TEAM) : TEAM < 64 ? threadIdx.x / TEAM : 0;
    long long row = p.row0 + (long long)blockIdx.x * kRows + mine;
    const long long end = p.row0 + p.row_count, step = (long long)gridDim.x * kRows;
    if (row >= end) return;                               // whole teams, of which only those of several waves have barriers
    unsigned *bits = s_bits + mine * kWords;
    const Team<TEAM> team = {s_red};
    const bool tail = p.teacher_lse != nullptr;
    constexpr bool kLoop = TEAM == 512 && R == 32;
    V v;
    v.t = t;
    v.whole = p.classes / N;
    v.more = p.classes - v.whole * N;
    const T *z = (const T *)p.logits + row * p.ld;

    // a lane's first entries stay in registers; further ones are read again each time
    constexpr int E = kEntries<TEAM>;
    Entry e0[E];
    const auto take = [&](Entry (&e)[E], long long of, bool any) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
            e[j] = Entry{-1, -INFINITY};
            if (any && t + j * TEAM < p.top) e[j] = entry_of(p, of, t + j * TEAM);
        }
    };
    take(e0, row, true);
#pragma unroll
    for (int r = 0; r < R; ++r) v.load(r, z, v.whole);
    v.load_rest(z);
    for (int i = t; i < kWords; i += TEAM) bits[i] = 0u;
    Team<TEAM>::sync();
    RowTerms f;
    f.l2 = (float)(kLog2eD / (double)p.tau);

    for (;;) {
        float z0[E];
#pragma unroll
        for (int j = 0; j < E; ++j) z0[j] = e0[j].at >= 0 ? (float)z[e0[j].at] : -INFINITY;
        // f(place among the registers' or E, k, entry, its logit) for each of the lane's entries
        const auto entries_of = [&](auto f) {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (e0[j].at >= 0) f(j, t + j * TEAM, e0[j], z0[j]);
            for (int k = t + E * TEAM; k < p.top; k += TEAM) {
                const Entry e = entry_of(p, row, k);
                if (e.at >= 0) f(E, k, e, (float)z[e.at]);
            }
        };
        float top[2] = {-INFINITY, -INFINITY};             // of the entries' logits, of the teacher's
        int entries = 0, inside = 0;
        unsigned first0 = 0u;
        entries_of([&](int j, int, const Entry &e, float ze) {
            top[0] = fmaxf(top[0], ze);
            top[1] = fmaxf(top[1], e.t);
            const unsigned bit = 1u << (e.at & 31);
            ++entries;
            if (!(atomicOr(&bits[e.at >> 5], bit) & bit)) {
                ++inside;
                first0 |= 1u << j;
            }
        });
        team.template maxima<2>(0, top);                   // its barrier shows the bits as well
        if constexpr (TEAM <= 64) Team<TEAM>::sync();
        f.sub = 0.0f;
        f.off = top[0] == -INFINITY ? 0.0f : fmaxf(top[0] * f.l2, -3e38f);
        const float off = f.off;
        float osub = 0.0f, so = 0.0f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            v.forget(r);
            const int i = r * TEAM + v.t;
            if (i < v.whole) {
                const unsigned in = tail ? bits[i * N >> 5] >> (i * N & 31) & ((1u << N) - 1u) : 0u;
                float e[N];
#pragma unroll
                for (int j = 0; j < N; ++j) e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(v.value(r, j), f.l2, -off));
                if (in)
#pragma unroll
                    for (int j = 0; j < N; ++j) e[j] = in >> j & 1u ? 0.0f : e[j];
#pragma unroll
                for (int j = 0; j < N; ++j) so += e[j];
            }
        }
        float beyond = 0.0f;
        if constexpr (kBeyond)
#pragma unroll 2
            for (int i = TEAM * R + t; i < v.whole; i += TEAM) {
                const typename V::Raw q = *(const typename V::Raw *)((const char *)z + (unsigned)i * 16u);
                const unsigned in = tail ? bits[i * N >> 5] >> (i * N & 31) & ((1u << N) - 1u) : 0u;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(V::value(q.w, j), f.l2, -off));
                    beyond += in >> j & 1u ? 0.0f : e;
                }
            }
        const int last = v.whole * N + t;
        if (t < v.more && !(tail && (bits[last >> 5] >> (last & 31) & 1u)))
            so += __builtin_amdgcn_exp2f(__builtin_fmaf(v.rest, f.l2, -off));
        double sum[4] = {(double)so + (double)beyond, 0.0, (double)inside + 65536.0 * (double)entries, 0.0};
        if (tail) {
#pragma unroll
            for (int j = 0; j < E; ++j)
                if (first0 >> j & 1u) sum[3] += (double)f.power(z0[j]);
        } else {
            entries_of([&](int, int, const Entry &e, float) {
                sum[1] += (double)__builtin_amdgcn_exp2f((e.t - top[1]) * f.l2);
            });
        }
        team.template sums<4>(1, sum);
        const int n_entries = (int)(sum[2] / 65536.0), n_inside = (int)(sum[2] - 65536.0 * n_entries);
        const bool dup = n_entries > n_inside, outside = n_inside < p.classes;
        // (a bucket without a class needs no reference: its sum of 0 is right)
        const bool slow = n_inside == 0 || (!(sum[0] > 0x1p-60 && sum[0] < 0x1p120) && (!tail || outside));
        if (slow && n_inside > 0) {
            float most[1] = {-INFINITY};
            for (int i = t; i < p.classes; i += TEAM)
                if (!tail || !(bits[i >> 5] >> (i & 31) & 1u)) most[0] = fmaxf(most[0], (float)z[i]);
            team.template maxima<1>(3, most);
            f.off = 0.0f;
            f.sub = tail ? fmaxf(most[0], top[0]) : most[0];
            if (f.sub == -INFINITY) f.sub = 0.0f;
            osub = most[0] == -INFINITY ? 0.0f : most[0];
            double again[1] = {0.0};
            for (int i = t; i < p.classes; i += TEAM)
                if (!tail || !(bits[i >> 5] >> (i & 31) & 1u))
                    again[0] += (double)__builtin_amdgcn_exp2f(((float)z[i] - osub) * f.l2);
            if constexpr (TEAM > 64) __syncthreads();      // place 3's maxima have been read
            team.template sums<1>(3, again);
            sum[0] = again[0];
        }
        if constexpr (kLoop) entries_of([&](int, int, const Entry &e, float) { bits[e.at >> 5] = 0u; });    // for the next row
        const long long next = row + step;
        const bool goes_on = kLoop && next < end;
        const T *zn = goes_on ? z + step * p.ld : z;
        const int limit = goes_on ? v.whole : 0;
        Entry en[E];
        take(en, next, goes_on);

        double s = sum[0];
        if (tail) {
            double in[1] = {sum[3]};
            if (slow || dup || p.top > E * TEAM) {
                in[0] = 0.0;
                entries_of([&](int, int k, const Entry &e, float ze) {
                    if (first_of(p, row, k, e, dup)) in[0] += (double)f.power(ze);
                });
                team.template sums<1>(0, in);
            }
            s = in[0] + s * (double)__builtin_amdgcn_exp2f((osub - f.sub) * f.l2);
        }
        f.inv_s = 1.0 / s;
        f.ln_s = ln_of(s);
        terms_teacher(f, p, row, top[1], sum[1]);
        double of_entries[3] = {0.0, 0.0, 0.0};
        entries_of([&](int, int k, const Entry &e, float ze) { add_entry(of_entries, f, p, row, k, e, ze, dup); });
        team.template sums<3>(2, of_entries);
        const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2], osub, sum[0], outside);
        if (t == 0) p.loss[row] = n_inside > 0 ? (float)loss : 0.0f;      // a row without an entry teaches nothing
        T *g = (T *)p.grad + row * p.classes;
        // Against a reference that the row's largest exponential exceeds by up to 2^120, out is as small, and what g tau takes off it
        // too may leave float32's range: such a row is read again, and the exponent of out is a factor of its own.
        const float out = (float)f.out;
        const bool in_range = (fabsf(out) >= 0x1p-100f && fabsf(out) <= 0x1p100f) || f.c == 0.0f;
        if (p.grad && !slow && in_range) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                v.forget(r);
                const int i = r * TEAM + v.t;
                if (i < v.whole) {
                    Piece<T> o;
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        o.v[j] = (T)(__builtin_amdgcn_exp2f(__builtin_fmaf(v.value(r, j), f.l2, -off)) * out);
                    o.store((T *)((char *)g + (unsigned)i * 16u), N);
                }
                if constexpr (kLoop) v.load(r, zn, limit);
            }
            if constexpr (kBeyond)
#pragma unroll 2
                for (int i = TEAM * R + t; i < v.whole; i += TEAM) {
                    const typename V::Raw q = *(const typename V::Raw *)((const char *)z + (unsigned)i * 16u);
                    Piece<T> o;
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        o.v[j] = (T)(__builtin_amdgcn_exp2f(__builtin_fmaf(V::value(q.w, j), f.l2, -off)) * out);
                    o.store((T *)((char *)g + (unsigned)i * 16u), N);
                }
            if (t < v.more)
                g[v.whole * N + t] = (T)(__builtin_amdgcn_exp2f(__builtin_fmaf(v.rest, f.l2, -off)) * out);
        } else {
            if (p.grad) {
                const float from = slow ? f.osub : 0.0f;   // (off is 0 of a row that took its own maximum)
                int e = (int)(__builtin_bit_cast(unsigned long long, f.out) >> 52 & 0x7FF) - 1023;
                e = e < -252 ? -252 : (e > 252 ? 252 : e);
                const float half = u2f((uint32_t)(127 + e / 2) << 23);
                const float rest = (float)(f.out * __builtin_bit_cast(double, (unsigned long long)(1023 - e / 2) << 52));
                for (int i = t; i < p.classes; i += TEAM) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf((float)z[i] - from, f.l2, -f.off));
                    g[i] = (T)(n_inside > 0 ? x * half * rest : 0.0f);
                }
            }
            if constexpr (kLoop)
#pragma unroll
                for (int r = 0; r < R; ++r) v.load(r, zn, limit);
        }
        if constexpr (kLoop) v.load_rest(zn);
        if (p.grad) {
            Team<TEAM>::sync();                            // the entries' own values come last
            entries_of([&](int, int, const Entry &e, float ze) {
                const double q = teacher_of(f, p, row, e, dup);
                g[e.at] = (T)(float)((double)f.c * ((double)f.share(ze) * f.whole - q));
            });
        }
        if (!goes_on) return;
        row = next;
        z = zn;
#pragma unroll
        for (int j = 0; j < E; ++j) e0[j] = en[j];
    }
}

// ----------------------------------------------------------------------- few classes a row
// G lanes a row, up to 4 classes and every G-th entry a lane.  Latency of the entries' chain of loads (408000 x 2 x 2 float32: 11 us, 1.6 TB/s).
// Joins by DPP: a lane's neighbour, the quad's other half, then the mirrored lane of eight and of sixteen, where the halves are
// the same in all their lanes already.  Both sides of every join are the same two values: all lanes get the same bits.
template <int CTRL>
SSD_DEV float across(float x)
{
    return dpp<CTRL, 0xf>(x, x);
}
template <int CTRL>
SSD_DEV double across(double x)
{
    return dpp<CTRL, 0xf>(x);
}
template <int CTRL>
SSD_DEV int across(int x)
{
    return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, false);
}
template <int G, typename X, typename F>
SSD_DEV X group(X x, F f)
{
    if constexpr (G >= 2) x = f(x, across<0xB1>(x));
    if constexpr (G >= 4) x = f(x, across<0x4E>(x));
    if constexpr (G >= 8) x = f(x, across<0x141>(x));
    if constexpr (G >= 16) x = f(x, across<0x140>(x));
    return x;
}

template <typename T, int G>
__global__ __launch_bounds__(256) void distill_small_kernel(const DistArgs p)
{
    const int l = threadIdx.x % G;
    const long long row = p.row0 + ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (row >= p.rows) return;                             // whole teams
    const auto more = [](float a, float b) { return fmaxf(a, b); };
    const auto plus = [](double a, double b) { return a + b; };
    const T *z = (const T *)p.logits + row * p.ld;
    float x[4];
    float m = -INFINITY, mo = -INFINITY, t_top = -INFINITY;
    unsigned in = 0u;
    int entries = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = l + G * i;
        x[i] = j < p.classes ? (float)z[j] : -INFINITY;
        m = fmaxf(m, x[i]);
    }
    // Entries are dealt to the lanes, G at a time; what a class's own lane has to know of them comes by shuffles.
    const int lane0 = (threadIdx.x & 63) - l;
    const auto entry = [&](int k) { return k < p.top ? entry_of(p, row, k) : Entry{-1, -INFINITY}; };
    for (int k0 = 0; k0 < p.top; k0 += G) {
        const Entry e = entry(k0 + l);
        if (e.at >= 0) {
            ++entries;
            t_top = fmaxf(t_top, e.t);
        }
        for (int j = 0; j < G && k0 + j < p.top; ++j) {
            const int at = __shfl(e.at, lane0 + j);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at == l + G * i) in |= 1u << i;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(in >> i & 1u)) mo = fmaxf(mo, x[i]);
    m = group<G>(m, more);
    mo = group<G>(mo, more);
    t_top = group<G>(t_top, more);
    entries = group<G>(entries | (int)__popc(in) << 16, [](int a, int b) { return a + b; });
    const int inside = entries >> 16;
    entries &= 0xFFFF;
    RowTerms f;
    f.l2 = (float)(kLog2eD / (double)p.tau);
    const float mref = m == -INFINITY ? 0.0f : m, oref = mo == -INFINITY ? 0.0f : mo;
    double sum[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum[0] += (double)__builtin_amdgcn_exp2f((x[i] - mref) * f.l2);
        if (!(in >> i & 1u)) sum[1] += (double)__builtin_amdgcn_exp2f((x[i] - oref) * f.l2);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) sum[i] = group<G>(sum[i], plus);
    T *g = (T *)p.grad + row * p.classes;
    if (entries == 0) {
        if (l == 0) p.loss[row] = 0.0f;
        if (p.grad)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (l + G * i < p.classes) g[l + G * i] = (T)0.0f;
        return;
    }
    double st = 0.0;
    if (!p.teacher_lse) {
        for (int k0 = 0; k0 < p.top; k0 += G) {
            const Entry e = entry(k0 + l);
            if (e.at >= 0) st += (double)__builtin_amdgcn_exp2f((e.t - t_top) * f.l2);
        }
        st = group<G>(st, plus);
    }
    f.sub = mref;
    f.off = 0.0f;
    f.inv_s = 1.0 / sum[0];
    f.ln_s = ln_of(sum[0]);
    terms_teacher(f, p, row, t_top, st);
    double of_entries[3] = {0.0, 0.0, 0.0}, q_at[4] = {0.0, 0.0, 0.0, 0.0};
    const bool dup = entries > inside;
    for (int k0 = 0; k0 < p.top; k0 += G) {
        const Entry e = entry(k0 + l);
        float q = 0.0f;
        if (e.at >= 0) {
            add_entry(of_entries, f, p, row, k0 + l, e, (float)z[e.at], dup);
            q = f.q(e.t);
        }
        if (p.grad)
            for (int j = 0; j < G && k0 + j < p.top; ++j) {
                const int at = __shfl(e.at, lane0 + j);
                const float of = __shfl(q, lane0 + j);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at == l + G * i) q_at[i] += (double)of;
            }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) of_entries[i] = group<G>(of_entries[i], plus);
    const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2], oref, sum[1],
                                     inside < p.classes);
    if (l == 0) p.loss[row] = (float)loss;
    if (!p.grad) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = l + G * i;
        if (j >= p.classes) continue;
        const float o = (in >> i & 1u) ? (float)((double)f.c * ((double)f.share(x[i]) * f.whole - q_at[i]))
                                       : __builtin_amdgcn_exp2f((x[i] - f.osub) * f.l2) * (float)f.out;
        g[j] = (T)o;
    }
}

// --------------------------------------------------------------------------- cut rows
constexpr int kSegThreads = 256;
constexpr int kSegMost = 1024;        // pieces of 16 bytes a segment

SSD_DEV void join_part(DistPart &a, const DistPart &b, float l2)
{
    const float m = fmaxf(a.m, b.m), mo = fmaxf(a.mo, b.mo);
    if (m != -INFINITY)
        a.s = a.s * (double)__builtin_amdgcn_exp2f((a.m - m) * l2) + b.s * (double)__builtin_amdgcn_exp2f((b.m - m) * l2);
    else
        a.s += b.s;
    if (mo != -INFINITY)
        a.so = a.so * (double)__builtin_amdgcn_exp2f((a.mo - mo) * l2) +
               b.so * (double)__builtin_amdgcn_exp2f((b.mo - mo) * l2);
    else
        a.so += b.so;
    a.m = m;
    a.mo = mo;
    a.outside += b.outside;
}

// The sums of cut rows.  grid: segments of a row back to back.  HBM (2832 x 117899 float32: 236 us, 5.7 TB/s)
template <typename T>
__global__ __launch_bounds__(kSegThreads) void distill_part_kernel(const DistArgs p)
{
    typedef Piece<T> P;
    constexpr int R = kSegMost / kSegThreads;
    __shared__ unsigned s_bits[kSegMost * P::N / 32];
    __shared__ double s_red[3 * Team<kSegThreads>::kPlace];
    const int t = threadIdx.x, seg = blockIdx.x % p.segments;
    const long long row = p.row0 + blockIdx.x / p.segments;
    const int first = seg * p.seg_pieces * P::N;
    const int here = p.classes - first < p.seg_pieces * P::N ? p.classes - first : p.seg_pieces * P::N;
    const Team<kSegThreads> team = {s_red};
    const T *z = (const T *)p.logits + row * p.ld + first;
    P x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * kSegThreads + t) * P::N;
        x[r].load(z + at, here - at);
    }
    const bool tail = p.teacher_lse != nullptr;
    int inside = 0;
    for (int i = t; i < (here + 31) / 32; i += kSegThreads) s_bits[i] = 0u;
    __syncthreads();
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        const int at = e.at - first;
        if (e.at < 0 || at < 0 || at >= here) continue;
        const unsigned bit = 1u << (at & 31);
        if (!(atomicOr(&s_bits[at >> 5], bit) & bit)) ++inside;
    }
    __syncthreads();
    float m = -INFINITY, mo = -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * kSegThreads + t) * P::N;
        const unsigned in = tail && at < here ? s_bits[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
            const float v = (float)x[r].v[i];
            m = fmaxf(m, v);
            if (tail && !(in >> i & 1u)) mo = fmaxf(mo, v);
        }
    }
    float top[2] = {m, mo};
    team.template maxima<2>(0, top);
    m = top[0];
    mo = top[1];
    const float l2 = (float)(kLog2eD / (double)p.tau);
    const float mref = m == -INFINITY ? 0.0f : m, oref = mo == -INFINITY ? 0.0f : mo;
    float s = 0.0f, so = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * kSegThreads + t) * P::N;
        const unsigned in = tail && at < here ? s_bits[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
            const float v = (float)x[r].v[i];
            s += __builtin_amdgcn_exp2f((v - mref) * l2);
            if (tail && !(in >> i & 1u)) so += __builtin_amdgcn_exp2f((v - oref) * l2);
        }
    }
    double sum[3] = {(double)s, (double)so, (double)inside};
    team.template sums<3>(1, sum);
    if (t == 0) p.part[row * p.segments + seg] = DistPart{m, mo, sum[0], sum[1], here - (int)sum[2], 0};
}

// grid: with a gradient as above, else one workgroup a row; each joins the row's parts in the same order
template <typename T>
__global__ __launch_bounds__(kSegThreads) void distill_segment_kernel(const DistArgs p)
{
    typedef Piece<T> P;
    constexpr int R = kSegMost / kSegThreads;
    __shared__ double s_red[3 * Team<kSegThreads>::kPlace];
    __shared__ DistPart s_part[kSegThreads];
    const int each = p.grad ? p.segments : 1;
    const int t = threadIdx.x, seg = blockIdx.x % each;
    const long long row = p.row0 + blockIdx.x / each;
    const int first = seg * p.seg_pieces * P::N;
    const int here = p.classes - first < p.seg_pieces * P::N ? p.classes - first : p.seg_pieces * P::N;
    const Team<kSegThreads> team = {s_red};
    const T *zr = (const T *)p.logits + row * p.ld;
    P x[R];
    if (p.grad)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int at = (r * kSegThreads + t) * P::N;
            x[r].load(zr + first + at, here - at);
        }
    RowTerms f;
    f.l2 = (float)(kLog2eD / (double)p.tau);
    DistPart mine = {-INFINITY, -INFINITY, 0.0, 0.0, 0, 0};
    for (int i = t; i < p.segments; i += kSegThreads) join_part(mine, p.part[row * p.segments + i], f.l2);
    s_part[t] = mine;
    __syncthreads();
    for (int o = kSegThreads / 2; o > 0; o >>= 1) {
        if (t < o) join_part(s_part[t], s_part[t + o], f.l2);
        __syncthreads();
    }
    const DistPart all = s_part[0];
    float t_top = -INFINITY;
    int entries = 0;
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        ++entries;
        t_top = fmaxf(t_top, e.t);
    }
    float most[1] = {t_top};
    team.template maxima<1>(0, most);
    t_top = most[0];
    double sum[2] = {(double)entries, 0.0};
    if (!p.teacher_lse)
        for (int k = t; k < p.top; k += kSegThreads) {
            const Entry e = entry_of(p, row, k);
            if (e.at >= 0) sum[1] += (double)__builtin_amdgcn_exp2f((e.t - t_top) * f.l2);
        }
    team.template sums<2>(1, sum);
    T *g = (T *)p.grad + row * p.classes + first;
    if (sum[0] == 0.0) {
        if (t == 0 && seg == 0) p.loss[row] = 0.0f;
        if (p.grad) {
            P zero;
#pragma unroll
            for (int i = 0; i < P::N; ++i) zero.v[i] = (T)0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int at = (r * kSegThreads + t) * P::N;
                zero.store(g + at, here - at);
            }
        }
        return;
    }
    f.sub = all.m == -INFINITY ? 0.0f : all.m;
    f.off = 0.0f;
    f.inv_s = 1.0 / all.s;
    f.ln_s = ln_of(all.s);
    terms_teacher(f, p, row, t_top, sum[1]);
    const bool dup = sum[0] > (double)(p.classes - all.outside);
    double of_entries[3] = {0.0, 0.0, 0.0};
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        add_entry(of_entries, f, p, row, k, e, (float)zr[e.at], dup);
    }
    team.template sums<3>(2, of_entries);
    const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2],
                                     all.mo == -INFINITY ? 0.0f : all.mo, all.so,
                                     all.outside > 0);
    if (t == 0 && seg == 0) p.loss[row] = (float)loss;
    if (!p.grad) return;
    const float out = (float)f.out;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * kSegThreads + t) * P::N;
        P o;
#pragma unroll
        for (int i = 0; i < P::N; ++i)
            o.v[i] = (T)(__builtin_amdgcn_exp2f(((float)x[r].v[i] - f.osub) * f.l2) * out);
        o.store(g + at, here - at);
    }
    __syncthreads();
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        const int at = e.at - first;
        if (e.at < 0 || at < 0 || at >= here) continue;
        const double q = teacher_of(f, p, row, e, dup);
        g[at] = (T)(float)((double)f.c * ((double)f.share((float)zr[e.at]) * f.whole - q));
    }
}

// --------------------------------------------------------------------------------- launch
struct DistPlan {
    bool cut;
    int segments, seg_pieces;
    size_t bytes;
};

template <typename T>
DistPlan dist_plan(long long rows, long long classes)
{
    constexpr int N = 16 / (int)sizeof(T);
    const long long pieces = (classes + N - 1) / N;
    DistPlan q = {};
    // Rows longer than a workgroup's registers: what does not fit is read twice, until that is half of the row; cut rows are
    // read twice whole (once without a gradient), but by more workgroups.  Measured (rows x classes, cut, not): 2832 x 117899
    // float32 924 587 us, its value alone 236 303, 1000 x 262144 bfloat16 505 274, 4000 x 262144 its value alone 665 519,
    // 100 x 117899 float32 50 33, 64 x 204000 float32 52 55, 16 x 250000 bfloat16 25 35.
    q.cut = pieces > 512 * kRegMost * (rows < 64 ? 1 : 2);
    if (q.cut) {
        long long segs = (pieces + kSegMost - 1) / kSegMost;
        while (segs * rows < 512 && pieces / (segs * 2) >= kSegThreads) segs *= 2;
        q.seg_pieces = (int)((pieces + segs - 1) / segs + 3) / 4 * 4;    // whole words of the bit map
        if (q.seg_pieces > kSegMost) q.seg_pieces = kSegMost;
        q.segments = (int)((pieces + q.seg_pieces - 1) / q.seg_pieces);
        q.bytes = (size_t)rows * q.segments * sizeof(DistPart);
    }
    return q;
}

template <typename T, int TEAM, int R>
void launch_row(ssdbox_ctx *ctx, const DistArgs &a, int rows)
{
    constexpr int kThreads = TEAM < 256 ? 256 : TEAM;
    // rows that fill half the registers: as many workgroups as run at once, each going on to its next row with its loads in
    // flight (shorter ones do without: 1021 x 50021 float16 46 us, 62 that way)
    constexpr int kEach = TEAM == 512 ? (R <= 8 ? 2 : 1) : 4;
    const int most = R == 32 ? ctx->num_cus * kEach : rows, need = (rows + kThreads / TEAM - 1) / (kThreads / TEAM);
    const unsigned grid = (unsigned)(need < most ? need : most);
    launch_stage(ctx, SSDBOX_STAGE_LOSS, distill_row_kernel<T, TEAM, R>, dim3(grid), dim3(kThreads), a);
}

template <typename T, int G>
void launch_small(ssdbox_ctx *ctx, const DistArgs &a, int rows)
{
    const unsigned grid = (unsigned)(((long long)rows * G + 255) / 256);
    launch_stage(ctx, SSDBOX_STAGE_LOSS, distill_small_kernel<T, G>, dim3(grid), dim3(256), a);
}

template <typename T>
void launch_distill(ssdbox_ctx *ctx, const DistArgs &a, const DistPlan &q, int rows)
{
    constexpr int N = 16 / (int)sizeof(T);
    const int pieces = (a.classes + N - 1) / N;
    if (q.cut) {
        launch_stage(ctx, SSDBOX_STAGE_LOSS, distill_part_kernel<T>, dim3((unsigned)rows * q.segments), dim3(kSegThreads), a);
        launch_stage(ctx, SSDBOX_STAGE_LOSS, distill_segment_kernel<T>, dim3((unsigned)rows * (a.grad ? q.segments : 1)),
                     dim3(kSegThreads), a);
    }
    // as many lanes a row as leave each of them four classes; twice as many (rows x classes x K, us): 408000 x 4 x 2 float32
    // 14.8, 16.4;  400000 x 8 x 3 bfloat16 24, 36;  400000 x 16 x 4 float32 35, 61;  300000 x 32 x 4 bfloat16 51, 91.  Against the
    // sixteen lanes of the next kernel: 487435 x 23 x 6 float32 80, 109, its value alone 62, 103;  400000 x 20 x 2 bfloat16 55, 96;
    // from 33 classes on they would be faster up to 64 entries (400000 x 60 x 2 float32 134, 122;  100000 x 40 x 8 float16 45, 37;
    // 200000 x 60 x 30 bfloat16 151, 64), which this border leaves
    else if (a.classes <= 4) launch_small<T, 1>(ctx, a, rows);
    else if (a.classes <= 8) launch_small<T, 2>(ctx, a, rows);
    else if (a.classes <= 16) launch_small<T, 4>(ctx, a, rows);
    else if (a.classes <= 32) launch_small<T, 8>(ctx, a, rows);
    else if (a.classes <= 64) launch_small<T, 16>(ctx, a, rows);
    // short rows: sixteen lanes a row rather than a wave, as long as the registers hold the entries (rows x classes x K, us:
    // 113154 x 164 x 8 float32 39, a wave 113;  35660 x 74 x 15 float32 18, 40;  50000 x 400 x 64 float32 44, 66;
    // 20000 x 1000 x 16 bfloat16 20, 31; past the registers' entries 20000 x 500 x 200 float32 133, 37), in registers for no more
    // pieces than there are (for 128 instead: 113154 x 100 x 8 float32 34, 40;  100000 x 200 x 8 44, 50;  60000 x 400 x 16 bfloat16
    // 30, 32)
    else if (pieces <= 128 && a.top <= 16 * kEntries<16>) {
        if (pieces <= 32) launch_row<T, 16, 2>(ctx, a, rows);
        else if (pieces <= 64) launch_row<T, 16, 4>(ctx, a, rows);
        else launch_row<T, 16, 8>(ctx, a, rows);
    }
    // (479494 x 728 x 2 float32 485, a wave 620, its value alone 266, 475;  50000 x 1000 x 60 float32 111, 88)
    else if (pieces <= 256 && a.top <= 16) launch_row<T, 16, 16>(ctx, a, rows);
    // (registers for 256 pieces instead: 60000 x 120 x 100 float32 72, 77;  60000 x 400 x 70 bfloat16 76, 80)
    else if (pieces <= 64) launch_row<T, 64, 1>(ctx, a, rows);
    else if (pieces <= 128) launch_row<T, 64, 2>(ctx, a, rows);
    else if (pieces <= 256) launch_row<T, 64, 4>(ctx, a, rows);
    // (a workgroup of 256 a row instead: 143928 x 2754 x 14 bfloat16 432 us, 852;  30000 x 8000 x 32 196, 224, its value alone
    // 84, 149;  100 x 2754 x 14 18.0, 17.2;  50000 x 4000 x 14 float32 315, 300)
    // (registers for 1024 pieces instead: 20000 x 2000 x 14 float32 57, 66;  20000 x 3900 x 14 bfloat16 64, 74)
    else if (pieces <= 512) launch_row<T, 64, 8>(ctx, a, rows);
    else if (pieces <= 1024) launch_row<T, 64, 16>(ctx, a, rows);
    // (a workgroup of 512 with registers for 8192 pieces instead: 8000 x 8000 x 14 float32 96, 135;  4000 x 16000 x 14 115, 119; and
    // with registers for 25600 instead of 16384: 2000 x 50000 x 14 float32 194, 193;  2000 x 120000 x 14 bfloat16 228, 237)
    else if (pieces <= 2048) launch_row<T, 256, 8>(ctx, a, rows);
    else if (pieces <= 4096) launch_row<T, 512, 8>(ctx, a, rows);
    else if (pieces <= 8192) launch_row<T, 512, 16>(ctx, a, rows);
    else if (pieces <= 16384) launch_row<T, 512, 32>(ctx, a, rows);
    else launch_row<T, 512, kRegMost>(ctx, a, rows);
}

template <typename T>
void run_distill(ssdbox_ctx *ctx, DistArgs a, const DistPlan &q)
{
    // a launch takes fewer than 2^32 threads: 2^22 rows at most, or that many workgroups of a cut row
    const int step = q.cut ? ((1 << 22) / q.segments > 0 ? (1 << 22) / q.segments : 1) : 1 << 22;
    a.segments = q.segments;
    a.seg_pieces = q.seg_pieces;
    for (long long r = 0; r < a.rows; r += step) {
        a.row0 = (int)r;
        a.row_count = (int)(a.rows - r < step ? a.rows - r : step);
        launch_distill<T>(ctx, a, q, a.row_count);
    }
}

int check_distill(int64_t rows, int64_t classes, int top, int dtype)
{
    SSD_REQUIRE(dtype == SSDBOX_DTYPE_F32 || dtype == SSDBOX_DTYPE_F16 || dtype == SSDBOX_DTYPE_BF16,
                "distill_topk: dtype %d", dtype);
    SSD_REQUIRE(rows >= 0 && rows < (1ll << 31) - 256, "distill_topk: %lld rows", (long long)rows);
    SSD_REQUIRE(classes >= 1 && classes <= (1 << 28), "distill_topk: %lld classes outside [1, 2^28]", (long long)classes);
    SSD_REQUIRE(top >= 1 && top <= SSDBOX_MAX_TOP, "distill_topk: %d teacher's entries outside [1, %d]", top,
                SSDBOX_MAX_TOP);
    return SSDBOX_OK;
}

DistPlan dist_plan_of(int64_t rows, int64_t classes, int dtype)
{
    return dtype == SSDBOX_DTYPE_F32 ? dist_plan<float>(rows, classes) : dist_plan<bf16_t>(rows, classes);
}

}  // namespace

extern "C" int ssdbox_distill_topk_workspace(int64_t rows, int64_t classes, int dtype, size_t *bytes)
{
    SSD_REQUIRE(bytes != nullptr, "distill_topk_workspace: bytes is NULL");
    int rc = check_distill(rows, classes, 1, dtype);
    if (rc != SSDBOX_OK) return rc;
    *bytes = dist_plan_of(rows, classes, dtype).bytes;
    return SSDBOX_OK;
}

extern "C" int ssdbox_distill_topk(ssdbox_ctx *ctx, const void *d_logits, int64_t logits_ld, int64_t rows, int64_t classes,
                                   int dtype, const float *d_values, const void *d_index, int index_bytes, int top,
                                   const float *d_teacher_lse, float temperature, const float *d_grad_loss, float *d_loss,
                                   void *d_grad, void *d_workspace, size_t workspace_bytes)
{
    SSD_REQUIRE(ctx != nullptr, "distill_topk: ctx is NULL");
    int rc = check_distill(rows, classes, top, dtype);
    if (rc != SSDBOX_OK) return rc;
    SSD_REQUIRE(logits_ld >= classes, "distill_topk: row stride %lld below %lld classes", (long long)logits_ld,
                (long long)classes);
    SSD_REQUIRE(index_bytes == 4 || index_bytes == 8, "distill_topk: index of %d bytes", index_bytes);
    SSD_REQUIRE(temperature >= 1e-3f && temperature <= 1e3f, "distill_topk: temperature %g outside [0.001, 1000]",
                temperature);
    if (rows == 0) return SSDBOX_OK;
    SSD_REQUIRE(d_logits && d_values && d_index && d_loss, "distill_topk: NULL buffer");
    const DistPlan q = dist_plan_of(rows, classes, dtype);
    SSD_REQUIRE(q.bytes == 0 || (d_workspace != nullptr && workspace_bytes >= q.bytes),
                "distill_topk: workspace of %zu bytes, %zu needed", workspace_bytes, q.bytes);

    DeviceGuard guard(ctx->device);
    DistArgs a = {};
    a.logits = d_logits;
    a.ld = logits_ld;
    a.rows = (int)rows;
    a.classes = (int)classes;
    a.values = d_values;
    a.index = d_index;
    a.index_bytes = index_bytes;
    a.top = top;
    a.teacher_lse = d_teacher_lse;
    a.tau = temperature;
    a.grad_loss = d_grad_loss;
    a.loss = d_loss;
    a.grad = d_grad;
    a.part = (DistPart *)d_workspace;
    if (dtype == SSDBOX_DTYPE_F32) run_distill<float>(ctx, a, q);
    else if (dtype == SSDBOX_DTYPE_F16) run_distill<f16_t>(ctx, a, q);
    else run_distill<bf16_t>(ctx, a, q);
    SSD_CHECK_HIP(hipGetLastError());
    return SSDBOX_OK;
}
