// Distillation from a teacher's top logits, with the gradient with respect to the student's logits.
//
// u = z / tau, p = softmax(u) over all classes; the teacher gives K (class, logit) pairs a row, S their classes:
//   without its log-sum-exp: q = softmax over the K of t / tau, no rest
//   with it (at tau):        q = exp(t / tau - lse), q_r = 1 - sum q; the classes outside S are one bucket, p_r of p
//   loss = tau^2 (sum_k q_k (log q_k - log p_k) + q_r (log q_r - log p_r))
//   grad_j = g tau (p_j (Q + q_r) - q_j)  in S,   g tau p_j (Q + q_r - q_r / p_r)  outside,   Q = sum q
//
// A row is read once, stays in registers for its maximum, its sum and its gradient, and is written once: 2 * V values a row
// is all the HBM traffic there is, which bounds the kernel.  Rows of up to 64 classes: a few lanes a row, each with its
// values in registers; up to 256 pieces of 16 bytes: a wave a row; longer: a workgroup a row.  Rows longer than the
// registers of a workgroup, and too few rows for the chip, are cut into segments with a launch for the sums before the
// one that writes.
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
    int row0;                         // the launch's first row
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

// log2 of a positive finite float64 to a float32's relative error of the mantissa's part alone
SSD_DEV double log2_of(double x)
{
    const unsigned long long u = __builtin_bit_cast(unsigned long long, x);
    const int e = (int)(u >> 52) - 1023;
    const float m = (float)__builtin_bit_cast(double, (u & 0x000FFFFFFFFFFFFFull) | 0x3FF0000000000000ull);
    return (double)e + (double)__builtin_amdgcn_logf(m);
}

SSD_DEV double ln_of(double x)
{
    if (!(x > 0.0) || x > 1e300) return log(x);
    return log2_of(x) * kLn2;
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

// ---- reductions over THREADS lanes that work on one row
template <int THREADS>
struct Team {
    static constexpr int kWaves = THREADS / 64 > 0 ? THREADS / 64 : 1;
    static constexpr int kWidth = THREADS < 64 ? THREADS : 64;
    double *lds;                      // kWaves * 4, unused by one wave

    SSD_DEV void sync() const
    {
        if constexpr (THREADS > 64) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");    // one wave's LDS accesses run in order
    }
    template <typename F>
    SSD_DEV void reduce(double (&x)[4], F f) const
    {
#pragma unroll
        for (int o = kWidth / 2; o > 0; o >>= 1) {
            double y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = __shfl_xor(x[i], o);
            f(x, y);
        }
        if constexpr (THREADS > 64) {
            const int wave = threadIdx.x >> 6;
            __syncthreads();
            if ((threadIdx.x & 63) == 0)
#pragma unroll
                for (int i = 0; i < 4; ++i) lds[wave * 4 + i] = x[i];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = lds[i];
            for (int w = 1; w < kWaves; ++w) {
                double y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = lds[w * 4 + i];
                f(x, y);
            }
        }
    }
    SSD_DEV void maxima(float &a, float &b, float &c) const
    {
        double x[4] = {(double)a, (double)b, (double)c, 0.0};
        reduce(x, [](double (&l)[4], const double (&r)[4]) {
            l[0] = fmax(l[0], r[0]);
            l[1] = fmax(l[1], r[1]);
            l[2] = fmax(l[2], r[2]);
        });
        a = (float)x[0];
        b = (float)x[1];
        c = (float)x[2];
    }
    SSD_DEV void sums(double (&x)[4]) const
    {
        reduce(x, [](double (&l)[4], const double (&r)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] += r[i];
        });
    }
};

// What a row's statistics make of an entry and of the classes outside.
struct RowTerms {
    float m, l2;                      // exp(u - max) = exp2((z - m) l2)
    double ln_s, inv_s;
    double t_top, ln_t;               // log q = (t - t_top) / tau - ln_t
    double inv_tau;
    double whole;                     // Q + q_r
    float ref, out;                   // outside: grad = exp2((z - ref) l2) * out
    float c;                          // g tau

    SSD_DEV double log_q(float t) const { return ((double)t - t_top) * inv_tau - ln_t; }
    SSD_DEV double log_p(float z) const { return ((double)z - (double)m) * inv_tau - ln_s; }
    SSD_DEV float q(float t) const { return __builtin_amdgcn_exp2f((float)(log_q(t) * kLog2eD)); }
    SSD_DEV float share(float z) const { return (float)((double)__builtin_amdgcn_exp2f((z - m) * l2) * inv_s); }
};

// The k-th entry's terms: (q, loss, p where it is the class's first).  dup: some class is given twice in this row.
SSD_DEV void add_entry(double (&sum)[4], const RowTerms &r, const DistArgs &p, long long row, int k, const Entry &e, float z,
                       bool dup)
{
    const float q = r.q(e.t);
    sum[0] += (double)q;
    if (q != 0.0f) sum[1] += (double)q * (r.log_q(e.t) - r.log_p(z));
    if (!p.teacher_lse) return;
    if (dup)
        for (int j = 0; j < k; ++j)
            if (entry_of(p, row, j).at == e.at) return;
    sum[2] += (double)r.share(z);
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
SSD_DEV double terms_finish(RowTerms &r, const DistArgs &p, long long row, double sum_q, double sum_loss, double sum_p,
                            float m, double s, float mo, double so, bool outside)
{
    r.m = m;
    r.ref = m;
    const double g = p.grad_loss ? (double)p.grad_loss[row] : 1.0 / (double)p.rows;
    r.c = (float)(g * (double)p.tau);
    r.whole = sum_q;
    double loss = sum_loss, out = r.whole * r.inv_s;
    if (p.teacher_lse) {
        double q_r = 1.0 - sum_q;
        if (q_r < 0.0) q_r = 0.0;
        if (outside && so > 0.0) {
            r.ref = mo;
            r.whole = sum_q + q_r;
            if (q_r > 0.0) {
                // near 1 a bucket's logarithm is what the entries leave of it, to their own relative error
                const double ln_pr = sum_p < 0.5 ? log1p(-sum_p)
                                                 : ((double)mo - (double)m) * r.inv_tau + log(so) - log(s);
                loss += q_r * ((sum_q < 0.5 ? log1p(-sum_q) : log(q_r)) - ln_pr);
            }
            const double down = (double)__builtin_amdgcn_exp2f((mo - m) * r.l2);
            out = r.whole * r.inv_s * down - q_r / so;
        }
    }
    r.out = (float)(out * (double)r.c);
    return loss * (double)p.tau * (double)p.tau;
}

// ------------------------------------------------------------------- a team of lanes a row
// TEAM lanes a row, R pieces of 16 bytes a lane.
template <typename T, int TEAM, int R>
__global__ __launch_bounds__(TEAM < 256 ? 256 : TEAM) void distill_row_kernel(const DistArgs p)
{
    typedef Piece<T> P;
    constexpr int kBlockThreads = TEAM < 256 ? 256 : TEAM;
    constexpr int kRows = kBlockThreads / TEAM;
    constexpr int kWords = TEAM * R * P::N / 32;
    __shared__ unsigned s_bits[kRows * kWords];
    __shared__ double s_red[kBlockThreads / 64 * 4];
    const int t = threadIdx.x % TEAM;
    const long long row = p.row0 + (long long)blockIdx.x * kRows + threadIdx.x / TEAM;
    if (row >= p.rows) return;                            // whole waves: a team is a wave or the workgroup
    unsigned *bits = s_bits + threadIdx.x / TEAM * kWords;
    const Team<TEAM> team = {s_red};
    const T *z = (const T *)p.logits + row * p.ld;

    P x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * TEAM + t) * P::N;
        x[r].load(z + at, p.classes - at);
    }
    for (int i = t; i < (p.classes + 31) / 32; i += TEAM) bits[i] = 0u;
    team.sync();
    float m = -INFINITY, mo = -INFINITY, t_top = -INFINITY;
    int twice = 0, inside = 0;
    for (int k = t; k < p.top; k += TEAM) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        t_top = fmaxf(t_top, e.t);
        const unsigned bit = 1u << (e.at & 31);
        if (atomicOr(&bits[e.at >> 5], bit) & bit) twice = 1;
        else ++inside;
    }
    team.sync();
    const bool tail = p.teacher_lse != nullptr;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * TEAM + t) * P::N;
        const unsigned in = tail && at < p.classes ? bits[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
            const float v = (float)x[r].v[i];
            m = fmaxf(m, v);
            if (tail && !(in >> i & 1u)) mo = fmaxf(mo, v);
        }
    }
    team.maxima(m, mo, t_top);
    RowTerms f;
    f.l2 = (float)(kLog2eD / (double)p.tau);
    const float mref = m == -INFINITY ? 0.0f : m, oref = mo == -INFINITY ? 0.0f : mo;
    float s = 0.0f, so = 0.0f, st = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * TEAM + t) * P::N;
        const unsigned in = tail && at < p.classes ? bits[at >> 5] >> (at & 31) : 0u;
#pragma unroll
        for (int i = 0; i < P::N; ++i) {
            const float v = (float)x[r].v[i];
            s += __builtin_amdgcn_exp2f((v - mref) * f.l2);
            if (tail && !(in >> i & 1u)) so += __builtin_amdgcn_exp2f((v - oref) * f.l2);
        }
    }
    if (!tail)
        for (int k = t; k < p.top; k += TEAM) {
            const Entry e = entry_of(p, row, k);
            if (e.at >= 0) st += __builtin_amdgcn_exp2f((e.t - t_top) * f.l2);
        }
    double sum[4] = {(double)s, (double)so, (double)st, (double)inside + 65536.0 * (double)twice};
    team.sums(sum);
    const int n_inside = (int)sum[3] % 65536;
    const bool dup = sum[3] >= 65536.0;
    if (n_inside == 0) {                                   // a row without an entry teaches nothing
        if (t == 0) p.loss[row] = 0.0f;
        if (p.grad) {
            P zero;
#pragma unroll
            for (int i = 0; i < P::N; ++i) zero.v[i] = (T)0.0f;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int at = (r * TEAM + t) * P::N;
                zero.store((T *)p.grad + row * p.classes + at, p.classes - at);
            }
        }
        return;
    }
    f.m = m;
    f.inv_s = 1.0 / sum[0];
    f.ln_s = ln_of(sum[0]);
    terms_teacher(f, p, row, t_top, sum[2]);
    double of_entries[4] = {0.0, 0.0, 0.0, 0.0};
    for (int k = t; k < p.top; k += TEAM) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        add_entry(of_entries, f, p, row, k, e, (float)z[e.at], dup);
    }
    team.sums(of_entries);
    const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2], m, sum[0], mo, sum[1],
                                     n_inside < p.classes);
    if (t == 0) p.loss[row] = (float)loss;
    if (!p.grad) return;
    T *g = (T *)p.grad + row * p.classes;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * TEAM + t) * P::N;
        P o;
#pragma unroll
        for (int i = 0; i < P::N; ++i)
            o.v[i] = (T)(__builtin_amdgcn_exp2f(((float)x[r].v[i] - f.ref) * f.l2) * f.out);
        o.store(g + at, p.classes - at);
    }
    team.sync();                                           // the entries' own values come last
    for (int k = t; k < p.top; k += TEAM) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        const double q = teacher_of(f, p, row, e, dup);
        g[e.at] = (T)(float)((double)f.c * ((double)f.share((float)z[e.at]) * f.whole - q));
    }
}

// ----------------------------------------------------------------------- few classes a row
// G lanes a row, up to 4 classes a lane.
template <typename T, int G>
__global__ __launch_bounds__(256) void distill_small_kernel(const DistArgs p)
{
    const int l = threadIdx.x % G;
    const long long row = p.row0 + ((long long)blockIdx.x * 256 + threadIdx.x) / G;
    if (row >= p.rows) return;                             // whole teams
    const Team<G> team = {nullptr};
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
    for (int k = 0; k < p.top; ++k) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        ++entries;
        t_top = fmaxf(t_top, e.t);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e.at == l + G * i) in |= 1u << i;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (!(in >> i & 1u)) mo = fmaxf(mo, x[i]);
    float unused = t_top;
    team.maxima(m, mo, unused);
    RowTerms f;
    f.l2 = (float)(kLog2eD / (double)p.tau);
    const float mref = m == -INFINITY ? 0.0f : m, oref = mo == -INFINITY ? 0.0f : mo;
    double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sum[0] += (double)__builtin_amdgcn_exp2f((x[i] - mref) * f.l2);
        if (!(in >> i & 1u)) sum[1] += (double)__builtin_amdgcn_exp2f((x[i] - oref) * f.l2);
        sum[2] += (double)(in >> i & 1u);
    }
    team.sums(sum);
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
    if (!p.teacher_lse)
        for (int k = 0; k < p.top; ++k) {
            const Entry e = entry_of(p, row, k);
            if (e.at >= 0) st += (double)__builtin_amdgcn_exp2f((e.t - t_top) * f.l2);
        }
    f.m = m;
    f.inv_s = 1.0 / sum[0];
    f.ln_s = ln_of(sum[0]);
    terms_teacher(f, p, row, t_top, st);
    double of_entries[4] = {0.0, 0.0, 0.0, 0.0}, q_at[4] = {0.0, 0.0, 0.0, 0.0};
    const bool dup = entries > (int)sum[2];
    for (int k = 0; k < p.top; ++k) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        add_entry(of_entries, f, p, row, k, e, (float)z[e.at], dup);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (e.at == l + G * i) q_at[i] += (double)f.q(e.t);
    }
    const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2], m, sum[0], mo, sum[1],
                                     (int)sum[2] < p.classes);
    if (l == 0) p.loss[row] = (float)loss;
    if (!p.grad) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int j = l + G * i;
        if (j >= p.classes) continue;
        const float o = (in >> i & 1u) ? (float)((double)f.c * ((double)f.share(x[i]) * f.whole - q_at[i]))
                                       : __builtin_amdgcn_exp2f((x[i] - f.ref) * f.l2) * f.out;
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

// grid: segments of a row back to back
template <typename T>
__global__ __launch_bounds__(kSegThreads) void distill_part_kernel(const DistArgs p)
{
    typedef Piece<T> P;
    constexpr int R = kSegMost / kSegThreads;
    __shared__ unsigned s_bits[kSegMost * P::N / 32];
    __shared__ double s_red[kSegThreads / 64 * 4];
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
    float m = -INFINITY, mo = -INFINITY, none = 0.0f;
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
    team.maxima(m, mo, none);
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
    double sum[4] = {(double)s, (double)so, (double)inside, 0.0};
    team.sums(sum);
    if (t == 0) p.part[row * p.segments + seg] = DistPart{m, mo, sum[0], sum[1], here - (int)sum[2], 0};
}

// grid: with a gradient as above, else one workgroup a row; each joins the row's parts in the same order
template <typename T>
__global__ __launch_bounds__(kSegThreads) void distill_segment_kernel(const DistArgs p)
{
    typedef Piece<T> P;
    constexpr int R = kSegMost / kSegThreads;
    __shared__ double s_red[kSegThreads / 64 * 4];
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
    float t_top = -INFINITY, a = 0.0f, b = 0.0f;
    int entries = 0;
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        ++entries;
        t_top = fmaxf(t_top, e.t);
    }
    team.maxima(t_top, a, b);
    double sum[4] = {(double)entries, 0.0, 0.0, 0.0};
    if (!p.teacher_lse)
        for (int k = t; k < p.top; k += kSegThreads) {
            const Entry e = entry_of(p, row, k);
            if (e.at >= 0) sum[1] += (double)__builtin_amdgcn_exp2f((e.t - t_top) * f.l2);
        }
    team.sums(sum);
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
    f.m = all.m;
    f.inv_s = 1.0 / all.s;
    f.ln_s = ln_of(all.s);
    terms_teacher(f, p, row, t_top, sum[1]);
    const bool dup = sum[0] > (double)(p.classes - all.outside);
    double of_entries[4] = {0.0, 0.0, 0.0, 0.0};
    for (int k = t; k < p.top; k += kSegThreads) {
        const Entry e = entry_of(p, row, k);
        if (e.at < 0) continue;
        add_entry(of_entries, f, p, row, k, e, (float)zr[e.at], dup);
    }
    team.sums(of_entries);
    const double loss = terms_finish(f, p, row, of_entries[0], of_entries[1], of_entries[2], all.m, all.s, all.mo, all.so,
                                     all.outside > 0);
    if (t == 0 && seg == 0) p.loss[row] = (float)loss;
    if (!p.grad) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int at = (r * kSegThreads + t) * P::N;
        P o;
#pragma unroll
        for (int i = 0; i < P::N; ++i)
            o.v[i] = (T)(__builtin_amdgcn_exp2f(((float)x[r].v[i] - f.ref) * f.l2) * f.out);
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
    q.cut = pieces > 2048 || (rows < 128 && pieces > 512);
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
    const unsigned grid = (unsigned)((rows + kThreads / TEAM - 1) / (kThreads / TEAM));
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
    else if (a.classes <= 4) launch_small<T, 1>(ctx, a, rows);
    else if (a.classes <= 8) launch_small<T, 2>(ctx, a, rows);
    else if (a.classes <= 16) launch_small<T, 4>(ctx, a, rows);
    else if (a.classes <= 32) launch_small<T, 8>(ctx, a, rows);
    else if (a.classes <= 64) launch_small<T, 16>(ctx, a, rows);
    else if (pieces <= 64) launch_row<T, 64, 1>(ctx, a, rows);
    else if (pieces <= 128) launch_row<T, 64, 2>(ctx, a, rows);
    else if (pieces <= 256) launch_row<T, 64, 4>(ctx, a, rows);
    else if (pieces <= 512) launch_row<T, 256, 2>(ctx, a, rows);
    else if (pieces <= 1024) launch_row<T, 256, 4>(ctx, a, rows);
    else launch_row<T, 256, 8>(ctx, a, rows);
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
        launch_distill<T>(ctx, a, q, (int)(a.rows - r < step ? a.rows - r : step));
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
