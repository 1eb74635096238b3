// A teacher's top logits and the loss that a student takes from them.
//
// top_logits: per row of V classes the k largest logits in order (ties to the lowest class, NaN above everything, -0 equal to +0), their
// classes, and lse = log sum_v exp(z_v / T).
//
// distillation, per row with teacher entries (i_k, t_k), an index outside 0 .. V-1 marking no entry:
//     p_k = exp(t_k / T - L),  L = the teacher's log-sum-exp at T if given, else log sum_k exp(t_k / T) (the entries renormalised);
//     q = softmax(z / T);   loss = T^2 [ sum_k p_k (log p_k - log q_{i_k}) + p_r (log p_r - log q_r) ]
// with p_r = max(0, 1 - sum p_k) and q_r = sum of q over the classes that no entry names, only if L is given and such classes have mass.
//     d loss / d z_v = T (q_v - sum_{k: i_k = v} p_k)      for a named class, and for every class when renormalised;
//                    = T q_v (1 - p_r / q_r)               for the others when L is given.
// The same class may be named twice (its p add up).  A row without entries, or with none but -inf to renormalise: loss 0, gradient 0.
//
// Numerics: q_v = 2^((z_v - o) c) / S with c = log2(e) / T and the row's largest logit o: fp32; the difference first, so that a row of the type's
// lowest values neither overflows nor loses its ratios.  Sums of exponentials in fp32, at most 128 per thread one after another, then joined in a tree across threads with
// their offsets: gradients are off by 2e-7 of the largest, the arguments' rounding included (the plain form with fp64 sums: 1e-7); fp64 here would be
// a conversion and a 64-bit addition per class more in passes that are bound by vector issue.  The row's few scalars -- lse, log p, log q,
// p_r, the loss -- are fp64: a small loss is the difference of logarithms that nearly cancel.
#include "cnm_common.h"

namespace {

constexpr int KMAX = 256;                    // entries per row
constexpr int VMAX = 1 << 20;                // classes per row
constexpr size_t LDS_BYTES = 160 * 1024;
constexpr float TMIN = 1e-37f;                // smallest temperature: log2(e) / T is finite
constexpr double LOG2E_D = 1.4426950408889634074, LN2_D = 0.69314718055994530942;

template <int DT> struct Elem;
template <> struct Elem<CNM_F32> { typedef float T; };
template <> struct Elem<CNM_F16> { typedef _Float16 T; };
template <> struct Elem<CNM_BF16> { typedef __bf16 T; };

__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Sums and maxima over a wave's 64 lanes (all of them active), the result in every lane: data-parallel moves within the vector unit -- shifts inside
// rows of 16, then the rows' last lanes handed on --, a few cycles a step where an exchange through LDS takes a hundred.
template <int CTRL, int ROWS>
__device__ inline float lane_move(float x, float none) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ inline double lane_move(double x) {                           // (lanes without a source: 0)
    const long long u = __double_as_longlong(x);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((long long)hi << 32 | (unsigned)lo);
}
__device__ inline float last_lane(float x) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63)); }
__device__ inline double last_lane(double x) {
    const long long u = __double_as_longlong(x);
    return __longlong_as_double((long long)__builtin_amdgcn_readlane((int)(u >> 32), 63) << 32 | (unsigned)__builtin_amdgcn_readlane((int)u, 63));
}
constexpr int SHR1 = 0x111, SHR2 = 0x112, SHR4 = 0x114, SHR8 = 0x118, BCAST15 = 0x142, BCAST31 = 0x143;
__device__ inline float sum_wave(float x) {
    x += lane_move<SHR1, 0xf>(x, 0.f); x += lane_move<SHR2, 0xf>(x, 0.f); x += lane_move<SHR4, 0xf>(x, 0.f); x += lane_move<SHR8, 0xf>(x, 0.f);
    x += lane_move<BCAST15, 0xa>(x, 0.f); x += lane_move<BCAST31, 0xc>(x, 0.f);
    return last_lane(x);
}
__device__ inline double sum_wave(double x) {
    x += lane_move<SHR1, 0xf>(x); x += lane_move<SHR2, 0xf>(x); x += lane_move<SHR4, 0xf>(x); x += lane_move<SHR8, 0xf>(x);
    x += lane_move<BCAST15, 0xa>(x); x += lane_move<BCAST31, 0xc>(x);
    return last_lane(x);
}
__device__ inline float max_wave(float x) {
    constexpr float none = -__builtin_huge_valf();
    x = fmaxf(x, lane_move<SHR1, 0xf>(x, none)); x = fmaxf(x, lane_move<SHR2, 0xf>(x, none)); x = fmaxf(x, lane_move<SHR4, 0xf>(x, none)); x = fmaxf(x, lane_move<SHR8, 0xf>(x, none));
    x = fmaxf(x, lane_move<BCAST15, 0xa>(x, none)); x = fmaxf(x, lane_move<BCAST31, 0xc>(x, none));
    return last_lane(x);
}

// (offset, sum) of exponentials 2^((x - offset) c); offset = -inf: none yet; +inf: the sum is +inf, or NaN
struct Lse { float o, s; };
__device__ inline float finite_or_0(float o) { return fabsf(o) == __builtin_huge_valf() ? 0.f : o; }   // what an offset is subtracted as
__device__ inline Lse lse_join(Lse a, Lse b, float c) {
    const float o = fmaxf(a.o, b.o);                                     // (fmaxf drops a NaN: it is in the sum then)
    const float so = finite_or_0(o);
    // an empty side has s = 0 and offset -inf: 0 * 2^-inf = 0
    return {o, a.s * exp2_((a.o - so) * c) + b.s * exp2_((b.o - so) * c)};
}
__device__ inline Lse lse_wave(Lse a, float c) {
    const float o = max_wave(a.o), so = finite_or_0(o);
    return {o, sum_wave(a.s * exp2_((a.o - so) * c))};
}
// the natural logarithm of the sum, in units of 1 / T
__device__ inline float lse_value(Lse l, float T) {
    return l.s == 0.f ? -__builtin_huge_valf() : (float)((double)finite_or_0(l.o) / (double)T + log((double)l.s));
}
// joined over NT threads in a fixed order; every thread gets the result.  `sh` holds 2 * NT / 64 floats
template <int NT>
__device__ inline Lse lse_block(Lse a, float c, float* sh) {
    a = lse_wave(a, c);
    if (NT == 64) return a;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) { sh[2 * (threadIdx.x >> 6)] = a.o; sh[2 * (threadIdx.x >> 6) + 1] = a.s; }
    __syncthreads();
    const int l = threadIdx.x & 63;
    a = l < NT / 64 ? Lse{sh[2 * l], sh[2 * l + 1]} : Lse{-__builtin_huge_valf(), 0.f};
    return lse_wave(a, c);
}
template <int NT>
__device__ inline double sum_block(double a, double* sh) {
    a = sum_wave(a);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = a;
    __syncthreads();
    return sum_wave((threadIdx.x & 63) < NT / 64 ? sh[threadIdx.x & 63] : 0.0);
}
// sixteen bytes of a row as they are in memory, elements beyond the row -inf.  hold(): conversions done so far are forgotten (left alone, hipcc
// keeps every converted element in a register of its own from one pass over the row to the next)
template <int DT>
struct Raw {
    typedef typename Elem<DT>::T T;
    static constexpr int E = 16 / sizeof(T);
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    u32x4 w;
    __device__ void load(const T* row, int at, int n) {
        if (at + E <= n) __builtin_memcpy(&w, row + at, 16);             // (whatever the row's alignment)
        else {
            T v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = at + j < n ? row[at + j] : (T)-__builtin_huge_valf();
            __builtin_memcpy(&w, v, 16);
        }
    }
    __device__ void hold() { asm volatile("" : "+v"(w)); }
    __device__ void drop(unsigned b) {                                   // the elements whose bit is set become -inf
        if constexpr (DT == CNM_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = b >> j & 1u ? 0xFF800000u : w[j];
        } else {
            constexpr unsigned none = DT == CNM_BF16 ? 0xFF80u : 0xFC00u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = b >> (2 * j) & 1u ? (w[j] & 0xFFFF0000u) | none : w[j];
                w[j] = b >> (2 * j + 1) & 1u ? (w[j] & 0xFFFFu) | none << 16 : w[j];
            }
        }
    }
    __device__ float get(int j) const {
        if constexpr (DT == CNM_F32) return __uint_as_float(w[j]);
        else if constexpr (DT == CNM_BF16) return __uint_as_float(j & 1 ? w[j / 2] & 0xFFFF0000u : w[j / 2] << 16);
        else { const unsigned short h = (unsigned short)(j & 1 ? w[j / 2] >> 16 : w[j / 2]); return (float)__builtin_bit_cast(_Float16, h); }
    }
};

// running largest value and sum of the exponentials 2^((x - o) c), o = the largest value (0 while there is none but -inf, and where it is +inf)
struct Run {
    float m = -__builtin_huge_valf(), o = 0.f, s = 0.f;
    __device__ void raise(float x, float c) {                            // a new largest value
        if (m != -__builtin_huge_valf()) s *= exp2_((m - x) * c);
        m = x; o = finite_or_0(x);
    }
    __device__ Lse lse() const { return {m == -__builtin_huge_valf() ? m : o, s}; }
};

__device__ inline long long load_index(const void* idx, bool wide, size_t at) {
    return wide ? static_cast<const long long*>(idx)[at] : (long long)static_cast<const int*>(idx)[at];
}
__device__ inline float load_any(const void* p, int dt, size_t at) {
    return dt == CNM_F32 ? static_cast<const float*>(p)[at] : dt == CNM_F16 ? (float)static_cast<const _Float16*>(p)[at] : (float)static_cast<const __bf16*>(p)[at];
}

struct DistillArgs {
    const void* z; long long ldz;            // rows of V classes, ldz apart; or [outer][V][inner]
    const void* idx; int wide;               // [rows][K] or [outer][K][inner], int32 / int64
    const void* val; int vdt;                // the entries' logits
    const float* lse;                        // [rows] or null: renormalised
    float T, c; double iT, l2T;              // temperature; log2(e) / T in fp32, 1 / T and log2(e) / T in fp64
    const float* weight;                     // [rows] or null
    const double* wpart; int nwpart;         // the weights' partial sums (gradients are divided by their sum), or null
    double inv_norm;                         // otherwise multiplied by this
    const float* go; int go_rows;            // upstream gradient: one value, or one per row; null: 1
    int skip_if_one;                         // *go == 1: the gradient is already there (written by the forward pass)
    float* loss;                             // [rows]: weight * loss, or null
    double* lpart;                           // per row or per workgroup: weight * loss, or null
    void* dz;                                // as z but dense, or null
    long long rows; int V, K; long long inner;
    struct DistillRow* rec; float* seg;      // rows cut into segments: what each amounts to, and [rows][segments][2] (offset, sum)
    int segments, seglen;
};

// What a row amounts to: an unnamed class's gradient is A 2^((z - orest) c), a named one's B (2^((z - oall) c) inv - p); B = 0: nothing.  A and B
// for an upstream gradient of 1, in fp64: with the upstream gradient they become fp32, and only that product has to be one
struct DistillRow { double L, A, B; float orest, oall, inv, pad; };

// sum of up to 64 partial sums, in a fixed order, by a whole wave
__device__ inline double wave_total(const double* part, int n) {
    return sum_wave((int)(threadIdx.x & 63) < n ? part[threadIdx.x & 63] : 0.0);
}

// what a mean multiplies by: inv_norm / (sum of the weights), 0 where they sum to 0.  A sum below 0 is a sum like any other, and one that is NaN or
// infinite goes on: a mask with a NaN in it gives NaN, not a loss of 0
__device__ inline double weight_norm(const double* part, int n, double inv_norm, bool* none = nullptr) {
    const double s = wave_total(part, n);
    if (none) *none = s == 0.0;
    return s == 0.0 ? 0.0 : inv_norm / s;
}

// 2^x, relative error of a few 2^-24 whatever x's size
__device__ inline float exp2_of(double x) {
    if (!(x > -160.0)) return x != x ? (float)x : 0.f;
    if (x > 130.0) return __builtin_huge_valf();
    const double n = rint(x);
    return ldexpf(exp2_((float)(x - n)), (int)n);
}

// What a row's entries say by themselves: the teacher's log-sum-exp, sum p, sum p log2 p, the named classes' exponentials.
struct Teacher { double L, P, lp; Lse named; int have; };

// The entries of a row, shared by the threads that work on it.
struct Entries {
    int idx[KMAX];                                                       // -1: none
    float z[KMAX], p[KMAX];                                              // the student's logit there; the teacher's logit, then the probability
    int dup;                                                             // some class is named twice
    Teacher teach;
    Lse rest[16];                                                        // the waves' statistics of the unnamed classes
    DistillRow row;
};
template <int NT>
__device__ inline void row_sync() {
    if (NT == 64) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }
    else __syncthreads();
}

template <int DT, int NT>
__device__ inline void load_entries(const DistillArgs& a, size_t r, const typename Elem<DT>::T* z, Entries& e, int t) {
    for (int k = t; k < a.K; k += NT) {
        const long long i = load_index(a.idx, a.wide, r * a.K + k);
        const bool ok = i >= 0 && i < a.V;
        e.idx[k] = ok ? (int)i : -1;
        e.p[k] = ok ? load_any(a.val, a.vdt, r * a.K + k) : 0.f;
        e.z[k] = ok ? (float)z[i] : 0.f;
    }
}
// the named classes' bits among the n from v0 on; a bit that is there already: a class named twice
template <int NT>
__device__ inline void mark_entries(Entries& e, int K, unsigned* bits, int v0, int n, int t) {
    for (int k = t; k < K; k += NT) {
        const int i = e.idx[k] - v0;
        if (e.idx[k] >= 0 && i >= 0 && i < n && (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31) & 1u)) e.dup = 1;
    }
}
__device__ inline double entry_log2p(const DistillArgs& a, float logit, double L) { return (double)logit * a.l2T - L * LOG2E_D; }

// a class that is named more than once: its first entry gets the sum, the others become none (one wave)
__device__ inline void join_entries(Entries& e, int K, int lane) {
    if (!e.dup) return;
    float s[KMAX / 64];
    bool first[KMAX / 64];
#pragma unroll
    for (int q = 0; q < KMAX / 64; ++q) {
        const int k = q * 64 + lane;
        first[q] = k < K && e.idx[k] >= 0; s[q] = 0.f;
        if (first[q])
            for (int j = 0; j < K; ++j) if (e.idx[j] == e.idx[k]) { if (j < k) first[q] = false; s[q] += e.p[j]; }
    }
    row_sync<64>();
#pragma unroll
    for (int q = 0; q < KMAX / 64; ++q) {
        const int k = q * 64 + lane;
        if (k < K) { e.p[k] = s[q]; if (!first[q]) e.idx[k] = -1; }
    }
    row_sync<64>();
}

// A row's numbers, by one wave while the others go over the classes: the fp64 logarithms are hundreds of instructions, too many for every wave.
// First what the entries alone say (e.p becomes the probabilities), then, with the unnamed classes' statistics, the loss and the gradient's
// coefficients for an upstream gradient of 1.
__device__ inline Teacher entry_numbers(const DistillArgs& a, size_t r, Entries& e, float c, int lane) {
    const float ninf = -__builtin_huge_valf();
    Teacher w;
    w.named = {ninf, 0.f};
    float best = ninf;
    bool have = false;
    for (int k = lane; k < a.K; k += 64) {
        const int i = e.idx[k];
        bool first = i >= 0;
        if (first) { have = true; best = fmaxf(best, e.p[k]); }
        if (e.dup) for (int j = 0; j < k && first; ++j) first = e.idx[j] != i;
        if (first) {
            const float x = e.z[k];
            w.named = lse_join(w.named, Lse{x, x == ninf ? 0.f : 1.f + (x - x)}, c);   // (NaN for an infinite or NaN logit: there is no softmax)
        }
    }
    w.have = __any(have);
    w.named = lse_wave(w.named, c);
    if (a.lse) w.L = (double)a.lse[r];
    else {
        best = max_wave(best);
        if (best == ninf) best = 0.f;
        double s = 0.0;
        for (int k = lane; k < a.K; k += 64) if (e.idx[k] >= 0) s += (double)exp2_of(((double)e.p[k] - (double)best) * a.l2T);
        s = sum_wave(s);
        w.L = (double)best * a.iT + log(s);
        if (s == 0.0) { w.L = 0.0; w.have = 0; }                         // entries of -inf: no mass, no entries
    }
    double P = 0.0, lp = 0.0;
    for (int k = lane; k < a.K; k += 64) {
        float p = 0.f;
        if (e.idx[k] >= 0) {
            const double l = entry_log2p(a, e.p[k], w.L);
            p = exp2_of(l);
            if (p != 0.f) lp += (double)p * l;                           // (a NaN is not 0)
            P += (double)p;
        }
        e.p[k] = p;
    }
    w.P = sum_wave(P); w.lp = sum_wave(lp);
    return w;
}
__device__ inline DistillRow finish_row(const DistillArgs& a, size_t r, Lse rest, const Teacher& w, Entries& e, float c, int lane) {
    const float ninf = -__builtin_huge_valf();
    const Lse all = lse_join(rest, w.named, c);
    DistillRow row;
    row.L = w.L;
    row.oall = all.o == ninf ? 0.f : all.o; row.orest = rest.o == ninf ? 0.f : rest.o;
    const double lq0 = -log2((double)all.s);                             // log2 q_v = (z_v - oall) c + lq0
    double loss = 0.0;
    for (int k = lane; k < a.K; k += 64)
        if (e.p[k] != 0.f) loss -= (double)e.p[k] * (((double)e.z[k] - (double)row.oall) * (double)c + lq0);
    loss = (w.lp + sum_wave(loss)) * LN2_D;
    double ratio = 0.0;                                                  // p_r / (sum of the unnamed exponentials)
    if (a.lse && rest.s != 0.f) {
        const double pr = 1.0 - w.P;
        if (!(pr <= 0.0)) {
            // q_r from the smaller side: 1 - Q keeps its digits where the named classes hold little
            const double Q = w.named.o == ninf ? 0.0 : (double)w.named.s * (double)exp2_of(((double)w.named.o - (double)row.oall) * (double)c + lq0);
            const double lqr = Q < 0.5 ? log1p(-Q) : (((double)row.orest - (double)row.oall) * (double)c + log2((double)rest.s) + lq0) * LN2_D;
            loss += pr * (log1p(-w.P) - lqr);
            ratio = pr / (double)rest.s;
        }
    }
    loss *= (double)a.T * (double)a.T;
    if (!w.have) loss = 0.0;
    const float wrow = a.weight ? a.weight[r] : 1.f;
    if (lane == 0) {
        const double l = wrow != 0.f ? (double)wrow * loss : 0.0;        // (weight 0: whatever the logits hold)
        if (a.loss) a.loss[r] = (float)l;
        if (a.lpart) a.lpart[r] = l;
    }
    double norm = a.inv_norm;
    if (a.wpart) norm = weight_norm(a.wpart, a.nwpart, a.inv_norm);
    const double scale = w.have ? (double)a.T * (double)wrow * norm : 0.0;
    row.inv = 1.f / all.s;
    row.A = rest.s == 0.f ? 0.0 : scale * ((double)exp2_((row.orest - row.oall) * c) / (double)all.s - ratio);   // (no mass outside the entries: nothing to scale)
    row.B = scale;
    row.pad = 0.f;
    return row;
}

// NT threads per row (MODE ROW) or segment of a row, which they hold in registers (NV vectors of 16 bytes each): z is read once, the gradient
// written once.  LDS: one bit per class (named by an entry), one byte (by which), the entries.
// bf16 4096 x 32768 with the gradient: about 140 us of launch (3.8 TB/s; a copy of the same bytes 99): 20 vector instructions per class, two of them
// exponentials, beside memory, three rows per CU at once.
// A row that no workgroup can hold, or one of few, is cut into segments: statistics of each (SEG_STATS), the row's numbers (distill_join_kernel),
// gradients of each (SEG_GRAD), the second reading from the caches.
enum { ROW, SEG_STATS, SEG_GRAD };
template <int DT, int NT, int NV, int MODE>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, NT == 512 && NV == 8 ? 6 : 1) void distill_rows_kernel(const DistillArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int RPB = NT == 64 ? 4 : 1, E = 16 / sizeof(T);
    extern __shared__ unsigned lds_words[];
    __shared__ Entries entries[RPB];
    const int sub = NT == 64 ? threadIdx.x >> 6 : 0, t = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    const int nw = (a.seglen + 31) / 32;
    unsigned* const bits = lds_words + sub * 9 * nw;                     // [nw], then a byte per class: the entry that names it, written where a bit is set
    unsigned char* const slot = reinterpret_cast<unsigned char*>(bits + nw);
    Entries& e = entries[sub];
    float go = 1.f;
    if (a.go && !a.go_rows) {
        go = a.go[0];
        if (a.skip_if_one && go == 1.f) return;
    }
    const long long unit = (long long)blockIdx.x * RPB + sub;
    if (unit >= a.rows * a.segments) return;                             // (whole waves only: NT == 64)
    const size_t r = (size_t)(unit / a.segments);
    const int seg = (int)(unit - (long long)r * a.segments), v0 = seg * a.seglen, n = min(a.V - v0, a.seglen);
    const T* const zrow = static_cast<const T*>(a.z) + r * a.ldz;
    const T* const z = zrow + v0;
    if (a.go && a.go_rows) go = a.go[r];
    const float c = a.c, ninf = -__builtin_huge_valf();
    Raw<DT> x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i].load(z, (i * NT + t) * E, n);
    for (int i = t; i < nw; i += NT) bits[i] = 0u;
    if (t == 0) e.dup = 0;
    load_entries<DT, NT>(a, r, zrow, e, t);
    row_sync<NT>();
    mark_entries<NT>(e, a.K, bits, v0, n, t);
    row_sync<NT>();
    const int lane = threadIdx.x & 63;
    // named classes leave the row: their places are -inf from here on
    const auto named = [&](int at) { return at < n ? bits[at >> 5] >> (at & 31) & ((1u << E) - 1) : 0u; };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const unsigned b = named((i * NT + t) * E);
        if (b) x[i].drop(b);
    }
    if constexpr (MODE != SEG_GRAD) {
        if (MODE == ROW && t < 64) { const Teacher teach = entry_numbers(a, r, e, c, lane); if (lane == 0) e.teach = teach; }
        float m = ninf;                                                  // statistics of the unnamed classes
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i].hold();
#pragma unroll
            for (int j = 0; j < E; ++j) m = fmaxf(m, x[i].get(j));
        }
        const float o = m == ninf ? 0.f : m;
        Lse rest = {m, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i].hold();
#pragma unroll
            for (int j = 0; j < E; ++j) rest.s += exp2_((x[i].get(j) - o) * c);
        }
        rest = lse_wave(rest, c);
        if (NT > 64) {
            if (lane == 0) e.rest[t >> 6] = rest;
            __syncthreads();
            if (t < 64) rest = lse_wave(lane < NT / 64 ? e.rest[lane] : Lse{ninf, 0.f}, c);
        }
        if constexpr (MODE == SEG_STATS) {
            if (t == 0) { a.seg[2 * unit] = rest.o; a.seg[2 * unit + 1] = rest.s; }
            return;
        }
        if (t < 64) {
            row_sync<64>();
            const DistillRow row = finish_row(a, r, rest, e.teach, e, c, lane);
            if (lane == 0) e.row = row;
            row_sync<64>();
        }
    } else {
        if (t == 0) e.row = a.rec[r];
        const double L = a.rec[r].L;
        for (int k = t; k < a.K; k += NT) e.p[k] = e.idx[k] >= 0 ? exp2_of(entry_log2p(a, e.p[k], L)) : 0.f;
        row_sync<NT>();
    }
    if (!a.dz) return;
    if (t < 64) {                                                        // the named classes' gradients, each once, and which class each belongs to
        join_entries(e, a.K, lane);
        const DistillRow w = e.row;
        const float B = (float)(w.B * (double)go);
        for (int k = lane; k < a.K; k += 64) {
            const int i = e.idx[k] - v0;
            if (e.idx[k] >= 0 && i >= 0 && i < n) {
                slot[i] = (unsigned char)k;
                // (a named class may lie far above the unnamed ones: its own exponent against the whole row's)
                e.p[k] = B == 0.f ? 0.f : B * (exp2_((e.z[k] - w.oall) * c) * w.inv - e.p[k]);
            }
        }
    }
    row_sync<NT>();
    const float A = (float)(e.row.A * (double)go), orest = e.row.orest;
    const bool zero = (float)(e.row.B * (double)go) == 0.f;                // rows that count for nothing: zeros, whatever the logits hold
    T* const dz = static_cast<T*>(a.dz) + r * a.V + v0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int at = (i * NT + t) * E;
        if (at < n) {
            x[i].hold();
            float g[E];
#pragma unroll
            for (int j = 0; j < E; ++j) g[j] = A * exp2_((x[i].get(j) - orest) * c);
            if (zero) {
#pragma unroll
                for (int j = 0; j < E; ++j) g[j] = 0.f;
            }
            const unsigned b = named(at);
            if (b) {
#pragma unroll
                for (int j = 0; j < E; ++j) if (b >> j & 1u) g[j] = e.p[slot[at + j]];
            }
            T out[E];
#pragma unroll
            for (int j = 0; j < E; ++j) out[j] = (T)g[j];
            if (at + E <= n) __builtin_memcpy(dz + at, out, 16);
            else {
#pragma unroll
                for (int j = 0; j < E; ++j) if (at + j < n) dz[at + j] = out[j];
            }
        }
    }
}

template <int DT>
__global__ __launch_bounds__(64) void distill_join_kernel(const DistillArgs a) {
    typedef typename Elem<DT>::T T;
    __shared__ Entries e;
    const int t = threadIdx.x;
    if (a.skip_if_one && a.go && a.go[0] == 1.f) return;
    const size_t r = blockIdx.x;
    const float c = a.c;
    if (t == 0) e.dup = 1;                                               // (no bits here to tell: looked up)
    load_entries<DT, 64>(a, r, static_cast<const T*>(a.z) + r * a.ldz, e, t);
    row_sync<64>();
    const Teacher teach = entry_numbers(a, r, e, c, t);
    Lse rest = {-__builtin_huge_valf(), 0.f};
    for (int i = t; i < a.segments; i += 64) rest = lse_join(rest, Lse{a.seg[2 * (r * a.segments + i)], a.seg[2 * (r * a.segments + i) + 1]}, c);
    const DistillRow row = finish_row(a, r, lse_wave(rest, c), teach, e, c, t);
    if (t == 0) a.rec[r] = row;
}

// The same with the classes in the middle: [outer][V][inner], a workgroup takes 64 neighbouring positions ("pixels"), one per lane.  The tile is
// read once, into LDS, and the gradient leaves from there.  Wave 0 takes the named classes out of the tile (-inf in their place) and works out
// the pixels' numbers -- it alone, for its fp64 logarithms --, the other three share the statistics of the rest; the gradient is everybody's.
// LDS: 64 floats per class, one bit per class and pixel, the entries.
// fp32 [4, 64, 192, 256], 8 entries: about 40 us (2.9 TB/s); 25 KB a
// workgroup, so that one's fp64 logarithms run beside the others' loads.
template <int DT>
__global__ __launch_bounds__(256) void distill_planes_kernel(const DistillArgs a, int tiles) {
    typedef typename Elem<DT>::T T;
    extern __shared__ unsigned lds_words[];
    const int V = a.V, K = a.K, nw = (V + 31) / 32;
    float* const tile = reinterpret_cast<float*>(lds_words);             // [V][64]
    unsigned* const bits = lds_words + V * 64;                           // [nw][64]
    int* const eidx = reinterpret_cast<int*>(bits + nw * 64);            // [K][64]: -1: none, or named by an earlier entry (then that class is -2 - eidx)
    float* const ep = reinterpret_cast<float*>(eidx + K * 64);           // [K][64]: the entry's logit, then its p
    float* const ez = ep + K * 64;                                       // [K][64]: the student's logit there
    float* const sh = ez + K * 64;                                       // [3][64][2]: the waves' statistics; then [4][64]: the pixels' numbers
    float go = 1.f;
    if (a.go && !a.go_rows) {
        go = a.go[0];
        if (a.skip_if_one && go == 1.f) return;
    }
    const int px = threadIdx.x & 63, w = threadIdx.x >> 6;
    const long long ob = blockIdx.x / tiles;
    const long long p0 = (long long)(blockIdx.x % tiles) * 64;
    const bool live = p0 + px < a.inner;
    const size_t at = live ? p0 + px : 0;                                // position in a plane
    const T* const z = static_cast<const T*>(a.z) + (size_t)ob * V * a.inner + at;
    const size_t ebase = (size_t)ob * K * a.inner + at, r = (size_t)ob * a.inner + at;
    const float c = a.c, ninf = -__builtin_huge_valf();

    for (int i = w; i < nw; i += 4) bits[i * 64 + px] = 0u;
    T first[16];                                                         // sixteen of the wave's classes are requested before anything waits
#pragma unroll
    for (int j = 0; j < 16; ++j) first[j] = z[(size_t)min(w + 4 * j, V - 1) * a.inner];
    for (int k = w; k < K; k += 4) {
        const long long i = live ? load_index(a.idx, a.wide, ebase + (size_t)k * a.inner) : -1;
        const bool ok = i >= 0 && i < V;
        eidx[k * 64 + px] = ok ? (int)i : -1;
        ep[k * 64 + px] = ok ? load_any(a.val, a.vdt, ebase + (size_t)k * a.inner) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) if (w + 4 * j < V) tile[(w + 4 * j) * 64 + px] = live ? (float)first[j] : 0.f;
#pragma unroll 8
    for (int v = w + 64; v < V; v += 4) tile[v * 64 + px] = live ? (float)z[(size_t)v * a.inner] : 0.f;
    __syncthreads();
    Lse named = {ninf, 0.f};
    bool have = false, dup = false;
    if (w == 0) {
        for (int k = 0; k < K; ++k) {
            const int i = eidx[k * 64 + px];
            if (i >= 0) {
                have = true;
                unsigned* const b = bits + (i >> 5) * 64 + px;
                if (*b >> (i & 31) & 1u) {                               // named before: the logit from that entry
                    dup = true;
                    for (int j = 0; j < k; ++j) if (eidx[j * 64 + px] == i) ez[k * 64 + px] = ez[j * 64 + px];
                    eidx[k * 64 + px] = -2 - i;
                } else {
                    *b |= 1u << (i & 31);
                    const float x = tile[i * 64 + px];
                    ez[k * 64 + px] = x;
                    tile[i * 64 + px] = ninf;
                    named = lse_join(named, Lse{x, x == ninf ? 0.f : 1.f + (x - x)}, c);
                }
            }
        }
    }
    __syncthreads();
    double L = 0.0, P = 0.0, loss = 0.0;
    if (w == 0) {                                                        // what the entries alone say
        if (a.lse) L = (double)a.lse[r];
        else {
            float best = ninf;
            for (int k = 0; k < K; ++k) if (eidx[k * 64 + px] != -1) best = fmaxf(best, ep[k * 64 + px]);
            if (best == ninf) best = 0.f;
            double s = 0.0;
            for (int k = 0; k < K; ++k) if (eidx[k * 64 + px] != -1) s += (double)exp2_of(((double)ep[k * 64 + px] - (double)best) * a.l2T);
            L = (double)best * a.iT + log(s);
            if (s == 0.0) { L = 0.0; have = false; }                     // entries of -inf: no mass, no entries
        }
        for (int k = 0; k < K; ++k) {
            float p = 0.f;
            if (eidx[k * 64 + px] != -1) {
                const double l = entry_log2p(a, ep[k * 64 + px], L);
                p = exp2_of(l);
                if (p != 0.f) loss += (double)p * l;                     // (a NaN is not 0)
                P += (double)p;
            }
            ep[k * 64 + px] = p;
        }
    } else {
        float m = ninf, s = 0.f;
        for (int v = w - 1; v < V; v += 3) m = fmaxf(m, tile[v * 64 + px]);
        const float o = m == ninf ? 0.f : m;
        for (int v = w - 1; v < V; v += 3) s += exp2_((tile[v * 64 + px] - o) * c);
        sh[((w - 1) * 64 + px) * 2] = m; sh[((w - 1) * 64 + px) * 2 + 1] = s;
    }
    __syncthreads();
    if (w == 0) {
        Lse rest = {sh[px * 2], sh[px * 2 + 1]};
        for (int i = 1; i < 3; ++i) rest = lse_join(rest, Lse{sh[(i * 64 + px) * 2], sh[(i * 64 + px) * 2 + 1]}, c);
        const Lse all = lse_join(rest, named, c);
        const float oall = all.o == ninf ? 0.f : all.o, orest = rest.o == ninf ? 0.f : rest.o;
        const double lq0 = -log2((double)all.s);
        for (int k = 0; k < K; ++k)
            if (ep[k * 64 + px] != 0.f) loss -= (double)ep[k * 64 + px] * (((double)ez[k * 64 + px] - (double)oall) * (double)c + lq0);
        loss *= LN2_D;
        double ratio = 0.0;
        if (a.lse && rest.s != 0.f) {
            const double pr = 1.0 - P;
            if (!(pr <= 0.0)) {
                const double Q = named.o == ninf ? 0.0 : (double)named.s * (double)exp2_of(((double)named.o - (double)oall) * (double)c + lq0);
                const double lqr = Q < 0.5 ? log1p(-Q) : (((double)orest - (double)oall) * (double)c + log2((double)rest.s) + lq0) * LN2_D;
                loss += pr * (log1p(-P) - lqr);
                ratio = pr / (double)rest.s;
            }
        }
        loss *= (double)a.T * (double)a.T;
        if (!have) loss = 0.0;
        const float wrow = live ? (a.weight ? a.weight[r] : 1.f) : 0.f;
        const double wloss = wrow != 0.f ? (double)wrow * loss : 0.0;
        if (a.loss && live) a.loss[r] = (float)wloss;
        if (a.lpart) {
            const double l = sum_wave(wloss);
            if (px == 0) a.lpart[blockIdx.x] = l;
        }
        if (a.dz) {
            double norm = a.inv_norm;
            if (a.wpart) norm = weight_norm(a.wpart, a.nwpart, a.inv_norm);
            if (a.go && a.go_rows) go = a.go[r];
            const double scale = have ? (double)a.T * (double)go * (double)wrow * norm : 0.0;
            const float B = (float)scale;
            const float A = rest.s == 0.f ? 0.f : (float)(scale * ((double)exp2_((orest - oall) * c) / (double)all.s - ratio));
            const float inv = 1.f / all.s;
            for (int k = 0; k < K; ++k) {                                // the named classes' gradients into their places
                const int i = eidx[k * 64 + px];
                if (i >= 0) {
                    float p = ep[k * 64 + px];
                    if (dup) for (int j = k + 1; j < K; ++j) if (eidx[j * 64 + px] == -2 - i) p += ep[j * 64 + px];
                    tile[i * 64 + px] = B == 0.f ? 0.f : B * (exp2_((ez[k * 64 + px] - oall) * c) * inv - p);
                }
            }
            sh[px] = A; sh[64 + px] = orest; sh[128 + px] = B;
        }
    }
    if (!a.dz) return;
    __syncthreads();
    if (!live) return;
    const float A = sh[px], o = sh[64 + px];
    const bool zero = sh[128 + px] == 0.f;                               // pixels that count for nothing: zeros, whatever the logits hold
    T* const dz = static_cast<T*>(a.dz) + (size_t)ob * V * a.inner + at;
    for (int v0 = 0; v0 < V; v0 += 32) {
        const unsigned b = bits[(v0 >> 5) * 64 + px] >> w;
        T* const d = dz + (size_t)(v0 + w) * a.inner;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int v = v0 + w + 4 * j;
            if (v < V) {
                const float x = tile[v * 64 + px];
                d[(size_t)(4 * j) * a.inner] = (T)(b >> (4 * j) & 1u ? x : zero ? 0.f : A * exp2_((x - o) * c));
            }
        }
    }
}

size_t planes_lds(int V, int K) { return (size_t)64 * 4 * ((size_t)V + (V + 31) / 32 + 3 * (size_t)K + 6); }

// partial sums of the weights, one per workgroup, each in a fixed order
constexpr int WPARTS = 64;
__global__ __launch_bounds__(1024) void weight_parts_kernel(const float* __restrict__ w, long long n, double* __restrict__ part) {
    __shared__ double sh[16];
    double s = 0.0;
    for (long long i = (long long)blockIdx.x * 1024 + threadIdx.x; i < n; i += (long long)gridDim.x * 1024) s += (double)w[i];
    s = sum_block<1024>(s, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// loss = sum of the workgroups' sums * inv_norm / (sum of the weights); no weight at all: 0
__global__ __launch_bounds__(1024) void loss_total_kernel(const double* __restrict__ part, long long n, const double* __restrict__ wpart, int nwpart, double inv_norm, float* __restrict__ out) {
    __shared__ double sh[16];
    double s = 0.0;
    for (long long i = threadIdx.x; i < n; i += 1024) s += part[i];
    s = sum_block<1024>(s, sh);
    if (threadIdx.x >= 64) return;
    double norm = inv_norm;
    bool none = false;
    if (wpart) norm = weight_norm(wpart, nwpart, inv_norm, &none);
    if (threadIdx.x == 0) out[0] = none ? 0.f : (float)(s * norm);
}

// How rows are split: 1024 threads hold 256 KB of a row in registers; longer rows, and long ones of fewer than 128, are cut into segments.
int distill_segments(long long rows, int V, int esize) {
    const size_t bytes = (size_t)V * esize;
    int want = (int)((bytes + (256 << 10) - 1) / (256 << 10));
    if (rows < 128 && bytes > (16 << 10)) {
        const int fit = (int)(bytes / (8 << 10)), fill = (int)(256 / rows);
        const int more = fit < fill ? fit : fill;
        want = more > want ? more : want;
    }
    return want;
}

// threads that share a row or segment of so many vectors
int distill_threads(int vecs) { return vecs <= 256 ? 64 : vecs <= 1024 ? 256 : vecs <= 4096 ? 512 : 1024; }
int top_threads(int vecs) { return vecs <= 64 ? 64 : vecs <= 256 ? 256 : vecs <= 2048 ? 512 : 256; }
// a launch holds fewer than 2^32 threads; rows by fours where a wave takes a whole one
bool launch_fits(long long units, int threads) { return (units + 3) * threads < (1ll << 32); }

template <int DT, int MODE>
void launch_rows(const DistillArgs& a, hipStream_t stream) {
    constexpr int E = 16 / (int)sizeof(typename Elem<DT>::T);
    const int vecs = a.seglen / E;
    const unsigned units = (unsigned)(a.rows * a.segments);
    const size_t lds = (size_t)((a.seglen + 31) / 32) * 4 * 9;           // a bit and a byte per class
    if (vecs <= 64) distill_rows_kernel<DT, 64, 1, MODE><<<(units + 3) / 4, 256, 4 * lds, stream>>>(a);
    else if (vecs <= 256) distill_rows_kernel<DT, 64, 4, MODE><<<(units + 3) / 4, 256, 4 * lds, stream>>>(a);
    else if (vecs <= 512) distill_rows_kernel<DT, 256, 2, MODE><<<units, 256, lds, stream>>>(a);
    else if (vecs <= 1024) distill_rows_kernel<DT, 256, 4, MODE><<<units, 256, lds, stream>>>(a);
    else if (vecs <= 2048) distill_rows_kernel<DT, 512, 4, MODE><<<units, 512, lds, stream>>>(a);
    else if (vecs <= 4096) distill_rows_kernel<DT, 512, 8, MODE><<<units, 512, lds, stream>>>(a);
    else if (vecs <= 8192) distill_rows_kernel<DT, 1024, 8, MODE><<<units, 1024, lds, stream>>>(a);
    else distill_rows_kernel<DT, 1024, 16, MODE><<<units, 1024, lds, stream>>>(a);
}

// ready: the workspace is as a call with the same arguments but for dz and the upstream gradient has left it
template <int DT>
int launch_distill(DistillArgs a, bool ready, hipStream_t stream) {
    constexpr int E = 16 / (int)sizeof(typename Elem<DT>::T);
    if (a.inner > 1) {
        const int tiles = (int)cnm_ceil_div_ll(a.inner, 64);
        const long long blocks = (a.rows / a.inner) * tiles;
        distill_planes_kernel<DT><<<(unsigned)blocks, 256, planes_lds(a.V, a.K), stream>>>(a, tiles);
        CNM_LAUNCH_CHECK();
        return CNM_OK;
    }
    a.seglen = cnm_ceil_div(cnm_ceil_div(a.V, a.segments), E) * E;
    const int cut = a.segments > 1;
    a.segments = cnm_ceil_div(a.V, a.seglen);
    if (!cut) {
        launch_rows<DT, ROW>(a, stream);
        CNM_LAUNCH_CHECK();
        return CNM_OK;
    }
    if (!ready) {
        launch_rows<DT, SEG_STATS>(a, stream);
        CNM_LAUNCH_CHECK();
        distill_join_kernel<DT><<<(unsigned)a.rows, 64, 0, stream>>>(a);
        CNM_LAUNCH_CHECK();
    }
    if (a.dz) {
        launch_rows<DT, SEG_GRAD>(a, stream);
        CNM_LAUNCH_CHECK();
    }
    return CNM_OK;
}

// ------------------------------------------------------------------ top logits
// order-preserving key of a logit: larger value, larger key; NaN above everything, -0 as +0
__device__ inline unsigned key_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    const unsigned u = __float_as_uint(x + 0.f);                         // -0 + 0 = +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A logit and its class as one number, unique within a row: larger logit first, then the lower class.  0 is below all of them.
typedef unsigned long long u64;
__device__ inline u64 rank_of(float x, unsigned v) { return (u64)key_of(x) << 32 | ~v; }

struct TopArgs {
    const void* z; long long ldz;
    float T, c;                              // temperature, log2(e) / T
    void* val; int* idx; float* lse;
    u64* part; float* lpart;                 // [rows][segments][K] ranks and [rows][segments][2] (offset, sum), where a row is split
    long long rows; int V, K; long long inner;
    int segments, seglen;                    // a row's classes by segments of seglen (a multiple of the vector length)
};

// What NT threads that share a row need: a barrier, a histogram, the candidates.
constexpr int CAND = 512;
struct TopShared {
    unsigned hist[256];
    unsigned sel[4];                                                     // digit, rank left within it, its count, output cursor
    float shf[32];
    unsigned nhits;
    int hits[CAND];                                                      // vectors with a number above the bound
    u64 cand[CAND];
};
template <int NT>
__device__ inline void group_sync() {
    if (NT == 64) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup"); __builtin_amdgcn_wave_barrier(); }
    else __syncthreads();
}

// the K-th largest of N numbers per thread (item(i), all distinct but for 0, at least K of them not 0): radix selection, eight bits a round,
// until a digit's numbers all belong
template <int NT, class F>
__device__ __noinline__ u64 kth_largest(F item, int N, int K, int t, TopShared& sh) {
    u64 prefix = 0;
    unsigned left = (unsigned)K;
    for (int shift = 56;; shift -= 8) {
        group_sync<NT>();
        for (int i = t; i < 256; i += NT) sh.hist[i] = 0u;
        group_sync<NT>();
        for (int i = 0; i < N; ++i) {
            const u64 k = item(i);
            if (k && (shift == 56 || (k ^ prefix) >> (shift + 8) == 0)) atomicAdd(&sh.hist[(unsigned)(k >> shift) & 255u], 1u);
        }
        group_sync<NT>();
        if (t < 64) {                                                    // four digits per lane, from the highest down
            unsigned n[4], own = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) { n[j] = sh.hist[255 - (4 * t + j)]; own += n[j]; }
            unsigned before = own;
            for (int d = 1; d < 64; d <<= 1) { const unsigned u = __shfl_up(before, d); if (t >= d) before += u; }
            before -= own;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (before < left && left <= before + n[j]) { sh.sel[0] = 255 - (4 * t + j); sh.sel[1] = left - before; sh.sel[2] = n[j]; }
                before += n[j];
            }
        }
        group_sync<NT>();
        prefix |= (u64)sh.sel[0] << shift; left = sh.sel[1];
        if (sh.sel[2] == left || shift == 0) return prefix;
    }
}

// Of N numbers per thread the K largest, in order, to emit(place, number).  `low`: a lower bound of the K-th largest that keeps the candidates
// few in the ordinary case; where more than CAND pass it (many equal logits), the K-th largest is selected exactly.  pass(put): calls put(number)
// for the thread's numbers that are not below the bound; item(i), i < N: the thread's numbers again, from memory.
template <int NT, class P, class F, class O>
__device__ inline void take_largest(P pass, F item, int N, int K, int t, TopShared& sh, O emit) {
    if (t == 0) sh.sel[3] = 0u;
    group_sync<NT>();
    pass([&](u64 k) { const unsigned at = atomicAdd(&sh.sel[3], 1u); if (at < CAND) sh.cand[at] = k; });
    group_sync<NT>();
    int C = (int)sh.sel[3];
    if (C > CAND) {
        const u64 least = kth_largest<NT>(item, N, K, t, sh);
        group_sync<NT>();
        if (t == 0) sh.sel[3] = 0u;
        group_sync<NT>();
        for (int i = 0; i < N; ++i) { const u64 k = item(i); if (k && k >= least) sh.cand[atomicAdd(&sh.sel[3], 1u)] = k; }   // exactly K
        group_sync<NT>();
        C = K;
    }
    for (int i = t; i < C; i += NT) {                                    // a candidate's place is the number of those above it
        const u64 mine = sh.cand[i];
        int place = 0;
        for (int j = 0; j < C; ++j) place += sh.cand[j] > mine;
        if (place < K) emit(place, mine);
    }
}

// a lower bound of the K-th largest of the NT threads' numbers: every wave's r-th largest, r = K / waves rounded up, the smallest of these
template <int NT>
__device__ inline float kth_bound(float m, int K, float* sh) {
    constexpr int W = NT / 64;
    const int r = (K + W - 1) / W;
    const float ninf = -__builtin_huge_valf();
    if (r > 64) return ninf;
    const int lane = threadIdx.x & 63;
    // the wave's numbers in order (bitonic, descending: 21 exchanges), or for the first of them six exchanges
    if (r == 1) m = max_wave(m);
    else {
#pragma unroll
        for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
            for (int d = size >> 1; d; d >>= 1) {
                const float other = __shfl_xor(m, d);
                const bool upper = (lane & d) == 0, down = (lane & size) == 0;   // the lane that keeps the larger one
                m = upper == down ? fmaxf(m, other) : fminf(m, other);
            }
    }
    float w = __shfl(m, r - 1);
    if (NT == 64) return w;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = w;
    __syncthreads();
    w = sh[0];
    for (int i = 1; i < W; ++i) w = fminf(w, sh[i]);
    return w;
}

// NT threads per row or segment of a row, which they hold in registers (NV vectors of 16 bytes each), read once.  Log-sum-exp, then a lower bound of
// the K-th largest logit from the threads' own maxima, the few logits above it to LDS, and their order by counting.
// bf16 4096 x 32768, 32 entries: 57 us (4.7 TB/s, what a large copy reaches); one row of 131072 in segments 9 us, their join 7: latency.
template <int DT, int NT, int NV>
__global__ __launch_bounds__(NT == 64 ? 256 : NT, NT == 256 && NV == 16 ? 4 : 1) void top_rows_kernel(const TopArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int E = 16 / sizeof(T), RPB = NT == 64 ? 4 : 1;
    __shared__ TopShared shared[RPB];
    const int sub = NT == 64 ? threadIdx.x >> 6 : 0, t = NT == 64 ? threadIdx.x & 63 : threadIdx.x;
    TopShared& sh = shared[sub];
    const long long unit = (long long)blockIdx.x * RPB + sub;            // row and segment
    if (unit >= a.rows * a.segments) return;                             // (whole waves only: NT == 64)
    const long long r = unit / a.segments;
    const int seg = (int)(unit - r * a.segments), v0 = seg * a.seglen, n = min(a.V - v0, a.seglen);
    const T* z = static_cast<const T*>(a.z) + (size_t)r * a.ldz + v0;
    const float c = a.c, ninf = -__builtin_huge_valf();
    Raw<DT> x[NV];
    float m = ninf;
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i].load(z, (i * NT + t) * E, n);
    float vm[NV];                                                        // the vectors' largest
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        x[i].hold();
        vm[i] = x[i].get(0);
#pragma unroll
        for (int j = 1; j < E; ++j) vm[i] = fmaxf(vm[i], x[i].get(j));
        m = fmaxf(m, vm[i]);
    }
    const float o = finite_or_0(m);
    Lse l = {m, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        x[i].hold();
#pragma unroll
        for (int j = 0; j < E; ++j) l.s += exp2_((x[i].get(j) - o) * c);
    }
    const bool odd = l.s != l.s;                                         // a NaN here: every vector is looked at
    l = lse_block<NT>(l, c, sh.shf);
    const float low = kth_bound<NT>(m, a.K, sh.shf);
    if (a.segments == 1) { if (t == 0) a.lse[r] = lse_value(l, a.T); }
    else if (t == 0) { a.lpart[2 * unit] = l.o; a.lpart[2 * unit + 1] = l.s; }
    // few lanes of a wave hold a vector with a logit above the bound: those vectors are listed, and looked at side by side
    const auto pass = [&](auto put) {
        if (t == 0) sh.nhits = 0u;
        group_sync<NT>();
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (odd || vm[i] >= low) { const unsigned h = atomicAdd(&sh.nhits, 1u); if (h < CAND) sh.hits[h] = i * NT + t; }
        group_sync<NT>();
        const unsigned H = sh.nhits;
        if (H > CAND) { if (t == 0) sh.sel[3] = CAND + 1; return; }       // too many: the exact selection
        for (unsigned h = t; h < H; h += NT) {
            const int at = sh.hits[h] * E;
            Raw<DT> y;
            y.load(z, at, n);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const float v = y.get(j);
                if (!(v < low) && at + j < n) put(rank_of(v, (unsigned)(v0 + at + j)));
            }
        }
    };
    const auto item = [=](int i) -> u64 { const int at = i * NT + t; return at < n ? rank_of((float)z[at], (unsigned)(v0 + at)) : 0ull; };
    const int K = min(a.K, n), N = (n + NT - 1) / NT;
    if (a.segments == 1)
        take_largest<NT>(pass, item, N, K, t, sh, [&](int place, u64 k) {
            const unsigned v = ~(unsigned)k;
            a.idx[(size_t)r * a.K + place] = (int)v;
            static_cast<T*>(a.val)[(size_t)r * a.K + place] = z[v];
        });
    else {
        take_largest<NT>(pass, item, N, K, t, sh, [&](int place, u64 k) { a.part[(size_t)unit * a.K + place] = k; });
        for (int i = K + t; i < a.K; i += NT) a.part[(size_t)unit * a.K + i] = 0ull;
    }
}

// joins a row's segments: N ranks per thread
template <int DT, int N>
__global__ __launch_bounds__(1024) void top_join_kernel(const TopArgs a) {
    typedef typename Elem<DT>::T T;
    __shared__ TopShared sh;
    const int t = threadIdx.x;
    const long long r = blockIdx.x;
    const int total = a.segments * a.K;
    const float c = a.c, ninf = -__builtin_huge_valf();
    u64 k[N];
    float m = ninf;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int at = i * 1024 + t;
        k[i] = at < total ? a.part[(size_t)r * total + at] : 0ull;
    }
    const auto value = [](u64 k) {                                       // key_of's inverse (NaN for NaN)
        const unsigned u = (unsigned)(k >> 32);
        return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
    };
#pragma unroll
    for (int i = 0; i < N; ++i) if (k[i]) m = fmaxf(m, value(k[i]));
    Lse l = {ninf, 0.f};
    if (t < a.segments) l = {a.lpart[2 * (r * a.segments + t)], a.lpart[2 * (r * a.segments + t) + 1]};
    l = lse_block<1024>(l, c, sh.shf);
    if (t == 0) a.lse[r] = lse_value(l, a.T);
    const float low = kth_bound<1024>(m, a.K, sh.shf);
    const T* z = static_cast<const T*>(a.z) + (size_t)r * a.ldz;
    const u64* const part = a.part + (size_t)r * total;
    take_largest<1024>([&](auto put) {
#pragma unroll
        for (int i = 0; i < N; ++i) if (k[i] && !(value(k[i]) < low)) put(k[i]);
    }, [=](int i) -> u64 { return i * 1024 + t < total ? part[i * 1024 + t] : 0ull; }, (total + 1023) / 1024, a.K, t, sh, [&](int place, u64 q) {
        const unsigned v = ~(unsigned)q;
        a.idx[(size_t)r * a.K + place] = (int)v;
        static_cast<T*>(a.val)[(size_t)r * a.K + place] = z[v];
    });
}

// Classes in the middle, [outer][V][inner]: a lane per position keeps the KM largest of what it has seen, in order, in registers.  Classes come
// in ascending order, so "strictly larger" keeps the lowest of equals in front.  Sixteen classes are requested ahead of their use.
// fp32 [4, 64, 192, 256], 8 entries: 27 us (2.4 TB/s), bound by vector issue: 56 instructions per class and pixel, 40 of them keep the order.
template <int DT, int KM>
__global__ __launch_bounds__(256) void top_planes_kernel(const TopArgs a) {
    typedef typename Elem<DT>::T T;
    constexpr int AHEAD = 16;
    const long long r = (long long)blockIdx.x * 256 + threadIdx.x;
    if (r >= a.rows) return;
    const long long ob = r / a.inner, at = r % a.inner;
    const T* z = static_cast<const T*>(a.z) + (size_t)ob * a.V * a.inner + at;
    const float c = a.c, ninf = -__builtin_huge_valf();
    unsigned key[KM];                                                    // 0 is below every key
    int cls[KM];
#pragma unroll
    for (int i = 0; i < KM; ++i) { key[i] = 0u; cls[i] = 0; }
    Run run;
    T next[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) next[j] = z[(size_t)min(j, a.V - 1) * a.inner];
    for (int v0 = 0; v0 < a.V; v0 += AHEAD) {
        float x[AHEAD], m = ninf;
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            x[j] = v0 + j < a.V ? (float)next[j] : ninf;
            m = fmaxf(m, x[j]);
        }
        if (v0 + AHEAD < a.V) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) next[j] = z[(size_t)min(v0 + AHEAD + j, a.V - 1) * a.inner];
        }
        if (m > run.m) run.raise(m, c);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            run.s += exp2_((x[j] - run.o) * c);
            const unsigned k = key_of(x[j]);
            const int v = v0 + j;
            if (v < a.V && k > key[KM - 1]) {                            // from the last place up: a place takes its upper neighbour if k goes above that, k if it goes here
#pragma unroll
                for (int i = KM - 1; i > 0; --i) {
                    cls[i] = k > key[i - 1] ? cls[i - 1] : k > key[i] ? v : cls[i];
                    key[i] = k > key[i - 1] ? key[i - 1] : k > key[i] ? k : key[i];
                }
                cls[0] = k > key[0] ? v : cls[0];
                key[0] = k > key[0] ? k : key[0];
            }
        }
    }
    const Lse l = run.lse();
    a.lse[r] = lse_value(l, a.T);
    const size_t base = (size_t)ob * a.K * a.inner + at;
#pragma unroll
    for (int i = 0; i < KM; ++i)
        if (i < a.K) {
            a.idx[base + (size_t)i * a.inner] = cls[i];
            static_cast<T*>(a.val)[base + (size_t)i * a.inner] = z[(size_t)cls[i] * a.inner];
        }
}

constexpr int TOP_PLANES_KMAX = 16;

// How rows are split: a workgroup of 512 threads holds 64 KB of a row; rows that are longer, or so few that they would leave most CUs idle,
// are cut into segments (at least 4 KB each) and joined by a second launch.
int top_segments(long long rows, int V, int K, int esize) {
    const int most = 512 * 8 * 16 / esize, least = cnm_ceil_div(V, most);
    if ((size_t)V * esize <= 8192 || rows >= 128) return least;
    int want = (int)(256 / rows);
    const int fit = (int)((size_t)V * esize / 4096), few = 2048 / K;     // (few: what is left to join is one number or two per thread)
    want = want < fit ? want : fit;
    want = want < few ? want : few;
    return want > least ? want : least;
}

template <int DT>
int launch_top(TopArgs a, hipStream_t stream) {
    typedef typename Elem<DT>::T T;
    constexpr int E = 16 / sizeof(T);
    if (a.inner > 1) {
        const unsigned blocks = (unsigned)cnm_ceil_div_ll(a.rows, 256);
        if (a.K <= 4) top_planes_kernel<DT, 4><<<blocks, 256, 0, stream>>>(a);
        else if (a.K <= 8) top_planes_kernel<DT, 8><<<blocks, 256, 0, stream>>>(a);
        else top_planes_kernel<DT, 16><<<blocks, 256, 0, stream>>>(a);
        CNM_LAUNCH_CHECK();
        return CNM_OK;
    }
    a.segments = top_segments(a.rows, a.V, a.K, (int)sizeof(T));
    a.seglen = cnm_ceil_div(cnm_ceil_div(a.V, a.segments), E) * E;
    a.segments = cnm_ceil_div(a.V, a.seglen);
    const int vecs = a.seglen / E;
    const unsigned units = (unsigned)(a.rows * a.segments);
    if (vecs <= 64) top_rows_kernel<DT, 64, 1><<<cnm_ceil_div((int)units, 4), 256, 0, stream>>>(a);
    else if (vecs <= 256) top_rows_kernel<DT, 256, 1><<<units, 256, 0, stream>>>(a);
    else if (vecs <= 512) top_rows_kernel<DT, 512, 1><<<units, 512, 0, stream>>>(a);
    else if (vecs <= 1024) top_rows_kernel<DT, 512, 2><<<units, 512, 0, stream>>>(a);
    else if (vecs <= 2048) top_rows_kernel<DT, 512, 4><<<units, 512, 0, stream>>>(a);
    else top_rows_kernel<DT, 256, 16><<<units, 256, 0, stream>>>(a);
    CNM_LAUNCH_CHECK();
    if (a.segments > 1) {
        const int total = a.segments * a.K;
        if (total <= 2048) top_join_kernel<DT, 2><<<(unsigned)a.rows, 1024, 0, stream>>>(a);
        else top_join_kernel<DT, 16><<<(unsigned)a.rows, 1024, 0, stream>>>(a);
        CNM_LAUNCH_CHECK();
    }
    return CNM_OK;
}

}  // namespace

extern "C" int cnm_top_logits_planes_max_entries(void) { return TOP_PLANES_KMAX; }
extern "C" int cnm_distill_max_entries(void) { return KMAX; }
extern "C" int cnm_distill_max_classes(void) { return VMAX; }
extern "C" int cnm_distill_planes_ok(int classes, int entries) { return classes > 0 && entries > 0 && entries <= KMAX && classes <= VMAX && planes_lds(classes, entries) <= LDS_BYTES; }

extern "C" size_t cnm_top_logits_workspace_bytes(int dtype, long long rows, int classes, int entries, long long inner) {
    if (rows <= 0 || classes <= 0 || entries <= 0 || inner != 1 || dtype < CNM_F32 || dtype > CNM_BF16) return 0;
    const int seg = top_segments(rows, classes, entries, dtype == CNM_F32 ? 4 : 2);
    return seg > 1 ? (size_t)rows * seg * ((size_t)entries * sizeof(u64) + 2 * sizeof(float)) : 0;
}

extern "C" int cnm_top_logits(const void* z, int dtype, long long ldz, float temperature, void* values, int* indices, float* lse, void* workspace, size_t workspace_bytes,
                              long long rows, int classes, int entries, long long inner, void* stream) {
    CNM_REQUIRE(z && values && indices && lse && rows > 0 && classes > 0 && inner > 0 && temperature >= TMIN && temperature < __builtin_huge_valf(), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(entries > 0 && entries <= classes && entries <= (inner > 1 ? TOP_PLANES_KMAX : KMAX) && rows % inner == 0 && (inner > 1 || ldz >= classes), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(dtype >= CNM_F32 && dtype <= CNM_BF16, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(rows < (1ll << 30) && classes <= VMAX, CNM_ERR_BAD_SHAPE);
    const int E = dtype == CNM_F32 ? 4 : 8, cut = inner > 1 ? 1 : top_segments(rows, classes, entries, 16 / E);
    CNM_REQUIRE(inner > 1 || launch_fits(rows * cut, top_threads(cnm_ceil_div(cnm_ceil_div(classes, cut), E))), CNM_ERR_BAD_SHAPE);
    const size_t need = cnm_top_logits_workspace_bytes(dtype, rows, classes, entries, inner);
    CNM_REQUIRE(!need || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 7) == 0), CNM_ERR_WORKSPACE);
    u64* const part = static_cast<u64*>(workspace);
    float* const lpart = need ? reinterpret_cast<float*>(part + (need - (size_t)2 * sizeof(float) * (need / ((size_t)entries * sizeof(u64) + 2 * sizeof(float)))) / sizeof(u64)) : nullptr;
    const TopArgs a = {z, ldz, temperature, (float)(LOG2E_D / (double)temperature), values, indices, lse, part, lpart, rows, classes, entries, inner, 1, 0};
    switch (dtype) {
        case CNM_F32: return launch_top<CNM_F32>(a, cnm_stream(stream));
        case CNM_F16: return launch_top<CNM_F16>(a, cnm_stream(stream));
        case CNM_BF16: return launch_top<CNM_BF16>(a, cnm_stream(stream));
    }
    return CNM_ERR_BAD_ARG;
}

// workspace: the weights' partial sums, the losses', and for rows cut into segments the rows' numbers and the segments'
extern "C" size_t cnm_distill_workspace_doubles(int dtype, long long rows, int classes, long long inner) {
    if (rows <= 0 || classes <= 0 || inner <= 0 || rows % inner || dtype < CNM_F32 || dtype > CNM_BF16) return 0;
    if (inner > 1) return (size_t)WPARTS + (size_t)(rows / inner) * (size_t)cnm_ceil_div_ll(inner, 64);
    const int seg = distill_segments(rows, classes, dtype == CNM_F32 ? 4 : 2);
    return (size_t)WPARTS + (size_t)rows + (seg > 1 ? (size_t)rows * (sizeof(DistillRow) / sizeof(double) + (size_t)seg) : 0);
}

extern "C" int cnm_distill(const void* z, int dtype, long long ldz, const void* indices, int wide_indices, const void* entry_logits, int entry_dtype,
                           const float* teacher_lse, float temperature, const float* weight, const float* grad_out, int grad_out_rows, int skip_if_one,
                           int reduction, float* loss, void* dz, double* workspace, size_t workspace_doubles, int workspace_ready,
                           long long rows, int classes, int entries, long long inner, void* stream) {
    CNM_REQUIRE(z && indices && entry_logits && rows > 0 && classes > 0 && entries > 0 && inner > 0 && (loss || dz), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(temperature >= TMIN && temperature < __builtin_huge_valf() && reduction >= 0 && reduction <= 2 && entries <= KMAX, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(rows % inner == 0 && (inner > 1 || ldz >= classes) && dtype >= CNM_F32 && dtype <= CNM_BF16 && entry_dtype >= CNM_F32 && entry_dtype <= CNM_BF16, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(!grad_out_rows || (grad_out && reduction == 0), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(!workspace_ready || !loss, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(rows < (1ll << 30) && classes <= VMAX && (inner == 1 || cnm_distill_planes_ok(classes, entries)), CNM_ERR_BAD_SHAPE);
    const int seg = inner > 1 ? 1 : distill_segments(rows, classes, dtype == CNM_F32 ? 4 : 2);
    const int E = dtype == CNM_F32 ? 4 : 8;
    const long long tiles = inner > 1 ? (rows / inner) * cnm_ceil_div_ll(inner, 64) : 0;
    CNM_REQUIRE(inner > 1 ? launch_fits(tiles, 256) : launch_fits(rows * seg, distill_threads(cnm_ceil_div(cnm_ceil_div(classes, seg), E))), CNM_ERR_BAD_SHAPE);
    CNM_REQUIRE(workspace && workspace_doubles >= cnm_distill_workspace_doubles(dtype, rows, classes, inner), CNM_ERR_WORKSPACE);
    const hipStream_t st = cnm_stream(stream);
    const bool mean = reduction == 1;
    double* const wpart = workspace;
    double* const lpart = workspace + WPARTS;
    const long long parts = inner > 1 ? tiles : rows;
    DistillRow* const rec = seg > 1 ? reinterpret_cast<DistillRow*>(lpart + parts) : nullptr;
    float* const segs = seg > 1 ? reinterpret_cast<float*>(rec + rows) : nullptr;
    const int nw = mean && weight ? (int)(cnm_ceil_div_ll(rows, 4096) < WPARTS ? cnm_ceil_div_ll(rows, 4096) : WPARTS) : 0;
    if (nw && !workspace_ready) { weight_parts_kernel<<<nw, 1024, 0, st>>>(weight, rows, wpart); CNM_LAUNCH_CHECK(); }
    const double inv_norm = mean && !weight ? 1.0 / (double)rows : 1.0;
    const bool total = reduction != 0 && loss;
    const DistillArgs a = {z, ldz, indices, wide_indices, entry_logits, entry_dtype, teacher_lse, temperature, (float)(LOG2E_D / (double)temperature), 1.0 / (double)temperature, LOG2E_D / (double)temperature, weight, nw ? wpart : nullptr, nw, inv_norm,
                           grad_out, grad_out_rows, skip_if_one, total ? nullptr : loss, total ? lpart : nullptr, dz, rows, classes, entries, inner, rec, segs, seg, 0};
    int rc = CNM_ERR_BAD_ARG;
    switch (dtype) {
        case CNM_F32: rc = launch_distill<CNM_F32>(a, workspace_ready != 0, st); break;
        case CNM_F16: rc = launch_distill<CNM_F16>(a, workspace_ready != 0, st); break;
        case CNM_BF16: rc = launch_distill<CNM_BF16>(a, workspace_ready != 0, st); break;
    }
    if (rc != CNM_OK || !total) return rc;
    loss_total_kernel<<<1, 1024, 0, st>>>(lpart, parts, nw ? wpart : nullptr, nw, inv_norm, loss);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}
