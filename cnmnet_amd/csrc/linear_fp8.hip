// 8-bit floating-point linear layer: block quantisation and the block-scaled product.
//
// Format.  A block of 128 values along the reduced axis (activations, gradients: 1 x 128; weights: 128 x 128) is held as e4m3 values q
// and ONE power of two 2^e, stored as the byte e + 127:
//     e = the smallest integer >= -127 with max |x| <= 448 * 2^e over the block's finite values,   q = e4m3(x * 2^-e), ties to even.
// The scale is a power of two by choice: x * 2^-e is exact, so the only rounding is the one to e4m3 (at most 2^-4 relative in its normal
// range) and every implementation of the definition gives the same bits; and the matrix instruction takes such a byte per 32 values of
// its reduced axis, so a block's scale costs no vector arithmetic: the accumulators stay in the matrix pipe over the whole reduction.
// inf and NaN become e4m3's NaN (they stay visible in the product); they do not take part in the block's maximum.
// The reduced axis is padded with zeros to a multiple of 128: no kernel below has a tail along it.
//
// Product.  c[m][n] = sum_kb 2^(ea[m][kb] + eb[n][kb]) sum_{k in kb} qa[m][k] qb[n][k], accumulated in fp32 by the matrix pipe, rounded once
// to the output type.  Both operands are [rows][K] with K contiguous ("NT"); the second one's scales are per row or per 128 rows.
//
// Two ways through the matrix pipe, by the type of the result.
//   16-bit results: v_mfma_scale_f32_32x32x64_f8f6f4 (tiles; 16x16x128 where rows are few) on the bytes as they are, twice the bf16 rate.  Its accumulator is fp32, but it adds
//     eight consecutive products at a time, each cut off at 2^-13 of the eight's largest exponent (measured: probes of single terms; rms
//     1.5e-5 of the result on normal data): a choice for results that are rounded to 2^-9 or 2^-12 anyway.
//   fp32 results: the bytes become bf16 with their scale applied (exact within bf16's exponent range) and v_mfma_f32_32x32x16_bf16 (16x16x32) adds them:
//     rms 1e-8 of the result, as fp32 sums are.  Below a block exponent of -117 an e4m3 value's low bits fall under bf16's normal range and are lost.
#include "cnm_common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr int QB = 128;                      // values per block

template <int DT> struct Elem;               // CNM_F32 / CNM_F16 / CNM_BF16: load to float, store from float (round to nearest, ties to even)
template <> struct Elem<CNM_F32> { typedef float T; static __device__ float up(float v) { return v; } static __device__ float down(float v) { return v; } };
template <> struct Elem<CNM_F16> { typedef _Float16 T; static __device__ float up(_Float16 v) { return (float)v; } static __device__ _Float16 down(float v) { return (_Float16)v; } };
template <> struct Elem<CNM_BF16> { typedef __bf16 T; static __device__ float up(__bf16 v) { return (float)v; } static __device__ __bf16 down(float v) { return (__bf16)v; } };

// byte e + 127 of a block whose largest finite magnitude is amax: 448 = 1.75 * 2^8, so the exponent of amax, minus 8, plus one if the
// fraction is above 0.75 -- integer arithmetic on the bits (adding 0x1FFFFF carries into the exponent exactly then)
__device__ inline int scale_byte(float amax) {
    const int e = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8;
    return e < 0 ? 0 : e;                                                // subnormal amax has exponent field 0: 2^-127 holds it as well
}
__device__ inline float inv_scale(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }   // 2^-(byte - 127), byte 0 .. 247

__device__ inline float finite_abs(float v) { const float a = fabsf(v); return a < __builtin_huge_valf() ? a : 0.f; }   // (NaN compares false)

// four values -> four e4m3 bytes; |v| <= 448 but for non-finite inputs, which the instruction turns into NaN (its overflow mode is off)
__device__ inline unsigned pack4(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
}

// eight consecutive values of a row, zero beyond `have` (16-byte loads whatever the row's alignment: global memory takes them)
template <int DT>
__device__ inline void load8(const typename Elem<DT>::T* p, int have, float v[8]) {
    typedef typename Elem<DT>::T T;
    if (have >= 8) {
        T a[8];
        __builtin_memcpy(a, p, sizeof(a));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = Elem<DT>::up(a[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < have ? Elem<DT>::up(p[j]) : 0.f;
    }
}

// One workgroup quantises a 128 x 128 tile, read once: 16 lanes per row (8 values each), a thread's four rows consecutive, so that the
// transposed copy leaves as 4-byte columns through LDS.  Row form: q [R][Cp], s [R][Cp/128] (BLK = false) or s [R/128][Cp/128] (BLK = true).
// Transposed form (optional): qt [C][Rp], blocked along R: st [C][Rp/128], or the same 128 x 128 block's byte at st [C/128][Rp/128].
// Bound by memory: bf16 8192 x 8192 without the transposed form 51 us (4.0 TB/s of read and written bytes, a large copy 4.6), 8192 x 4096
// with it 45 us (3.0 TB/s: 128-byte pieces of 128 transposed rows per workgroup; through a tile without the chunk permutation 50).
template <int DT, bool BLK>
__global__ __launch_bounds__(512) void quantize_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx, int R, int C, int Cb, int Rb,
                                                       unsigned char* __restrict__ q, unsigned char* __restrict__ s,
                                                       unsigned char* __restrict__ qt, unsigned char* __restrict__ st) {
    constexpr int NR = 4;                                                // rows per thread
    __shared__ float cmax[8][QB];
    __shared__ __attribute__((aligned(16))) unsigned char tile[QB][QB];  // transposed; a row's 16-byte chunks permuted by (row >> 3) & 7: the rows that a wave writes at once are multiples of eight apart
    __shared__ float bmax[8];
    const int tid = threadIdx.x, lc = tid & 15, lr = tid >> 4;
    const int cb = blockIdx.x % Cb, rb = blockIdx.x / Cb;
    const int c0 = cb * QB + lc * 8, r0 = rb * QB + lr * NR;
    float v[NR][8];
#pragma unroll
    for (int p = 0; p < NR; ++p) {
        const int r = r0 + p;
        load8<DT>(x + (size_t)(r < R ? r : 0) * ldx + (c0 < C ? c0 : 0), r < R ? C - c0 : 0, v[p]);
    }
    int byte[NR];
    float am[NR];
#pragma unroll
    for (int p = 0; p < NR; ++p) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[p][j]));
        for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        am[p] = m;
    }
    if (BLK) {
        float m = 0.f;
#pragma unroll
        for (int p = 0; p < NR; ++p) m = fmaxf(m, am[p]);
        m = fmaxf(m, __shfl_xor(m, 16)); m = fmaxf(m, __shfl_xor(m, 32));
        if ((tid & 63) == 0) bmax[tid >> 6] = m;
        __syncthreads();
        m = bmax[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, bmax[i]);
#pragma unroll
        for (int p = 0; p < NR; ++p) byte[p] = scale_byte(m);
        if (tid == 0) {
            if (s) s[(size_t)rb * Cb + cb] = (unsigned char)byte[0];
            if (st) st[(size_t)cb * Rb + rb] = (unsigned char)byte[0];
        }
    } else {
#pragma unroll
        for (int p = 0; p < NR; ++p) {
            byte[p] = scale_byte(am[p]);
            if (s && lc == 0 && r0 + p < R) s[(size_t)(r0 + p) * Cb + cb] = (unsigned char)byte[p];
        }
    }
    if (q) {
#pragma unroll
        for (int p = 0; p < NR; ++p) {
            if (r0 + p < R) {
                const float k = inv_scale(byte[p]);
                uint2 u;
                u.x = pack4(v[p][0] * k, v[p][1] * k, v[p][2] * k, v[p][3] * k);
                u.y = pack4(v[p][4] * k, v[p][5] * k, v[p][6] * k, v[p][7] * k);
                *reinterpret_cast<uint2*>(q + (size_t)(r0 + p) * ((size_t)Cb * QB) + c0) = u;
            }
        }
    }
    if (!qt) return;
    float k8[8];
    if (!BLK) {                                                          // the transposed rows' own maxima: over this tile's 128 rows
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = 0.f;
#pragma unroll
            for (int p = 0; p < NR; ++p) m = fmaxf(m, finite_abs(v[p][j]));
            m = fmaxf(m, __shfl_xor(m, 16)); m = fmaxf(m, __shfl_xor(m, 32));
            if ((tid & 63) < 16) cmax[tid >> 6][lc * 8 + j] = m;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = cmax[0][lc * 8 + j];
#pragma unroll
            for (int g = 1; g < 8; ++g) m = fmaxf(m, cmax[g][lc * 8 + j]);
            const int b = scale_byte(m);
            k8[j] = inv_scale(b);
            if (lr == 0 && c0 + j < C) st[(size_t)(c0 + j) * Rb + rb] = (unsigned char)b;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) k8[j] = inv_scale(byte[0]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        *reinterpret_cast<unsigned*>(&tile[lc * 8 + j][(lr * NR) ^ (16 * (lc & 7))]) = pack4(v[0][j] * k8[j], v[1][j] * k8[j], v[2][j] * k8[j], v[3][j] * k8[j]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {                                        // 8 lanes x 16 bytes = one transposed row of the tile
        const int c = i * 64 + (tid >> 3), l = tid & 7;
        if (cb * QB + c < C)
            *reinterpret_cast<uint4*>(qt + (size_t)(cb * QB + c) * ((size_t)Rb * QB) + (size_t)rb * QB + l * 16) = *reinterpret_cast<const uint4*>(&tile[c][16 * (l ^ ((c >> 3) & 7))]);
    }
}

template <int DT, bool BLK>
int launch_quantize(const void* x, long long ldx, int R, int C, void* q, void* s, void* qt, void* st, hipStream_t stream) {
    typedef typename Elem<DT>::T T;
    const int Cb = cnm_ceil_div(C, QB), Rb = cnm_ceil_div(R, QB);
    auto* xp = static_cast<const T*>(x);
    auto* qp = static_cast<unsigned char*>(q); auto* sp = static_cast<unsigned char*>(s);
    auto* qtp = static_cast<unsigned char*>(qt); auto* stp = static_cast<unsigned char*>(st);
    quantize_kernel<DT, BLK><<<Cb * Rb, 512, 0, stream>>>(xp, ldx, R, C, Cb, Rb, qp, sp, qtp, stp);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

// ------------------------------------------------------------------ product
// eight e4m3 bytes times 2^(byte - 127) -> bf16
__device__ inline bf16x8 widen(int lo, int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ inline float scale_float(unsigned word, int shift) { return __uint_as_float((word >> shift & 255u) << 23); }   // only its exponent field is used

struct MatArgs {
    const unsigned char *a, *sa, *b, *sb;    // a [M][K], b [N][K] e4m3; sa [M][K/128]; sb [N >> bshift][K/128]
    void* c;                                 // [M][ldc]
    int M, N, Kb, bshift;
    long long ldc;
    int tiles_m, tiles_n;
    int splits, chunk;                       // SPLIT: ranges of `chunk` blocks (a multiple of four) along the reduced axis, c = [splits][M][N] fp32
};

// Tiles in an order that keeps neighbours on one XCD near each other: workgroups are dealt to XCDs in contiguous ranges (xcd_remap), and a
// range walks bands of four tile rows, column by column, so that the 32 CUs of an XCD share four row blocks and eight column blocks in its L2.
__device__ inline void tile_of(int id, const MatArgs& g, int& tm, int& tn) {
    const int band = id / (4 * g.tiles_n), in = id - band * 4 * g.tiles_n;
    const int rows = min(4, g.tiles_m - 4 * band);
    tm = 4 * band + in % rows; tn = in / rows;
}

// TM x TN outputs per workgroup, WM x WN waves, each IM x IN tiles of 32 x 32.  The reduced axis goes by in half blocks of 64: both operands' rows
// (64 bytes each) come to LDS by DMA, a ring of four half blocks, three ahead of their use; a wave reads the fragments of the next half block
// under the matrix instructions of this one (two register sets).  One barrier per half block, behind a counted vmcnt: two half blocks stay
// in flight across it.
// LDS: row r at r * 64, its four 16-byte chunks permuted by (r >> 2) & 3: the 16 rows that a fragment read touches at one chunk then fall on
// all 64 banks.  The DMA writes 64 lanes x 16 bytes in order, so the permutation is in the lanes' source addresses.
// Scale bytes: rows of SC blocks in LDS, refilled every SC blocks; a lane reads four blocks' bytes as one word.
// The weight is the instruction's first operand: a lane then holds outputs of one row, in fours.
// 8192 x 8192 x 8192, bf16 results, one launch after another: 408 to 430 us from card to card, 2.6 to 2.7 PF (a library product of plain bytes 2.6),
// held back by the package's power limit (under a profiler's kernel trace 513 us); 8192 x 4096 x 4096: 110 us back to back (2.5 PF), 125 to 136 between
// the quantisations of a training step, of which 9 us per tile are its first loads and its stores.  fp32 results: 4096^3 122 us (1.1 PF), 8192^3 870
// (1.26 PF): half the instruction rate, and the conversions.
// The order within a half block: its NM matrix instructions start at once, the next fragments' ND reads and the NV DMA instructions go evenly
// between them (left alone, the scheduler puts all of these in front, or the matrix instructions of two half blocks behind one barrier).
template <int I, int NM, int ND, int NV>
struct Interleave {
    static __device__ __forceinline__ void go() {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if constexpr (ND * (I + 1) / NM > ND * I / NM) __builtin_amdgcn_sched_group_barrier(0x100, ND * (I + 1) / NM - ND * I / NM, 0);
        if constexpr (NV * (I + 1) / NM > NV * I / NM) __builtin_amdgcn_sched_group_barrier(0x010, NV * (I + 1) / NM - NV * I / NM, 0);
        if constexpr (I + 1 < NM) Interleave<I + 1, NM, ND, NV>::go();
    }
};

template <int TM, int TN, int WM, int WN, int DT, bool BLK>
struct Mat {
    static constexpr int NW = WM * WN, NT = NW * 64, IM = TM / WM / 32, IN = TN / WN / 32, NST = 4;
    static constexpr int STAGE = (TM + TN) * 64, PA = TM / 16 / NW, PB = TN / 16 / NW, DMA = PA + PB;   // DMA instructions per wave and half block: 16 rows each
    static constexpr int SC = BLK ? 64 : 32, SROW = SC + 4, BROWS = BLK ? TN / QB : TN;                 // scale rows: four bytes apart from a power of two
    static constexpr int LDS = NST * STAGE + (TM + BROWS) * SROW;
    static_assert(TM % (16 * NW) == 0 && TN % (16 * NW) == 0 && LDS <= 160 * 1024 && (!BLK || (TN % QB == 0 && TN / WN <= QB)), "tile");
};

template <int TM, int TN, int WM, int WN, int DT, bool BLK, bool SPLIT>
__global__ __launch_bounds__(WM * WN * 64) void matmul_fp8_kernel(const MatArgs g) {
    typedef Mat<TM, TN, WM, WN, DT, BLK> C;
    constexpr int IM = C::IM, IN = C::IN;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char* const sca = smem + C::NST * C::STAGE;
    char* const scb = sca + TM * C::SROW;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN;
    int tm, tn;
    const int id = xcd_remap(blockIdx.x, gridDim.x), split = SPLIT ? id / (g.tiles_m * g.tiles_n) : 0;
    tile_of(SPLIT ? id - split * g.tiles_m * g.tiles_n : id, g, tm, tn);
    const int m0 = tm * TM, n0 = tn * TN, Kb = g.Kb, K = Kb * QB;
    // buffer ranges that end with the operands' last rows: beyond them the DMA writes zeros
    const unsigned bytes_a = (unsigned)min(g.M - m0, TM) * (unsigned)K, bytes_b = (unsigned)min(g.N - n0, TN) * (unsigned)K;
    const int kb0 = SPLIT ? split * g.chunk : 0, kb1 = SPLIT ? min(Kb, kb0 + g.chunk) : Kb, S = 2 * kb1;
    const unsigned chunk = (unsigned)((lane & 3) ^ ((lane >> 4) & 3)) * 16u;
    const unsigned va = (unsigned)(wave * C::PA * 16 + (lane >> 2)) * (unsigned)K + chunk, vb = (unsigned)(wave * C::PB * 16 + (lane >> 2)) * (unsigned)K + chunk;
    auto issue = [&](int s) {                                            // half block s into its place in the ring; beyond the last one an empty range: zeros, no traffic, the same count
        const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(g.a) + (size_t)m0 * K, 0, s < S ? bytes_a : 0u, 0x00020000);
        const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(g.b) + (size_t)n0 * K, 0, s < S ? bytes_b : 0u, 0x00020000);
        char* const dst = smem + (s & (C::NST - 1)) * C::STAGE;
#pragma unroll
        for (int p = 0; p < C::PA; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)(dst + (wave * C::PA + p) * 1024), 16, va + (unsigned)p * 16u * (unsigned)K, s * 64, 0, 0);
#pragma unroll
        for (int p = 0; p < C::PB; ++p)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)(dst + TM * 64 + (wave * C::PB + p) * 1024), 16, vb + (unsigned)p * 16u * (unsigned)K, s * 64, 0, 0);
    };
    // scale bytes of blocks kb .. kb + SC - 1: 16 at a time, never beyond the arrays
    auto fill = [&](char* dst, const unsigned char* s, int row0, int rows, int last, int kb) {
        constexpr int P = C::SC / 16;
        for (int i = tid; i < rows * P; i += C::NT) {
            const int r = i / P, p = i % P;
            if (kb + 16 * p >= Kb) continue;
            const size_t off = (size_t)min(row0 + r, last) * Kb + kb + 16 * p, total = ((size_t)last + 1) * Kb;
            unsigned w[4] = {0u, 0u, 0u, 0u};
            if (off + 16 <= total) __builtin_memcpy(w, s + off, 16);
            else {
#pragma unroll
                for (int j = 0; j < 16; ++j) if (off + j < total) w[j >> 2] |= (unsigned)s[off + j] << (8 * (j & 3));
            }
            unsigned* const d = reinterpret_cast<unsigned*>(dst + r * C::SROW + 16 * p);
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j] = w[j];
        }
    };
    f32x16 acc[IM][IN] = {};
    const int fr = lane & 31, fh = lane >> 5;
    const int sw = (fr >> 2) & 3, c0 = ((2 * fh) ^ sw) * 16, c1 = ((2 * fh + 1) ^ sw) * 16;
    const char* const pa = smem + (wm * (TM / WM) + fr) * 64;
    const char* const pb = smem + (TM + wn * (TN / WN) + fr) * 64;
    i32x8 fa[2][IM], fb[2][IN];
    // (typed f16x8: with integer vectors hipcc orders the reads behind vmcnt(0), i.e. behind the DMA just issued for later half blocks)
    auto frag = [&](const char* p) {
        const i32x4 lo = __builtin_bit_cast(i32x4, *reinterpret_cast<const f16x8*>(p + c0)), hi = __builtin_bit_cast(i32x4, *reinterpret_cast<const f16x8*>(p + c1));
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto load = [&](int s, int set) {
        const int base = (s & (C::NST - 1)) * C::STAGE;
#pragma unroll
        for (int j = 0; j < IN; ++j) fb[set][j] = frag(pb + base + j * 32 * 64);
#pragma unroll
        for (int i = 0; i < IM; ++i) fa[set][i] = frag(pa + base + i * 32 * 64);
    };
    unsigned wa[IM], wb[IN];
    auto words = [&](int kb) {
        const int at = kb & (C::SC - 1);
#pragma unroll
        for (int i = 0; i < IM; ++i) wa[i] = *reinterpret_cast<const unsigned*>(sca + (wm * (TM / WM) + i * 32 + fr) * C::SROW + at);
#pragma unroll
        for (int j = 0; j < IN; ++j) wb[j] = *reinterpret_cast<const unsigned*>(scb + (BLK ? (wn * (TN / WN) + j * 32) / QB : wn * (TN / WN) + j * 32 + fr) * C::SROW + at);
    };
    auto ready = [&]() {                                                 // all but the newest half block in flight have landed, for every wave
        __builtin_amdgcn_sched_barrier(0);
        // not __syncthreads(): its fence would drain the DMA left in flight
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" :: "n"(C::DMA) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    };
    auto multiply = [&](int set, int sh) {
        if constexpr (DT == CNM_F32) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                bf16x8 xb[IN];
#pragma unroll
                for (int j = 0; j < IN; ++j) xb[j] = widen(fb[set][j][2 * h], fb[set][j][2 * h + 1], scale_float(wb[j], sh));
#pragma unroll
                for (int i = 0; i < IM; ++i) {
                    const bf16x8 xa = widen(fa[set][i][2 * h], fa[set][i][2 * h + 1], scale_float(wa[i], sh));
#pragma unroll
                    for (int j = 0; j < IN; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xb[j], xa, acc[i][j], 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < IM; ++i)
#pragma unroll
                for (int j = 0; j < IN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[set][j], fa[set][i], acc[i][j], 0, 0, 0, (int)((wb[j] >> sh) & 255u), 0, (int)((wa[i] >> sh) & 255u));
        }
    };

    issue(2 * kb0);
    issue(2 * kb0 + 1);
    fill(sca, g.sa, m0, TM, g.M - 1, kb0 & ~(C::SC - 1));
    fill(scb, g.sb, n0 >> g.bshift, C::BROWS, (g.N - 1) >> g.bshift, kb0 & ~(C::SC - 1));
    issue(2 * kb0 + 2);
    __syncthreads();                                                     // everything issued so far is in LDS
    load(2 * kb0, 0);
    for (int kb = kb0; kb < kb1; ++kb) {
        if (kb != kb0 && (kb & (C::SC - 1)) == 0) {
            __syncthreads();
            fill(sca, g.sa, m0, TM, g.M - 1, kb);
            fill(scb, g.sb, n0 >> g.bshift, C::BROWS, (g.N - 1) >> g.bshift, kb);
            __syncthreads();
        }
        if ((kb & 3) == 0) words(kb);
        const int s = 2 * kb, sh = 8 * (kb & 3);
        ready();                                                         // half block s + 1 is in LDS; nobody reads s - 1 any more
        issue(s + 3);
        load(s + 1, 1);
        multiply(0, sh);
        if constexpr (DT != CNM_F32) Interleave<0, IM * IN, 2 * (IM + IN), C::DMA>::go();
        ready();
        issue(s + 4);
        load(s + 2, 0);                                                  // (behind the last one: a stale or zeroed half block, not used)
        multiply(1, sh);
        if constexpr (DT != CNM_F32) Interleave<0, IM * IN, 2 * (IM + IN), C::DMA>::go();
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // no DMA outlives the loop
    // the last products stay above the stores' bounds checks: a matrix instruction sunk into divergent code would find its scales written for
    // some lanes only
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) asm volatile("" : "+v"(acc[i][j]));
    // the wave's outputs through LDS (its own part of the ring), so that they leave as whole 128-byte lines: straight from the accumulators a
    // store instruction would touch 32 rows, 16 bytes each
    constexpr int ST = SPLIT ? CNM_F32 : DT;                             // what is stored
    typedef typename Elem<ST>::T T;
    constexpr int WTM = TM / WM, WTN = TN / WN, E = 16 / (int)sizeof(T), CH = WTN / E;    // 16-byte chunks per row, permuted by the row
    static_assert(TM * TN * (int)sizeof(T) <= C::NST * C::STAGE && CH % 8 == 0, "epilogue");
    typedef T T4 __attribute__((ext_vector_type(4)));
    typedef T TE __attribute__((ext_vector_type(E)));
    asm volatile("s_barrier" ::: "memory");                              // every wave has read its last fragments
    char* const mine = smem + wave * WTM * WTN * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int row = i * 32 + fr;
#pragma unroll
        for (int j = 0; j < IN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = j * 32 + 8 * q + 4 * fh;
                const T4 v = {Elem<ST>::down(acc[i][j][4 * q]), Elem<ST>::down(acc[i][j][4 * q + 1]), Elem<ST>::down(acc[i][j][4 * q + 2]), Elem<ST>::down(acc[i][j][4 * q + 3])};
                *reinterpret_cast<T4*>(mine + (row * CH + ((n / E) ^ (row & 7))) * 16 + (n % E) * (int)sizeof(T)) = v;
            }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    T* const c = static_cast<T*>(g.c) + (SPLIT ? (size_t)split * g.M * g.N : 0);
    const bool whole = g.ldc % E == 0 && (reinterpret_cast<uintptr_t>(c) & 15) == 0;
    constexpr int RPI = 64 / CH;                                         // rows per store instruction
#pragma unroll 4
    for (int p = 0; p < WTM / RPI; ++p) {
        const int row = p * RPI + lane / CH, ch = lane % CH;
        const int m = m0 + wm * WTM + row, n = n0 + wn * WTN + ch * E;
        const TE v = *reinterpret_cast<const TE*>(mine + (row * CH + (ch ^ (row & 7))) * 16);
        if (m < g.M && n < g.N) {
            T* const d = c + (size_t)m * g.ldc + n;
            if (whole && n + E <= g.N) *reinterpret_cast<TE*>(d) = v;
            else {
#pragma unroll
                for (int e = 0; e < E; ++e) if (n + e < g.N) d[e] = v[e];
            }
        }
    }
}

// the ranges' sums, in their order
template <int DT>
__global__ __launch_bounds__(256) void join_splits_kernel(const float* __restrict__ part, int splits, long long MN, int N, typename Elem<DT>::T* __restrict__ c, long long ldc) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < MN; i += (long long)gridDim.x * 256) {
        float s = part[i];
        for (int k = 1; k < splits; ++k) s += part[(size_t)k * MN + i];
        const long long m = i / N;
        c[m * ldc + (i - m * N)] = Elem<DT>::down(s);
    }
}

// Into ranges of how many blocks (a multiple of four) the reduced axis is cut where there are few output tiles; Kb: not cut.  About one workgroup
// per CU in all, at least eight blocks each, at most 16 ranges, and of those numbers the one with the least of: the tiles' time per block
// (measured 0.4 us with 16-bit, 0.85 us with fp32 results) over the ranges, and for the ranges' fp32 sums a launch (4 us) and their way out and
// back (8 bytes each at 4.6 TB/s).  300 x 520 x 8192: bf16 28.9 -> 14.5 us, fp32 57.4 -> 18.0; 200 x 4096 x 4096: bf16 17.7 us as it is and 21.0 cut in
// four, fp32 32.5 -> 24.4.
int split_chunk(bool f32, long long M, long long N, int Kb) {
    const long long tiles = cnm_ceil_div_ll(M, 128) * cnm_ceil_div_ll(N, 128);
    if (tiles > 128 || Kb < 16) return Kb;
    const double per_block = f32 ? 0.85 : 0.4, join = 8.0 * (double)M * (double)N / 4.6e6;
    int best = Kb;
    double t = per_block * Kb;
    for (int n = 2; n <= 16 && n <= 256 / tiles && n <= Kb / 8; ++n) {
        const int chunk = ((Kb + n - 1) / n + 3) / 4 * 4, ranges = cnm_ceil_div(Kb, chunk);
        const double tn = per_block * chunk + 4.0 + ranges * join;
        if (tn < t) { t = tn; best = chunk; }
    }
    return best;
}

template <int TM, int TN, int WM, int WN, int DT, bool SPLIT = false>
int launch_tiles(MatArgs g, hipStream_t stream) {
    g.tiles_m = cnm_ceil_div(g.M, TM); g.tiles_n = cnm_ceil_div(g.N, TN);
    const unsigned blocks = (unsigned)(g.tiles_m * g.tiles_n * (SPLIT ? g.splits : 1));
    if (g.bshift) matmul_fp8_kernel<TM, TN, WM, WN, DT, true, SPLIT><<<blocks, WM * WN * 64, Mat<TM, TN, WM, WN, DT, true>::LDS, stream>>>(g);
    else matmul_fp8_kernel<TM, TN, WM, WN, DT, false, SPLIT><<<blocks, WM * WN * 64, Mat<TM, TN, WM, WN, DT, false>::LDS, stream>>>(g);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

template <int DT>
int launch_matmul(MatArgs g, float* ws, hipStream_t stream) {
    // 256 x 256 tiles (eight waves of 128 x 64, one workgroup per CU) from more tiles than half the CUs on; below that twice as many CUs
    // work on 128 x 128 tiles (four waves of 64 x 64, two workgroups per CU).  bf16, 4096 x 4096 x 8192 (256 / 1024 tiles): 117 us against
    // 166; 2048 x 2048 x 2048 (64 / 256 tiles): 25 us against 13.5.  fp32 results convert their operands on the way: 128 x 128 only
    // (64 accumulators per lane leave room for the bf16 fragments).
    if constexpr (DT != CNM_F32)
        if ((long long)cnm_ceil_div(g.M, 256) * cnm_ceil_div(g.N, 256) > 128) return launch_tiles<256, 256, 2, 4, DT>(g, stream);
    const int chunk = split_chunk(DT == CNM_F32, g.M, g.N, g.Kb);
    if (chunk >= g.Kb) return launch_tiles<128, 128, 2, 2, DT>(g, stream);
    MatArgs p = g;
    p.c = ws; p.ldc = g.N; p.chunk = chunk; p.splits = cnm_ceil_div(g.Kb, chunk);
    const int rc = launch_tiles<128, 128, 2, 2, DT, true>(p, stream);
    if (rc != CNM_OK) return rc;
    const long long MN = (long long)g.M * g.N, blocks = cnm_ceil_div_ll(MN, 256);
    join_splits_kernel<DT><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, stream>>>(ws, p.splits, MN, g.N, static_cast<typename Elem<DT>::T*>(g.c), g.ldc);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

// ------------------------------------------------------------------ few rows, or few columns
// Where one side is small the product reads the other side once and is bound by that: no LDS staging, fragments straight from memory, MT tiles
// of 16 rows of x against NT_ tiles of 16 rows of w per wave, PF blocks of 128 requested before the first is used.
//   few rows (single tokens up to 64): a workgroup takes 16 weight rows, its eight waves share the reduced axis (KS = 8) and join their sums in LDS
//     in a fixed order;
//   few columns (N <= 128): a wave takes 16 MT rows of x and all of w, which stays in the caches (KS = 1).
// QUANT: x comes as it is (float32 / float16 / bfloat16) and is quantised in registers: a lane holds 32 consecutive values of one row, its
// block's maximum is two exchanges away; x is then read once and never written in 8 bits.
// bf16 1 x 4096 x 4096: 7.0 us (2.4 TB/s of the 16 MB weight, the launch's own latency half of it); fp32 49152 x 64 x 512: 26.7 us (4.2 TB/s).
struct StreamArgs {
    const void* x; long long ldx;            // [M][ldx] as it is, or e4m3 [M][Kb * 128] with scale sx [M][Kb]
    const unsigned char *sx, *w, *sw;
    void* c; long long ldc;
    int M, N, K, Kb, bshift;                 // K: columns of x that exist (QUANT)
};

constexpr int stream_waves(int ks) { return ks > 1 ? ks : 4; }            // per workgroup: small ones where nothing is shared, so that all fit the CUs at once
template <int DT, bool QUANT, int MT, int NT_, int KS, int PF>
__global__ __launch_bounds__(stream_waves(KS) * 64) void stream_kernel(const StreamArgs g) {
    typedef typename Elem<DT>::T T;
    constexpr int MG = stream_waves(KS) / KS;                                           // row groups per workgroup
    __shared__ float part[KS > 1 ? KS : 1][KS > 1 ? NT_ * 16 : 1][KS > 1 ? MT * 16 + 1 : 1];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ks = wave % KS, mg = wave / KS, fr = lane & 15, fg = lane >> 4;
    const int nblocks = (g.N + NT_ * 16 - 1) / (NT_ * 16);
    const int nb = blockIdx.x % nblocks;
    const int n0 = nb * NT_ * 16, m0 = (int)(blockIdx.x / nblocks * MG + mg) * MT * 16;
    const unsigned char* wp[NT_]; const unsigned char* swp[NT_];
#pragma unroll
    for (int j = 0; j < NT_; ++j) {
        const int n = min(n0 + j * 16 + fr, g.N - 1);
        wp[j] = g.w + (size_t)n * g.Kb * QB + fg * 32;
        swp[j] = g.sw + (size_t)(n >> g.bshift) * g.Kb;
    }
    const T* xp[MT]; const unsigned char* qp[MT]; const unsigned char* sxp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int m = min(m0 + i * 16 + fr, g.M - 1);
        if (QUANT) xp[i] = static_cast<const T*>(g.x) + (size_t)m * g.ldx + fg * 32;
        else { qp[i] = static_cast<const unsigned char*>(g.x) + (size_t)m * g.Kb * QB + fg * 32; sxp[i] = g.sx + (size_t)m * g.Kb; }
    }
    f32x4 acc[MT][NT_] = {};
    i32x8 fw[PF][NT_], fa[PF][MT];
    int bw[PF][NT_], ba[PF][MT];
    T raw[PF][QUANT ? MT : 1][32];
    const auto request_x = [&](int p, int kb) {
        if (kb >= g.Kb) return;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (QUANT) {
                const T* const src = xp[i] + (size_t)kb * QB;
                const int have = g.K - kb * QB - fg * 32;
                if (have >= 32) __builtin_memcpy(raw[p][i], src, 32 * sizeof(T));
                else {
#pragma unroll
                    for (int e = 0; e < 32; ++e) raw[p][i][e] = e < have ? src[e] : (T)0.f;
                }
            } else {
                __builtin_memcpy(&fa[p][i], qp[i] + (size_t)kb * QB, 32);
                ba[p][i] = sxp[i][kb];
            }
        }
    };
    const auto request_w = [&](int p, int kb) {
        if (kb >= g.Kb) return;
#pragma unroll
        for (int j = 0; j < NT_; ++j) {
            __builtin_memcpy(&fw[p][j], wp[j] + (size_t)kb * QB, 32);
            bw[p][j] = swp[j][kb];
        }
    };
    const auto quantize_x = [&](int p, int kb) {
        if (kb >= g.Kb) return;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            float v[32], m = 0.f;
#pragma unroll
            for (int e = 0; e < 32; ++e) { v[e] = Elem<DT>::up(raw[p][QUANT ? i : 0][e]); m = fmaxf(m, fabsf(v[e])); }
            m = fmaxf(m, __shfl_xor(m, 16)); m = fmaxf(m, __shfl_xor(m, 32));
            if (__any(m == __builtin_huge_valf())) {                     // an infinity in some row's block: it does not take part in the maximum
                m = 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) m = fmaxf(m, finite_abs(v[e]));
                m = fmaxf(m, __shfl_xor(m, 16)); m = fmaxf(m, __shfl_xor(m, 32));
            }
            ba[p][i] = scale_byte(m);
            const float k = inv_scale(ba[p][i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) fa[p][i][e] = (int)pack4(v[4 * e] * k, v[4 * e + 1] * k, v[4 * e + 2] * k, v[4 * e + 3] * k);
        }
    };
    const auto multiply = [&](int p, int kb) {
        if (kb >= g.Kb) return;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (DT == CNM_F32) {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const bf16x8 xa = widen(fa[p][i][2 * h], fa[p][i][2 * h + 1], scale_float((unsigned)ba[p][i], 0));
#pragma unroll
                    for (int j = 0; j < NT_; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(fw[p][j][2 * h], fw[p][j][2 * h + 1], scale_float((unsigned)bw[p][j], 0)), xa, acc[i][j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < NT_; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[p][j], fa[p][i], acc[i][j], 0, 0, 0, bw[p][j], 0, ba[p][i]);
            }
        }
    };
    if constexpr (KS == 1) {
        // x is what streams: the next block is requested once this one's registers are free, behind this one's w (loads return in order: w
        // from the caches must not wait for x)
        static_assert(PF == 1, "one block ahead");
        request_x(0, 0);
        for (int kb = 0; kb < g.Kb; ++kb) {
            request_w(0, kb);
            quantize_x(0, kb);
            request_x(0, kb + 1);
            multiply(0, kb);
        }
    } else {                                                             // w is what streams
        for (int g0 = ks; g0 < g.Kb; g0 += KS * PF) {
#pragma unroll
            for (int p = 0; p < PF; ++p) { request_x(p, g0 + p * KS); request_w(p, g0 + p * KS); }   // (x first: loads return in order, and x has to be quantised)
#pragma unroll
            for (int p = 0; p < PF; ++p) {
                if constexpr (QUANT) quantize_x(p, g0 + p * KS);
                multiply(p, g0 + p * KS);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT_; ++j) asm volatile("" : "+v"(acc[i][j]));  // above the bounds checks (see the tile kernel)
    T* const c = static_cast<T*>(g.c);
    if constexpr (KS > 1) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT_; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) part[ks][j * 16 + 4 * fg + e][i * 16 + fr] = acc[i][j][e];
        __syncthreads();
        for (int o = threadIdx.x; o < MT * 16 * NT_ * 16; o += stream_waves(KS) * 64) {
            const int n = o % (NT_ * 16), m = o / (NT_ * 16);
            float s = part[0][n][m];
#pragma unroll
            for (int k = 1; k < KS; ++k) s += part[k][n][m];
            if (m0 + m < g.M && n0 + n < g.N) c[(size_t)(m0 + m) * g.ldc + n0 + n] = Elem<DT>::down(s);
        }
    } else {
        const bool four = (g.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(c) & (4 * sizeof(T) - 1)) == 0;
        typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const int m = m0 + i * 16 + fr;
#pragma unroll
            for (int j = 0; j < NT_; ++j) {
                const int n = n0 + j * 16 + 4 * fg;
                if (m < g.M && n < g.N) {
                    T* const d = c + (size_t)m * g.ldc + n;
                    if (four && n + 4 <= g.N) *reinterpret_cast<T4*>(d) = T4{Elem<DT>::down(acc[i][j][0]), Elem<DT>::down(acc[i][j][1]), Elem<DT>::down(acc[i][j][2]), Elem<DT>::down(acc[i][j][3])};
                    else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) if (n + e < g.N) d[e] = Elem<DT>::down(acc[i][j][e]);
                    }
                }
            }
        }
    }
}

template <int DT, bool QUANT, int MT, int NT_, int KS, int PF>
int launch_stream(const StreamArgs& g, hipStream_t stream) {
    const long long blocks = (long long)cnm_ceil_div(g.N, NT_ * 16) * cnm_ceil_div(g.M, stream_waves(KS) / KS * MT * 16);
    stream_kernel<DT, QUANT, MT, NT_, KS, PF><<<(unsigned)blocks, stream_waves(KS) * 64, 0, stream>>>(g);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

// few rows of 8-bit x
template <int DT>
int launch_few_rows(const StreamArgs& g, hipStream_t stream) {
    if (g.M <= 16) return launch_stream<DT, false, 1, 1, 8, 4>(g, stream);
    if (g.M <= 32) return launch_stream<DT, false, 2, 1, 8, 2>(g, stream);
    if (g.M <= 48) return launch_stream<DT, false, 3, 1, 8, 2>(g, stream);
    return launch_stream<DT, false, 4, 1, 8, 2>(g, stream);
}

// x as it is: few columns, or at most 16 rows.  The few-columns form splits nothing: it pays with many rows (fp32 49152 x 64 x 512: 27 us,
// quantised first and multiplied in tiles 21 + 14; 16384 x 128 x 512: 15 against 10 + 11) and is the slower one where few rows meet a long reduced
// axis, one workgroup per 64 rows walking it alone (bf16 4096 x 64 x 2048: 24 us against 9 + 11; 1000 x 64 x 8192: 87 against 9 + 15;
// 64 x 128 x 8192: 143 against 9 + 27).
template <int DT>
int launch_quantizing(const StreamArgs& g, hipStream_t stream) {
    if (g.M <= 16) return launch_stream<DT, true, 1, 1, 8, 4>(g, stream);
    if (g.N <= 64) return launch_stream<DT, true, 1, 4, 1, 1>(g, stream);
    return launch_stream<DT, true, 1, 8, 1, 1>(g, stream);
}

constexpr int FEW_ROWS = 64, FEW_COLS = 128;

// a launch holds fewer than 2^32 threads: what the kernels above take for a matrix or product of these sizes
bool launch_fits(long long blocks, int threads) { return blocks < (1ll << 32) / threads; }
bool quantize_fits(long long rows, long long cols) { return launch_fits(cnm_ceil_div_ll(rows, QB) * cnm_ceil_div_ll(cols, QB), 512); }
bool matmul_fits(long long M, long long N) {
    return M <= FEW_ROWS ? launch_fits(cnm_ceil_div_ll(N, 16), 512) : launch_fits(cnm_ceil_div_ll(M, 128) * cnm_ceil_div_ll(N, 128), 256);
}

}  // namespace

extern "C" int cnm_quantize_fp8(const void* x, int dtype, long long ldx, long long rows, long long cols, int block_rows,
                                void* q, void* scale, void* q_t, void* scale_t, void* stream) {
    CNM_REQUIRE(x && rows > 0 && cols > 0 && ldx >= cols && (block_rows == 1 || block_rows == QB), CNM_ERR_BAD_ARG);
    CNM_REQUIRE((q || q_t) && !q == !scale && !q_t == !scale_t, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_t)) & 15) == 0, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(rows < (1ll << 31) - QB && cols < (1ll << 31) - QB && quantize_fits(rows, cols), CNM_ERR_BAD_SHAPE);
    const int R = (int)rows, C = (int)cols;
    const hipStream_t st = cnm_stream(stream);
#define CNM_Q(DT) return block_rows == 1 ? launch_quantize<DT, false>(x, ldx, R, C, q, scale, q_t, scale_t, st) : launch_quantize<DT, true>(x, ldx, R, C, q, scale, q_t, scale_t, st)
    switch (dtype) {
        case CNM_F32: CNM_Q(CNM_F32);
        case CNM_F16: CNM_Q(CNM_F16);
        case CNM_BF16: CNM_Q(CNM_BF16);
    }
#undef CNM_Q
    return CNM_ERR_BAD_ARG;
}

extern "C" size_t cnm_matmul_fp8_workspace_bytes(int dtype, long long M, long long N, long long K) {
    if (M <= FEW_ROWS || N <= 0 || K <= 0 || K > (1ll << 23)) return 0;
    const int kb = (int)cnm_ceil_div_ll(K, QB), chunk = split_chunk(dtype == CNM_F32, M, N, kb);
    return chunk < kb ? (size_t)cnm_ceil_div(kb, chunk) * (size_t)M * (size_t)N * sizeof(float) : 0;
}
// of either kind of result
static size_t matmul_workspace(long long M, long long N, long long K) {
    const size_t a = cnm_matmul_fp8_workspace_bytes(CNM_F32, M, N, K), b = cnm_matmul_fp8_workspace_bytes(CNM_BF16, M, N, K);
    return a > b ? a : b;
}

extern "C" int cnm_matmul_fp8(const void* a, const void* a_scale, const void* b, const void* b_scale, int b_block_rows, void* c, int dtype,
                              long long ldc, long long M, long long N, long long K, void* workspace, size_t workspace_bytes, void* stream) {
    CNM_REQUIRE(a && a_scale && b && b_scale && c && M > 0 && N > 0 && K > 0 && K % QB == 0 && ldc >= N, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(b_block_rows == 1 || b_block_rows == QB, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && K <= (1ll << 23), CNM_ERR_BAD_SHAPE);   // 256 rows of an operand are one 32-bit buffer range
    CNM_REQUIRE(matmul_fits(M, N), CNM_ERR_BAD_SHAPE);
    MatArgs g = {static_cast<const unsigned char*>(a), static_cast<const unsigned char*>(a_scale), static_cast<const unsigned char*>(b), static_cast<const unsigned char*>(b_scale),
                 c, (int)M, (int)N, (int)(K / QB), b_block_rows == 1 ? 0 : 7, ldc, 0, 0, 1, 0};
    const size_t need = cnm_matmul_fp8_workspace_bytes(dtype, M, N, K);
    CNM_REQUIRE(!need || (workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0), CNM_ERR_WORKSPACE);
    float* const ws = static_cast<float*>(workspace);
    const StreamArgs f = {a, 0, g.sa, g.b, g.sb, c, ldc, g.M, g.N, (int)K, g.Kb, g.bshift};
    const hipStream_t st = cnm_stream(stream);
#define CNM_M(DT) return M <= FEW_ROWS ? launch_few_rows<DT>(f, st) : launch_matmul<DT>(g, ws, st)
    switch (dtype) {
        case CNM_F32: CNM_M(CNM_F32);
        case CNM_F16: CNM_M(CNM_F16);
        case CNM_BF16: CNM_M(CNM_BF16);
    }
#undef CNM_M
    return CNM_ERR_BAD_ARG;
}

// ---- one training step of the layer.  A matrix in 8 bits, values then scales, in a byte buffer of fp8_bytes
static size_t fp8_bytes(long long rows, long long cols, bool blocks) {
    const size_t kb = (size_t)cnm_ceil_div_ll(cols, QB), n = (size_t)rows * kb * QB + (size_t)(blocks ? cnm_ceil_div_ll(rows, QB) : rows) * kb;
    return (n + 15) / 16 * 16;
}
struct Fp8 { unsigned char *q = nullptr, *s = nullptr; };
static Fp8 fp8_take(unsigned char*& at, long long rows, long long cols, bool blocks) {
    Fp8 m;
    m.q = at; m.s = at + (size_t)rows * cnm_ceil_div_ll(cols, QB) * QB;
    at += fp8_bytes(rows, cols, blocks);
    return m;
}
static bool dtype_ok(int d) { return d >= CNM_F32 && d <= CNM_BF16; }
static bool train_shape_ok(long long M, long long N, long long K) {
    const long long most = 1ll << 23;                                    // each of them is a reduced axis of some product
    return M <= most - QB && N <= most - QB && K <= most - QB
        && quantize_fits(M, K) && quantize_fits(N, K) && quantize_fits(M, N) && matmul_fits(M, N) && matmul_fits(M, K) && matmul_fits(N, K);
}

extern "C" size_t cnm_linear_fp8_keep_bytes(long long M, long long N, long long K, int need_dx, int need_dw) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return (need_dx ? fp8_bytes(K, N, true) : 0) + (need_dw ? fp8_bytes(K, M, false) : 0);
}
extern "C" size_t cnm_linear_fp8_train_workspace_bytes(long long M, long long N, long long K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const auto up = [](long long n) { return cnm_ceil_div_ll(n, QB) * QB; };
    const size_t dx = matmul_workspace(M, K, up(N)), dw = matmul_workspace(N, K, up(M));
    const size_t fwd = fp8_bytes(M, K, false) + fp8_bytes(N, K, true) + matmul_workspace(M, N, up(K)), bwd = fp8_bytes(M, N, false) + fp8_bytes(N, M, false) + (dx > dw ? dx : dw);
    return fwd > bwd ? fwd : bwd;
}

extern "C" int cnm_linear_fp8_forward(const void* x, int x_dtype, long long ldx, const void* w, int w_dtype, long long ldw, void* y,
                                      long long M, long long N, long long K, int need_dx, int need_dw, void* keep, size_t keep_bytes,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    CNM_REQUIRE(x && w && y && M > 0 && N > 0 && K > 0 && ldx >= K && ldw >= K && dtype_ok(x_dtype) && dtype_ok(w_dtype), CNM_ERR_BAD_ARG);   // (everything before the first launch)
    CNM_REQUIRE(train_shape_ok(M, N, K), CNM_ERR_BAD_SHAPE);
    CNM_REQUIRE(workspace && workspace_bytes >= cnm_linear_fp8_train_workspace_bytes(M, N, K) && keep_bytes >= cnm_linear_fp8_keep_bytes(M, N, K, need_dx, need_dw)
                && (keep || !(need_dx || need_dw)) && ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(keep)) & 15) == 0, CNM_ERR_WORKSPACE);
    unsigned char *ws = static_cast<unsigned char*>(workspace), *kp = static_cast<unsigned char*>(keep);
    const Fp8 xq = fp8_take(ws, M, K, false), wq = fp8_take(ws, N, K, true);
    Fp8 wt, xt;
    if (need_dx) wt = fp8_take(kp, K, N, true);
    if (need_dw) xt = fp8_take(kp, K, M, false);
    int rc = cnm_quantize_fp8(w, w_dtype, ldw, N, K, QB, wq.q, wq.s, wt.q, wt.s, stream);
    if (rc == CNM_OK) rc = cnm_quantize_fp8(x, x_dtype, ldx, M, K, 1, xq.q, xq.s, xt.q, xt.s, stream);
    return rc != CNM_OK ? rc : cnm_matmul_fp8(xq.q, xq.s, wq.q, wq.s, QB, y, x_dtype, N, M, N, cnm_ceil_div_ll(K, QB) * QB, ws, workspace_bytes - (ws - static_cast<unsigned char*>(workspace)), stream);
}

extern "C" int cnm_linear_fp8_backward(const void* dy, int dy_dtype, long long lddy, const void* keep, size_t keep_bytes, void* dx, int dx_dtype, void* dw, int dw_dtype,
                                       long long M, long long N, long long K, int kept_dx, int kept_dw, void* workspace, size_t workspace_bytes, void* stream) {
    CNM_REQUIRE(dy && keep && (dx || dw) && M > 0 && N > 0 && K > 0 && lddy >= N && (!dx || kept_dx) && (!dw || kept_dw), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(dtype_ok(dy_dtype) && (!dx || dtype_ok(dx_dtype)) && (!dw || dtype_ok(dw_dtype)), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(train_shape_ok(M, N, K), CNM_ERR_BAD_SHAPE);
    CNM_REQUIRE(workspace && workspace_bytes >= cnm_linear_fp8_train_workspace_bytes(M, N, K) && keep_bytes >= cnm_linear_fp8_keep_bytes(M, N, K, kept_dx, kept_dw)
                && ((reinterpret_cast<uintptr_t>(workspace) | reinterpret_cast<uintptr_t>(keep)) & 15) == 0, CNM_ERR_WORKSPACE);
    unsigned char *ws = static_cast<unsigned char*>(workspace), *kp = static_cast<unsigned char*>(const_cast<void*>(keep));
    Fp8 wt, xt, dyq, dyt;
    if (kept_dx) wt = fp8_take(kp, K, N, true);
    if (kept_dw) xt = fp8_take(kp, K, M, false);
    if (dx) dyq = fp8_take(ws, M, N, false);
    if (dw) dyt = fp8_take(ws, N, M, false);
    const size_t left = workspace_bytes - (ws - static_cast<unsigned char*>(workspace));
    int rc = cnm_quantize_fp8(dy, dy_dtype, lddy, M, N, 1, dyq.q, dyq.s, dyt.q, dyt.s, stream);
    if (rc == CNM_OK && dx) rc = cnm_matmul_fp8(dyq.q, dyq.s, wt.q, wt.s, QB, dx, dx_dtype, K, M, K, cnm_ceil_div_ll(N, QB) * QB, ws, left, stream);
    if (rc == CNM_OK && dw) rc = cnm_matmul_fp8(dyt.q, dyt.s, xt.q, xt.s, 1, dw, dw_dtype, K, N, K, cnm_ceil_div_ll(M, QB) * QB, ws, left, stream);
    return rc;
}

extern "C" size_t cnm_linear_fp8_workspace_bytes(long long M, long long N, long long K) {
    if (M <= 0 || N <= 0 || K <= 0 || M <= 16 || N <= FEW_COLS) return 0;
    return fp8_bytes(M, K, false) + matmul_workspace(M, N, cnm_ceil_div_ll(K, QB) * QB);
}

extern "C" int cnm_linear_fp8(const void* x, int dtype, long long ldx, const void* w, const void* w_scale, void* y, long long ldy,
                              long long M, long long N, long long K, void* workspace, size_t workspace_bytes, void* stream) {
    CNM_REQUIRE(x && w && w_scale && y && M > 0 && N > 0 && K > 0 && ldx >= K && ldy >= N, CNM_ERR_BAD_ARG);
    CNM_REQUIRE((reinterpret_cast<uintptr_t>(w) & 15) == 0 && dtype_ok(dtype), CNM_ERR_BAD_ARG);
    CNM_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && K <= (1ll << 23), CNM_ERR_BAD_SHAPE);
    CNM_REQUIRE(M <= 16 ? launch_fits(cnm_ceil_div_ll(N, 16), 512) : N <= FEW_COLS ? launch_fits(cnm_ceil_div_ll(M, 64), 256) : quantize_fits(M, K) && matmul_fits(M, N), CNM_ERR_BAD_SHAPE);
    const size_t need = cnm_linear_fp8_workspace_bytes(M, N, K);
    const long long kb = cnm_ceil_div_ll(K, QB);
    if (need) {                                                          // quantise, then multiply
        CNM_REQUIRE(workspace && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0, CNM_ERR_WORKSPACE);
        unsigned char* at = static_cast<unsigned char*>(workspace);
        const Fp8 q = fp8_take(at, M, K, false);
        const int rc = cnm_quantize_fp8(x, dtype, ldx, M, K, 1, q.q, q.s, nullptr, nullptr, stream);
        return rc != CNM_OK ? rc : cnm_matmul_fp8(q.q, q.s, w, w_scale, QB, y, dtype, ldy, M, N, kb * QB, at, need, stream);
    }
    const StreamArgs f = {x, ldx, nullptr, static_cast<const unsigned char*>(w), static_cast<const unsigned char*>(w_scale), y, ldy, (int)M, (int)N, (int)K, (int)kb, 7};
    const hipStream_t st = cnm_stream(stream);
    switch (dtype) {
        case CNM_F32: return launch_quantizing<CNM_F32>(f, st);
        case CNM_F16: return launch_quantizing<CNM_F16>(f, st);
        case CNM_BF16: return launch_quantizing<CNM_BF16>(f, st);
    }
    return CNM_ERR_BAD_ARG;
}
