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
//   16-bit results: v_mfma_scale_f32_16x16x128_f8f6f4 on the bytes as they are, twice the bf16 rate.  Its accumulator is fp32, but it adds
//     eight consecutive products at a time, each cut off at 2^-13 of the eight's largest exponent (measured: probes of single terms; rms
//     1.5e-5 of the result on normal data): a choice for results that are rounded to 2^-9 or 2^-12 anyway.
//   fp32 results: the bytes become bf16 with their scale applied (exact within bf16's exponent range) and v_mfma_f32_16x16x32_bf16 adds them:
//     rms 1e-8 of the result, as fp32 sums are.
#include "cnm_common.h"

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
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

// four values -> four e4m3 bytes; |v| <= 448 but for non-finite inputs
__device__ inline unsigned pack4(float a, float b, float c, float d) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, p, true);
    unsigned u = (unsigned)p;
    if (!(fabsf(a) < __builtin_huge_valf())) u = (u & ~0x000000FFu) | 0x0000007Fu;
    if (!(fabsf(b) < __builtin_huge_valf())) u = (u & ~0x0000FF00u) | 0x00007F00u;
    if (!(fabsf(c) < __builtin_huge_valf())) u = (u & ~0x00FF0000u) | 0x007F0000u;
    if (!(fabsf(d) < __builtin_huge_valf())) u = (u & ~0xFF000000u) | 0x7F000000u;
    return u;
}

// eight consecutive values of a row, zero beyond `have`
template <int DT, bool VEC>
__device__ inline void load8(const typename Elem<DT>::T* p, int have, float v[8]) {
    if (VEC && have >= 8) {
        if constexpr (DT == CNM_F32) {
            const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
        } else {
            typedef typename Elem<DT>::T T8 __attribute__((ext_vector_type(8)));
            const T8 a = *reinterpret_cast<const T8*>(p);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = Elem<DT>::up(a[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < have ? Elem<DT>::up(p[j]) : 0.f;
    }
}

// One workgroup quantises a 128 x 128 tile, read once: 16 lanes per row (8 values each), a thread's eight rows consecutive, so that the
// transposed copy leaves as 8-byte columns through LDS.  Row form: q [R][Cp], s [R][Cp/128] (BLK = false) or s [R/128][Cp/128] (BLK = true).
// Transposed form (optional): qt [C][Rp], blocked along R: st [C][Rp/128], or the same 128 x 128 block's byte at st [C/128][Rp/128].
template <int DT, bool BLK, bool VEC>
__global__ __launch_bounds__(256) void quantize_kernel(const typename Elem<DT>::T* __restrict__ x, long long ldx, int R, int C, int Cb, int Rb,
                                                       unsigned char* __restrict__ q, unsigned char* __restrict__ s,
                                                       unsigned char* __restrict__ qt, unsigned char* __restrict__ st) {
    __shared__ float cmax[16][QB];
    __shared__ unsigned char tile[QB][QB + 8];
    __shared__ float bmax[4];
    const int tid = threadIdx.x, lc = tid & 15, lr = tid >> 4;
    const int cb = blockIdx.x % Cb, rb = blockIdx.x / Cb;
    const int c0 = cb * QB + lc * 8, r0 = rb * QB + lr * 8;
    float v[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = r0 + p;
        load8<DT, VEC>(x + (size_t)(r < R ? r : 0) * ldx + (c0 < C ? c0 : 0), r < R ? C - c0 : 0, v[p]);
    }
    int byte[8];
    float am[8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        float m = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[p][j]));
        for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        am[p] = m;
    }
    if (BLK) {
        float m = 0.f;
#pragma unroll
        for (int p = 0; p < 8; ++p) m = fmaxf(m, am[p]);
        m = fmaxf(m, __shfl_xor(m, 16)); m = fmaxf(m, __shfl_xor(m, 32));
        if ((tid & 63) == 0) bmax[tid >> 6] = m;
        __syncthreads();
        m = fmaxf(fmaxf(bmax[0], bmax[1]), fmaxf(bmax[2], bmax[3]));
#pragma unroll
        for (int p = 0; p < 8; ++p) byte[p] = scale_byte(m);
        if (tid == 0) {
            if (s) s[(size_t)rb * Cb + cb] = (unsigned char)byte[0];
            if (st) st[(size_t)cb * Rb + rb] = (unsigned char)byte[0];
        }
    } else {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            byte[p] = scale_byte(am[p]);
            if (s && lc == 0 && r0 + p < R) s[(size_t)(r0 + p) * Cb + cb] = (unsigned char)byte[p];
        }
    }
    if (q) {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
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
            for (int p = 0; p < 8; ++p) m = fmaxf(m, finite_abs(v[p][j]));
            cmax[lr][lc * 8 + j] = m;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = 0.f;
            for (int g = 0; g < 16; ++g) m = fmaxf(m, cmax[g][lc * 8 + j]);
            const int b = scale_byte(m);
            k8[j] = inv_scale(b);
            if (lr == 0 && c0 + j < C) st[(size_t)(c0 + j) * Rb + rb] = (unsigned char)b;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) k8[j] = inv_scale(byte[0]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        uint2 u;
        u.x = pack4(v[0][j] * k8[j], v[1][j] * k8[j], v[2][j] * k8[j], v[3][j] * k8[j]);
        u.y = pack4(v[4][j] * k8[j], v[5][j] * k8[j], v[6][j] * k8[j], v[7][j] * k8[j]);
        *reinterpret_cast<uint2*>(&tile[lc * 8 + j][lr * 8]) = u;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {                                        // 16 lanes x 8 bytes = one transposed row of the tile
        const int c = i * 16 + lr;
        if (cb * QB + c < C)
            *reinterpret_cast<uint2*>(qt + (size_t)(cb * QB + c) * ((size_t)Rb * QB) + (size_t)rb * QB + lc * 8) = *reinterpret_cast<const uint2*>(&tile[c][lc * 8]);
    }
}

template <int DT, bool BLK>
int launch_quantize(const void* x, long long ldx, int R, int C, void* q, void* s, void* qt, void* st, hipStream_t stream) {
    typedef typename Elem<DT>::T T;
    const int Cb = cnm_ceil_div(C, QB), Rb = cnm_ceil_div(R, QB);
    const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0 && (ldx * (long long)sizeof(T)) % 16 == 0;   // every row starts on 16 bytes, so does every group of eight
    auto* xp = static_cast<const T*>(x);
    auto* qp = static_cast<unsigned char*>(q); auto* sp = static_cast<unsigned char*>(s);
    auto* qtp = static_cast<unsigned char*>(qt); auto* stp = static_cast<unsigned char*>(st);
    if (vec) quantize_kernel<DT, BLK, true><<<Cb * Rb, 256, 0, stream>>>(xp, ldx, R, C, Cb, Rb, qp, sp, qtp, stp);
    else quantize_kernel<DT, BLK, false><<<Cb * Rb, 256, 0, stream>>>(xp, ldx, R, C, Cb, Rb, qp, sp, qtp, stp);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

// ------------------------------------------------------------------ product
// Four consecutive scale bytes of a row (blocks kb .. kb + 3) as one word: an unaligned load that never leaves the array -- near its end it
// reads the last four bytes and shifts; bytes beyond the row belong to the next one and are not used.
__device__ inline unsigned scale_word(const unsigned char* s, size_t off, size_t total) {
    if (total < 4) {
        unsigned w = 0;
        for (size_t i = 0; i < 4; ++i) if (off + i < total) w |= (unsigned)s[off + i] << (8 * i);
        return w;
    }
    const size_t at = off < total - 4 ? off : total - 4;
    unsigned w;
    __builtin_memcpy(&w, s + at, 4);
    return w >> (8 * (off - at));
}

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
};

// TM x TN outputs per workgroup, WM x WN waves; a k-step is one block of 128: 128 bytes per operand row, brought to LDS by DMA one step ahead.
// LDS: row r at r * 128, its eight 16-byte chunks permuted by (r >> 1) & 7: the 16 rows that a fragment read touches at one chunk then fall on
// all 64 banks.  The DMA writes 64 lanes x 16 bytes in order, so the permutation is in the lanes' source addresses.
// The weight is the instruction's first operand: a lane then holds four consecutive outputs of one row.
template <int TM, int TN, int WM, int WN, int DT>
__global__ __launch_bounds__(WM * WN * 64) void matmul_fp8_kernel(const MatArgs g) {
    constexpr int NW = WM * WN, IM = TM / WM / 16, IN = TN / WN / 16;
    constexpr int ROWS = TM + TN, STAGE = ROWS * QB, PIECES = ROWS / 8 / NW;   // a piece: one DMA instruction, eight rows
    extern __shared__ char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave / WN, wn = wave % WN;
    const int blk = xcd_remap(blockIdx.x, gridDim.x);
    const int tm = blk / g.tiles_n, tn = blk % g.tiles_n;
    const int m0 = tm * TM, n0 = tn * TN;
    const int K = g.Kb * QB;
    const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(g.a) + (size_t)m0 * K, 0, (unsigned)min(g.M - m0, TM) * (unsigned)K, 0x00020000);
    const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(g.b) + (size_t)n0 * K, 0, (unsigned)min(g.N - n0, TN) * (unsigned)K, 0x00020000);
    auto issue = [&](int kb, int buf) {
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int piece = wave * PIECES + p, row = piece * 8 + (lane >> 3);
            const int chunk = (lane & 7) ^ ((row >> 1) & 7);
            char* dst = smem + buf * STAGE + piece * 1024;
            if (piece * 8 < TM) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)dst, 16, (unsigned)row * (unsigned)K + chunk * 16, kb * QB, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)dst, 16, (unsigned)(row - TM) * (unsigned)K + chunk * 16, kb * QB, 0, 0);
        }
    };
    f32x4 acc[IM][IN] = {};
    const int fr = lane & 15, fg = lane >> 4;
    size_t oa[IM], ob[IN];
    const size_t ta = (size_t)g.M * g.Kb, tb = (size_t)(((g.N - 1) >> g.bshift) + 1) * g.Kb;
#pragma unroll
    for (int i = 0; i < IM; ++i) oa[i] = (size_t)min(m0 + wm * (TM / WM) + i * 16 + fr, g.M - 1) * g.Kb;
#pragma unroll
    for (int j = 0; j < IN; ++j) ob[j] = (size_t)(min(n0 + wn * (TN / WN) + j * 16 + fr, g.N - 1) >> g.bshift) * g.Kb;
    unsigned wa[IM], wb[IN];
    issue(0, 0);
    for (int kb = 0; kb < g.Kb; ++kb) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();                                                 // step kb is in LDS; everyone has read step kb - 1
        if ((kb & 3) == 0) {
#pragma unroll
            for (int i = 0; i < IM; ++i) wa[i] = scale_word(g.sa, oa[i] + kb, ta);
#pragma unroll
            for (int j = 0; j < IN; ++j) wb[j] = scale_word(g.sb, ob[j] + kb, tb);
        }
        if (kb + 1 < g.Kb) issue(kb + 1, (kb + 1) & 1);
        const char* base = smem + (kb & 1) * STAGE;
        i32x8 fb[IN];
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const int r = TM + wn * (TN / WN) + j * 16 + fr, sw = (r >> 1) & 7;
            const i32x4 lo = *reinterpret_cast<const i32x4*>(base + r * QB + ((2 * fg) ^ sw) * 16), hi = *reinterpret_cast<const i32x4*>(base + r * QB + ((2 * fg + 1) ^ sw) * 16);
            fb[j] = i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
        const int sh = 8 * (kb & 3);
#pragma unroll
        for (int i = 0; i < IM; ++i) {
            const int r = wm * (TM / WM) + i * 16 + fr, sw = (r >> 1) & 7;
            const i32x4 lo = *reinterpret_cast<const i32x4*>(base + r * QB + ((2 * fg) ^ sw) * 16), hi = *reinterpret_cast<const i32x4*>(base + r * QB + ((2 * fg + 1) ^ sw) * 16);
            const i32x8 fa = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if constexpr (DT == CNM_F32) {
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const bf16x8 xa = widen(fa[2 * h], fa[2 * h + 1], scale_float(wa[i], sh));
#pragma unroll
                    for (int j = 0; j < IN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(fb[j][2 * h], fb[j][2 * h + 1], scale_float(wb[j], sh)), xa, acc[i][j], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int j = 0; j < IN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, (int)((wb[j] >> sh) & 255u), 0, (int)((wa[i] >> sh) & 255u));
            }
        }
    }
    // the last products stay above the stores' bounds checks: a matrix instruction sunk into divergent code would find its scales written for
    // some lanes only
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) asm volatile("" : "+v"(acc[i][j]));
    typedef typename Elem<DT>::T T;
    T* c = static_cast<T*>(g.c);
    const bool four = (g.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(c) & (4 * sizeof(T) - 1)) == 0;
#pragma unroll
    for (int i = 0; i < IM; ++i) {
        const int m = m0 + wm * (TM / WM) + i * 16 + fr;
#pragma unroll
        for (int j = 0; j < IN; ++j) {
            const int n = n0 + wn * (TN / WN) + j * 16 + 4 * fg;
            if (m < g.M && n < g.N) {
                T* p = c + (size_t)m * g.ldc + n;
                if (four && n + 3 < g.N) {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    *reinterpret_cast<T4*>(p) = T4{Elem<DT>::down(acc[i][j][0]), Elem<DT>::down(acc[i][j][1]), Elem<DT>::down(acc[i][j][2]), Elem<DT>::down(acc[i][j][3])};
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (n + e < g.N) p[e] = Elem<DT>::down(acc[i][j][e]);
                }
            }
        }
    }
}

template <int DT>
int launch_matmul(MatArgs g, hipStream_t stream) {
    constexpr int TM = 128, TN = 128;
    g.tiles_m = cnm_ceil_div(g.M, TM); g.tiles_n = cnm_ceil_div(g.N, TN);
    matmul_fp8_kernel<TM, TN, 2, 2, DT><<<g.tiles_m * g.tiles_n, 256, 2 * (TM + TN) * QB, stream>>>(g);
    CNM_LAUNCH_CHECK();
    return CNM_OK;
}

}  // namespace

extern "C" int cnm_quantize_fp8(const void* x, int dtype, long long ldx, long long rows, long long cols, int block_rows,
                                void* q, void* scale, void* q_t, void* scale_t, void* stream) {
    CNM_REQUIRE(x && rows > 0 && cols > 0 && ldx >= cols && (block_rows == 1 || block_rows == QB), CNM_ERR_BAD_ARG);
    CNM_REQUIRE((q || q_t) && !q == !scale && !q_t == !scale_t, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_t)) & 15) == 0, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(rows < (1ll << 31) - QB && cols < (1ll << 31) - QB && cnm_ceil_div_ll(rows, QB) * cnm_ceil_div_ll(cols, QB) < (1ll << 31), CNM_ERR_BAD_SHAPE);
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

extern "C" int cnm_matmul_fp8(const void* a, const void* a_scale, const void* b, const void* b_scale, int b_block_rows, void* c, int dtype,
                              long long ldc, long long M, long long N, long long K, void* stream) {
    CNM_REQUIRE(a && a_scale && b && b_scale && c && M > 0 && N > 0 && K > 0 && K % QB == 0 && ldc >= N, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(b_block_rows == 1 || b_block_rows == QB, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0, CNM_ERR_BAD_ARG);
    CNM_REQUIRE(M < (1ll << 31) - 256 && N < (1ll << 31) - 256 && K <= (1ll << 23), CNM_ERR_BAD_SHAPE);   // 256 rows of an operand are one 32-bit buffer range
    CNM_REQUIRE(cnm_ceil_div_ll(M, 16) * cnm_ceil_div_ll(N, 16) < (1ll << 31), CNM_ERR_BAD_SHAPE);
    MatArgs g = {static_cast<const unsigned char*>(a), static_cast<const unsigned char*>(a_scale), static_cast<const unsigned char*>(b), static_cast<const unsigned char*>(b_scale),
                 c, (int)M, (int)N, (int)(K / QB), b_block_rows == 1 ? 0 : 7, ldc, 0, 0};
    switch (dtype) {
        case CNM_F32: return launch_matmul<CNM_F32>(g, cnm_stream(stream));
        case CNM_F16: return launch_matmul<CNM_F16>(g, cnm_stream(stream));
        case CNM_BF16: return launch_matmul<CNM_BF16>(g, cnm_stream(stream));
    }
    return CNM_ERR_BAD_ARG;
}
