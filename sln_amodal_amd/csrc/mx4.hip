// Microscaled 4-bit operands: rounding, values, and the product of two rounded matrices (gfx950).
//
// Format (the OCP microscaling MXFP4 one): 32 neighbouring values of a row share a power-of-two scale
//   2^s, s = clamp(floor(log2 max|x|) - 2, -127, 127)   (all zero: s = -127),
// each value is the e2m1 number (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) nearest to x / 2^s, ties to the even
// code, saturated at 6.  A block that holds an infinity or a NaN gets scale code 255: all of its values are NaN, and so
// is every sum they enter.
//
// Memory: codes, two per byte, the lower nibble first; a row is padded with zero codes to whole steps of MX_STEP = 256
// values (128 B: one cache line and one LDS-DMA row); scales, one byte s + 127 per block, [Kp / 256][R][8] (mx_scale_at).
// Padding blocks have scale code 0.
//
// Product y[m][n] = act(sum_k a[m][k] b[n][k] * scale[n] + bias[n]) on v_mfma_scale_f32_32x32x64_f8f6f4 /
// 16x16x128: a lane's operand is 32 codes of ONE row = one block, with that block's scale: nothing is unpacked, the
// scales enter the instruction as a byte of a register.  Products of two values are exact, sums are fp32.
#include "mx4.h"

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// ------------------------------------------------------------------------------------------------ rounding
// Eight values of a thread, four neighbouring threads a block: amax over |bits| (a NaN is the largest).
__device__ __forceinline__ unsigned mx_absbits(const float *v) {
    unsigned a = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = max(a, __float_as_uint(v[e]) & 0x7fffffffu);
    return a;
}
__device__ __forceinline__ unsigned mx_scale_code(unsigned amax_bits) {
    const unsigned e = amax_bits >> 23;
    return e == 255u ? 255u : (e < 2u ? 0u : e - 2u);
}
__device__ __forceinline__ unsigned mx_codes8(const float *v, unsigned scale_code) {
    // 2^s as a float; s = -127 is subnormal
    const float s = __uint_as_float(scale_code ? scale_code << 23 : 0x00400000u);
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return scale_code == 255u ? 0u : q;
}

// One matrix to round: `threads` = rows * per_row, one thread per eight values of the padded row.
struct MxRound {
    const void *x;
    unsigned *codes;
    uint8_t *scales;
    int64_t stride, R, r0;               // rows of the whole matrix, first row of this job
    unsigned threads, per_row;
    int K, vec;
};

template <typename T>
__device__ __forceinline__ void mx_round8(const MxRound &p, unsigned at) {
    if (at >= p.threads) return;                    // whole blocks of 32: per_row is a multiple of 32 threads
    const unsigned row = at / p.per_row, c = at - row * p.per_row;
    float v[8];
    mx_load8((const T *)p.x + (int64_t)row * p.stride, (int)c * 8, p.K, p.vec, v);
    unsigned a = mx_absbits(v);
    a = max(a, (unsigned)__shfl_xor((int)a, 1));
    a = max(a, (unsigned)__shfl_xor((int)a, 2));
    const unsigned sc = mx_scale_code(a);
    p.codes[at] = mx_codes8(v, sc);
    if ((c & 3) == 0) p.scales[mx_scale_at(p.R, p.r0 + row, (int)(c >> 2))] = (uint8_t)sc;
}

// 4 (2) B read and 0.53 B written per value: bound by the read (1600 x 12544 f32: 14.6 us = 6.2 TB/s, the input in the
// Infinity Cache; 16000 x 12544: 157 us = 5.8 TB/s).  A second matrix (float32: the weight of a training step) rides in
// the same launch behind the first one's `blocks`.
template <typename T>
__global__ __launch_bounds__(256) void mx4_round_kernel(const MxRound a, const MxRound b, unsigned blocks) {
    if (blockIdx.x < blocks) mx_round8<T>(a, blockIdx.x * 256u + threadIdx.x);
    else mx_round8<float>(b, (blockIdx.x - blocks) * 256u + threadIdx.x);
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_values_kernel(const unsigned *__restrict__ codes,
                                                         const uint8_t *__restrict__ scales, int64_t R, int64_t r0,
                                                         unsigned rows, int K, unsigned per_row, T *__restrict__ out,
                                                         int vec) {
    const unsigned at = blockIdx.x * 256u + threadIdx.x;
    if (at >= rows * per_row) return;
    const unsigned row = at / per_row, c = at - row * per_row;
    if ((int)c * 8 >= K) return;
    float v[8];
    mx_values8(codes[at], scales[mx_scale_at(R, r0 + row, (int)(c >> 2))], v);
    mx_store8(out + (int64_t)row * K, (int)c * 8, K, vec, v);
}

// ------------------------------------------------------------------------------------------------ product, many rows
// Tile TA x TB, WR x WC waves; a step is 256 values of k = 128 B of every row, two LDS stages filled by DMA.  The order in
// which the eight blocks of a step enter the sum is free, so the two halves of a wave take blocks 0 ... 3 and 4 ... 7: a
// lane's four scales are one aligned dword of the scale row, and the instruction picks its byte.  The scales come by DMA
// too: with ordinary loads among the DMA's the compiler waits for all of them before the first LDS read of a step, and
// nothing overlaps (16000 x 12544 x 1024: 155 us instead of 130).
template <int TA_, int TB_, int WR_, int WC_>
struct MxShape {
    static constexpr int TA = TA_, TB = TB_, WR = WR_, WC = WC_, NW = WR * WC, THREADS = NW * 64;
    static constexpr int FA = TA / WR / 32, FB = TB / WC / 32, QA = TA / 8 / NW, QB = TB / 8 / NW;
    static constexpr int SCALES = (TA + TB) * 128, STAGE = SCALES + (TA + TB) * 8, LDS = 2 * STAGE;
    static constexpr int OCC = 163840 / LDS * NW / 4;                             // waves per SIMD
    static constexpr int RA = TA / NW, RB = TB / NW;                              // rows whose scales a wave fetches
    static_assert(RA <= 32 && RB <= 32, "64 lanes fetch two dwords of at most 32 rows");
};
// Small: two workgroups per CU (1000 x 12544 x 1024: 20 us, with four waves each 24).  Large: one (16000 rows: 130 us; with
// 16 waves 128, small tiles 155; 256 x 128 with a third stage 168: the reads out of L2, not their latency, are the bound).
typedef MxShape<128, 128, 2, 4> MxSmall;
typedef MxShape<256, 256, 2, 4> MxLarge;
struct MxGemm {
    const uint8_t *a, *b, *sa, *sb;
    int64_t a_pitch, b_pitch;          // bytes per code row
    int M, N, steps, nsplit;
    const float *scale, *bias;
    void *y;
    float *slab;                       // nsplit > 1: [nsplit][M][N] partial sums
    int relu;
};

// One rounding for scale, one for bias, one to the type, so that every kernel of this file, with and without ReLU, ends
// alike.  (The file is built with contraction on: without the pragma these are fused multiply-adds, in float16 without a
// rounding between the sum and the type.)
__device__ __forceinline__ float mx_act(float v, float scale, float bias, int relu) {
#pragma clang fp contract(off)
    v = v * scale;
    v = v + bias;
    return relu && v < 0.f ? 0.f : v;              // (a NaN stays)
}
template <typename T>
__device__ __forceinline__ void mx_finish(const MxGemm &p, int m, int n, float v) {
    ((T *)p.y)[(int64_t)m * p.N + n] = (T)mx_act(v, p.scale ? p.scale[n] : 1.f, p.bias ? p.bias[n] : 0.f, p.relu);
}

// (a vector type: behind a read of HIP's int4 the compiler waits for the DMA in flight)
__device__ __forceinline__ i32x8 mx_frag(const char *at) {
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    const i32x4 v = *(const i32x4 *)at;
    const i32x8 r = {v.x, v.y, v.z, v.w, 0, 0, 0, 0};
    return r;
}

template <typename T, typename S>
__global__ __launch_bounds__(S::THREADS, S::OCC) void mx4_product_kernel(const MxGemm p, int tiles) {
#ifdef __HIP_DEVICE_COMPILE__                      // (the host pass knows no buffer descriptors in templates)
    constexpr int NW = S::NW, OPA = S::TA * 128;
    __shared__ __attribute__((aligned(128))) char smem[S::LDS];
    const int at = nt_xcd_order(blockIdx.x, tiles);
    const int tn = (p.N + S::TB - 1) / S::TB;
    const int split = at % p.nsplit, tile = at / p.nsplit;
    const int m0 = tile / tn * S::TA, n0 = tile % tn * S::TB;
    const int s0 = (int)((int64_t)p.steps * split / p.nsplit), s1 = (int)((int64_t)p.steps * (split + 1) / p.nsplit);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wr = wave / S::WC, wc = wave % S::WC;
    const int half = lane >> 5, frow = lane & 31;
    unsigned aoff[S::QA], boff[S::QB];
#pragma unroll
    for (int q = 0; q < S::QA; ++q) {
        const int slot = (q * NW + wave) * 64 + lane, row = slot >> 3, c = (slot & 7) ^ ((row >> 1) & 7);
        aoff[q] = (unsigned)(min(row, p.M - 1 - m0) * p.a_pitch + c * 16);
    }
#pragma unroll
    for (int q = 0; q < S::QB; ++q) {
        const int slot = (q * NW + wave) * 64 + lane, row = slot >> 3, c = (slot & 7) ^ ((row >> 1) & 7);
        boff[q] = (unsigned)(min(row, p.N - 1 - n0) * p.b_pitch + c * 16);
    }
    const uint8_t *ga = p.a + (int64_t)m0 * p.a_pitch, *gb = p.b + (int64_t)n0 * p.b_pitch;
    // scales: lane l of wave w fetches dword l & 1 of rows RA w + l / 2 and RB w + l / 2
    const unsigned qa = (unsigned)min(m0 + S::RA * wave + (lane >> 1), p.M - 1) * 8u + (lane & 1) * 4u;
    const unsigned qb = (unsigned)min(n0 + S::RB * wave + (lane >> 1), p.N - 1) * 8u + (lane & 1) * 4u;
    const __amdgpu_buffer_rsrc_t ra = nt_buffer(ga, INT64_MAX), rb = nt_buffer(gb, INT64_MAX);
    auto issue = [&](int s, int stage) {
        char *l = smem + stage * S::STAGE + wave * 1024;
#pragma unroll
        for (int q = 0; q < S::QA; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (nt_lds *)(l + q * (NW * 1024)), 16, aoff[q], (unsigned)s * 128u, 0,
                                                     0);
#pragma unroll
        for (int q = 0; q < S::QB; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (nt_lds *)(l + OPA + q * (NW * 1024)), 16, boff[q],
                                                     (unsigned)s * 128u, 0, 0);
        char *ls = smem + stage * S::STAGE + S::SCALES;
        if (S::RA == 32 || lane < 2 * S::RA)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(nt_buffer(p.sa + (int64_t)s * p.M * 8, INT64_MAX),
                                                     (nt_lds *)(ls + wave * (S::RA * 8)), 4, qa, 0, 0, 0);
        if (S::RB == 32 || lane < 2 * S::RB)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(nt_buffer(p.sb + (int64_t)s * p.N * 8, INT64_MAX),
                                                     (nt_lds *)(ls + S::TA * 8 + wave * (S::RB * 8)), 4, qb, 0, 0, 0);
    };
    f32x16 acc[S::FA][S::FB];
#pragma unroll
    for (int i = 0; i < S::FA; ++i)
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    if (s0 < s1) issue(s0, 0);
    for (int s = s0; s < s1; ++s) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int stage = (s - s0) & 1;
        if (s + 1 < s1) issue(s + 1, stage ^ 1);
        const char *la = smem + stage * S::STAGE, *lb = la + OPA;
        int ca[S::FA], cb[S::FB];
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
            ca[i] = *(const int *)(la + S::SCALES + (S::TA / S::WR * wr + 32 * i + frow) * 8 + 4 * half);
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
            cb[j] = *(const int *)(la + S::SCALES + (S::TA + S::TB / S::WC * wc + 32 * j + frow) * 8 + 4 * half);
#define MX_QUARTER(Q)                                                                                        \
        {                                                                                                    \
            i32x8 fa[S::FA], fb[S::FB];                                                                      \
            _Pragma("unroll") for (int j = 0; j < S::FB; ++j) {                                              \
                const int row = S::TB / S::WC * wc + 32 * j + frow;                                          \
                fb[j] = mx_frag(lb + row * 128 + (((4 * half + Q) ^ ((row >> 1) & 7)) << 4));                \
            }                                                                                                \
            _Pragma("unroll") for (int i = 0; i < S::FA; ++i) {                                              \
                const int row = S::TA / S::WR * wr + 32 * i + frow;                                          \
                fa[i] = mx_frag(la + row * 128 + (((4 * half + Q) ^ ((row >> 1) & 7)) << 4));                \
            }                                                                                                \
            _Pragma("unroll") for (int i = 0; i < S::FA; ++i)                                                \
                _Pragma("unroll") for (int j = 0; j < S::FB; ++j)                                            \
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], 4,  \
                                                                                4, Q, ca[i], Q, cb[j]);      \
        }
        MX_QUARTER(0)
        MX_QUARTER(1)
        MX_QUARTER(2)
        MX_QUARTER(3)
#undef MX_QUARTER
    }
    // a lane's elements are rows row0 + 32 i + (r & 3) + 8 (r >> 2): uniform steps from one address
    const int row0 = m0 + S::TA / S::WR * wr + 4 * half, col0 = n0 + S::TB / S::WC * wc + frow;
    const bool inside = m0 + S::TA <= p.M && n0 + S::TB <= p.N;                   // (uniform: no test per element)
    const int64_t first = (int64_t)row0 * p.N + col0;
    const bool part = p.nsplit > 1;
    float *slab = part ? p.slab + (int64_t)split * p.M * p.N + first : nullptr;
    T *y = (T *)p.y + first;
#pragma unroll
    for (int j = 0; j < S::FB; ++j) {
        const int n = min(col0 + 32 * j, p.N - 1);
        const float cs = !part && p.scale ? p.scale[n] : 1.f, cb = !part && p.bias ? p.bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int down = 32 * i + (r & 3) + 8 * (r >> 2);
                if (!inside && (row0 + down >= p.M || col0 + 32 * j >= p.N)) continue;
                const int64_t e = (int64_t)down * p.N + 32 * j;
                if (part) slab[e] = acc[i][j][r];
                else y[e] = (T)mx_act(acc[i][j][r], cs, cb, p.relu);
            }
    }
#endif
}

// The cuts of the contraction, added in order, and the epilogue.  (1000 x 1024, four cuts: 5.8 us, 20 MB.)
template <typename T>
__global__ __launch_bounds__(256) void mx4_join_kernel(const MxGemm p) {
    const int64_t total = (int64_t)p.M * p.N;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int k = 0; k < p.nsplit; ++k) v += p.slab[k * total + e];
        const int m = (int)(e / p.N);
        mx_finish<T>(p, m, (int)(e - (int64_t)m * p.N), v);
    }
}

// ------------------------------------------------------------------------------------------------ product, few rows
// Up to 16 rows of x, not rounded yet: the weight's codes are the traffic (K N / 2 B) and are read straight into
// registers, 16 output channels x 128 values per instruction; a lane rounds its own block of x (32 values of one row) in
// registers, so there is no launch in front of this one.  Four waves cut a workgroup's part of the contraction, the
// grid cuts it further until the chip is full; the sums meet in LDS, then (several cuts) in mx4_join_kernel.  Bound by
// latency: one row of 12544 by 1024 outputs (6.8 MB of codes) 15 us with its launches, where a copy takes 1.5.
template <typename T>
__global__ __launch_bounds__(256) void mx4_rows_kernel(const MxGemm p, const T *__restrict__ x, int64_t stride, int K,
                                                       int vec) {
    __shared__ float part[4][16][17];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int r16 = lane & 15, blk = lane >> 4;
    const int n0 = blockIdx.x * 16, split = blockIdx.y * 4 + wave, cuts = p.nsplit * 4;
    const int steps = p.steps * 2;                 // of 128 values
    const int s0 = (int)((int64_t)steps * split / cuts), s1 = (int)((int64_t)steps * (split + 1) / cuts);
    const int wrow = min(n0 + r16, p.N - 1);
    const uint8_t *wb = p.b + (int64_t)wrow * p.b_pitch + blk * 16;
    const uint8_t *ws = p.sb + (int64_t)wrow * 8 + blk;
    const T *xr = x + (int64_t)min(r16, p.M - 1) * stride;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = s0; s < s1; ++s) {
        const i32x8 fw = mx_frag((const char *)wb + (int64_t)s * 64);
        const int sw = ws[(int64_t)(s >> 1) * p.N * 8 + (s & 1) * 4];
        i32x8 fx = {0, 0, 0, 0, 0, 0, 0, 0};
        int sx = 0;
        const int k = s * 128 + blk * 32;
        if (r16 < p.M && k < K) {
            float v[4][8];
            unsigned a = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                mx_load8(xr, k + q * 8, K, vec, v[q]);
                a = max(a, mx_absbits(v[q]));
            }
            sx = (int)mx_scale_code(a);
#pragma unroll
            for (int q = 0; q < 4; ++q) fx[q] = (int)mx_codes8(v[q], (unsigned)sx);
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw, fx, acc, 4, 4, 0, sw, 0, sx);
    }
    // rows of the result block: output channels 4 blk ... 4 blk + 3, column: row of x
#pragma unroll
    for (int r = 0; r < 4; ++r) part[wave][r16][4 * blk + r] = acc[r];
    __syncthreads();
    const int m = t >> 4, n = n0 + (t & 15);
    if (m >= p.M || n >= p.N) return;
    const float v = (part[0][m][t & 15] + part[1][m][t & 15]) + (part[2][m][t & 15] + part[3][m][t & 15]);
    if (p.nsplit > 1) p.slab[((int64_t)blockIdx.y * p.M + m) * p.N + n] = v;
    else mx_finish<T>(p, m, n, v);
}

// ------------------------------------------------------------------------------------------------ host side
static inline int mx_bad_dtype(int d) { return d != SLN_DTYPE_F32 && d != SLN_DTYPE_BF16 && d != SLN_DTYPE_F16; }

extern "C" int64_t sln_mx4_row_values(int64_t K) { return K < 0 ? 0 : (K + MX_STEP - 1) / MX_STEP * MX_STEP; }

// Rows [r, r + n) of a matrix, n * per_row < 2^31.
static MxRound mx_round_job(const void *x, int es, int64_t stride, int64_t R, int64_t r, int64_t n, int K,
                            uint8_t *codes, uint8_t *scales) {
    const int64_t kp = sln_mx4_row_values(K);
    MxRound p;
    p.x = (const char *)x + r * stride * es;
    p.codes = (unsigned *)(codes + r * (kp / 2));
    p.scales = scales;
    p.stride = stride;
    p.R = R;
    p.r0 = r;
    p.per_row = (unsigned)(kp / 8);
    p.threads = (unsigned)n * p.per_row;
    p.K = K;
    p.vec = ((uintptr_t)x % 16 == 0) && (stride * es) % 16 == 0;
    return p;
}
static inline int64_t mx_round_rows(int64_t K) { return ((int64_t)1 << 31) / (sln_mx4_row_values(K) / 8); }

template <typename T>
static void mx_round(const void *x, int64_t stride, int64_t R, int K, uint8_t *codes, uint8_t *scales, const MxRound *also,
                     hipStream_t st) {
    const int64_t most = mx_round_rows(K);
    MxRound none = {};
    for (int64_t r = 0; r < R; r += most) {
        const MxRound a = mx_round_job(x, sizeof(T), stride, R, r, R - r < most ? R - r : most, K, codes, scales);
        const MxRound b = also && r == 0 ? *also : none;
        const unsigned blocks = (a.threads + 255u) / 256u;
        hipLaunchKernelGGL((mx4_round_kernel<T>), dim3(blocks + (b.threads + 255u) / 256u), dim3(256), 0, st, a, b, blocks);
    }
}

extern "C" int sln_mx4_round(const void *x, int dtype, int64_t R, int64_t K, int64_t stride, uint8_t *codes,
                             uint8_t *scales, sln_stream_t stream) {
    if (mx_bad_dtype(dtype) || R < 0 || K < 1 || K > MX_MAX_K || stride < K) return SLN_ERR_INVALID_ARG;
    if (R == 0) return SLN_OK;
    if (!x || !codes || !scales || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 7)) return SLN_ERR_INVALID_ARG;
    sln_enter();
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SLN_DTYPE_F32) mx_round<float>(x, stride, R, (int)K, codes, scales, nullptr, st);
    else if (dtype == SLN_DTYPE_BF16) mx_round<__bf16>(x, stride, R, (int)K, codes, scales, nullptr, st);
    else mx_round<_Float16>(x, stride, R, (int)K, codes, scales, nullptr, st);
    return sln_launch_status();
}

template <typename T>
static void mx_values(const uint8_t *codes, const uint8_t *scales, int64_t R, int K, void *out, hipStream_t st) {
    const int64_t kp = sln_mx4_row_values(K);
    const unsigned per_row = (unsigned)(kp / 8);
    const int64_t max_rows = ((int64_t)1 << 31) / per_row;
    const int vec = ((uintptr_t)out % 16 == 0) && (K * sizeof(T)) % 16 == 0;
    for (int64_t r = 0; r < R; r += max_rows) {
        const unsigned n = (unsigned)(R - r < max_rows ? R - r : max_rows);
        hipLaunchKernelGGL((mx4_values_kernel<T>), dim3((n * per_row + 255) / 256), dim3(256), 0, st,
                           (const unsigned *)(codes + r * (kp / 2)), scales, R, r, n, K, per_row,
                           (T *)out + r * K, vec);
    }
}

extern "C" int sln_mx4_values(const uint8_t *codes, const uint8_t *scales, int64_t R, int64_t K, void *out, int dtype,
                              sln_stream_t stream) {
    if (mx_bad_dtype(dtype) || R < 0 || K < 1 || K > MX_MAX_K) return SLN_ERR_INVALID_ARG;
    if (R == 0) return SLN_OK;
    if (!out || !codes || !scales || ((uintptr_t)codes & 15)) return SLN_ERR_INVALID_ARG;
    sln_enter();
    hipStream_t st = (hipStream_t)stream;
    if (dtype == SLN_DTYPE_F32) mx_values<float>(codes, scales, R, (int)K, out, st);
    else if (dtype == SLN_DTYPE_BF16) mx_values<__bf16>(codes, scales, R, (int)K, out, st);
    else mx_values<_Float16>(codes, scales, R, (int)K, out, st);
    return sln_launch_status();
}

// Cuts of the contraction for M x N outputs of `steps` 256-value steps.
static inline int mx_cuts(int64_t tiles, int64_t target, int64_t steps, int64_t least) {
    int64_t c = target / (tiles < 1 ? 1 : tiles), most = steps / least;
    if (c > most) c = most;
    if (c > 64) c = 64;
    return c < 1 ? 1 : (int)c;
}
static inline int mx_rows_cuts(int64_t N, int64_t K) {
    return mx_cuts((N + 15) / 16, 512, 2 * ((K + MX_STEP - 1) / MX_STEP), 8);
}
static inline int64_t mx_tiles(int64_t M, int64_t N, int tile) { return ((M + tile - 1) / tile) * ((N + tile - 1) / tile); }
// Large tiles where three quarters of the CUs get one (16000 x 12544 x 1024: 155 us with 128 x 128, 130 so).
static inline bool mx_large(int64_t M, int64_t N) { return mx_tiles(M, N, 256) >= 192; }
static inline int mx_product_cuts(int64_t M, int64_t N, int64_t K) {
    return mx_large(M, N) ? 1 : mx_cuts(mx_tiles(M, N, 128), 256, (K + MX_STEP - 1) / MX_STEP, 2);
}

extern "C" size_t sln_mx4_product_workspace_bytes(int64_t M, int64_t N, int64_t K, int rounded) {
    if (M < 1 || N < 1 || K < 1) return 0;
    const int c = rounded ? mx_product_cuts(M, N, K) : mx_rows_cuts(N, K);
    return c > 1 ? (size_t)c * M * N * 4 : 0;
}

template <typename T>
static void mx_join(const MxGemm &p, hipStream_t st) {
    if (p.nsplit == 1) return;
    const int64_t blocks = ((int64_t)p.M * p.N + 255) / 256;
    hipLaunchKernelGGL((mx4_join_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, p);
}

static int mx_gemm(MxGemm &p, const uint8_t *b, const uint8_t *sb, int64_t M, int64_t N, int64_t K, const float *scale,
                   const float *bias, int relu, void *y, int nsplit, void *ws, size_t ws_bytes) {
    if (M > (1 << 28) || N > (1 << 28) || K > MX_MAX_K) return SLN_ERR_UNSUPPORTED;   // rows of scales below 2^32 B
    if (!b || !sb || !y || ((uintptr_t)b & 15) || ((uintptr_t)sb & 7)) return SLN_ERR_INVALID_ARG;
    p.b = b; p.sb = sb; p.b_pitch = sln_mx4_row_values(K) / 2;
    p.M = (int)M; p.N = (int)N; p.steps = (int)(sln_mx4_row_values(K) / MX_STEP);
    p.scale = scale; p.bias = bias; p.relu = relu; p.y = y;
    p.nsplit = nsplit;
    p.slab = (float *)ws;
    if (p.nsplit > 1 && (!ws || ((uintptr_t)ws & 3) || ws_bytes < (size_t)p.nsplit * M * N * 4)) return SLN_ERR_WORKSPACE;
    return SLN_OK;
}

extern "C" int sln_mx4_product(const uint8_t *a_codes, const uint8_t *a_scales, const uint8_t *b_codes,
                               const uint8_t *b_scales, int64_t M, int64_t N, int64_t K, const float *scale,
                               const float *bias, int relu, void *y, int dtype, void *workspace, size_t workspace_bytes,
                               sln_stream_t stream) {
    if (mx_bad_dtype(dtype) || M < 0 || N < 0 || K < 1) return SLN_ERR_INVALID_ARG;
    if (M == 0 || N == 0) return SLN_OK;
    MxGemm p = {};
    const int rc = mx_gemm(p, b_codes, b_scales, M, N, K, scale, bias, relu, y, mx_product_cuts(M, N, K), workspace,
                           workspace_bytes);
    if (rc != SLN_OK) return rc;
    if (!a_codes || !a_scales || ((uintptr_t)a_codes & 15) || ((uintptr_t)a_scales & 7)) return SLN_ERR_INVALID_ARG;
    p.a = a_codes; p.sa = a_scales; p.a_pitch = p.b_pitch;
    const bool large = mx_large(M, N);
    const int64_t tiles = mx_tiles(M, N, large ? 256 : 128) * p.nsplit;
    if (tiles > (1 << 30)) return SLN_ERR_UNSUPPORTED;
    sln_enter();
    hipStream_t st = (hipStream_t)stream;
#define MX_GO(T)                                                                                             \
    if (large)                                                                                               \
        hipLaunchKernelGGL((mx4_product_kernel<T, MxLarge>), dim3((unsigned)tiles), dim3(MxLarge::THREADS),  \
                           0, st, p, (int)tiles);                                                            \
    else                                                                                                     \
        hipLaunchKernelGGL((mx4_product_kernel<T, MxSmall>), dim3((unsigned)tiles), dim3(MxSmall::THREADS),  \
                           0, st, p, (int)tiles);                                                            \
    mx_join<T>(p, st)
    if (dtype == SLN_DTYPE_F32) { MX_GO(float); }
    else if (dtype == SLN_DTYPE_BF16) { MX_GO(__bf16); }
    else { MX_GO(_Float16); }
#undef MX_GO
    return sln_launch_status();
}

extern "C" int sln_mx4_rows_product(const void *x, int dtype, int64_t M, int64_t K, int64_t stride,
                                    const uint8_t *b_codes, const uint8_t *b_scales, int64_t N, const float *scale,
                                    const float *bias, int relu, void *y, void *workspace, size_t workspace_bytes,
                                    sln_stream_t stream) {
    if (mx_bad_dtype(dtype) || M < 0 || N < 0 || K < 1 || stride < K) return SLN_ERR_INVALID_ARG;
    if (M == 0 || N == 0) return SLN_OK;
    if (M > 16) return SLN_ERR_UNSUPPORTED;
    if (!x) return SLN_ERR_INVALID_ARG;
    MxGemm p = {};
    const int rc = mx_gemm(p, b_codes, b_scales, M, N, K, scale, bias, relu, y, mx_rows_cuts(N, K), workspace,
                           workspace_bytes);
    if (rc != SLN_OK) return rc;
    const int64_t es = dtype == SLN_DTYPE_F32 ? 4 : 2;
    const int vec = ((uintptr_t)x % 16 == 0) && (stride * es) % 16 == 0;
    const dim3 grid((unsigned)((N + 15) / 16), (unsigned)p.nsplit);
    sln_enter();
    hipStream_t st = (hipStream_t)stream;
#define MX_GO(T)                                                                                                       \
    hipLaunchKernelGGL((mx4_rows_kernel<T>), grid, dim3(256), 0, st, p, (const T *)x, stride, (int)K, vec);            \
    mx_join<T>(p, st)
    if (dtype == SLN_DTYPE_F32) { MX_GO(float); }
    else if (dtype == SLN_DTYPE_BF16) { MX_GO(__bf16); }
    else { MX_GO(_Float16); }
#undef MX_GO
    return sln_launch_status();
}

extern "C" int sln_mx4_linear_fwd(const void *x, int dtype, int64_t M, int64_t K, int64_t stride, uint8_t *x_codes,
                                  uint8_t *x_scales, const float *w, int64_t w_stride, uint8_t *w_codes, uint8_t *w_scales,
                                  int64_t N, const float *scale, const float *bias, int relu, void *y, void *workspace,
                                  size_t workspace_bytes, sln_stream_t stream) {
    if (mx_bad_dtype(dtype) || M < 0 || N < 0 || K < 1 || K > MX_MAX_K || stride < K || (w && w_stride < K))
        return SLN_ERR_INVALID_ARG;
    if (M == 0 || N == 0) return SLN_OK;
    if (!x || !w_codes || !w_scales || ((uintptr_t)w_codes & 15) || ((uintptr_t)w_scales & 7)) return SLN_ERR_INVALID_ARG;
    if (x_codes && (!x_scales || ((uintptr_t)x_codes & 15) || ((uintptr_t)x_scales & 7))) return SLN_ERR_INVALID_ARG;
    if (!x_codes && M > 16) return SLN_ERR_UNSUPPORTED;
    if (workspace_bytes < sln_mx4_product_workspace_bytes(M, N, K, x_codes ? 1 : 0)) return SLN_ERR_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    sln_enter();
    const MxRound *also = nullptr;
    MxRound job;
    if (w) {
        if (x_codes && N <= mx_round_rows(K)) {
            job = mx_round_job(w, 4, w_stride, N, 0, N, (int)K, w_codes, w_scales);
            also = &job;
        } else {
            mx_round<float>(w, w_stride, N, (int)K, w_codes, w_scales, nullptr, st);
        }
    }
    if (!x_codes)
        return sln_mx4_rows_product(x, dtype, M, K, stride, w_codes, w_scales, N, scale, bias, relu, y, workspace,
                                    workspace_bytes, stream);
    if (dtype == SLN_DTYPE_F32) mx_round<float>(x, stride, M, (int)K, x_codes, x_scales, also, st);
    else if (dtype == SLN_DTYPE_BF16) mx_round<__bf16>(x, stride, M, (int)K, x_codes, x_scales, also, st);
    else mx_round<_Float16>(x, stride, M, (int)K, x_codes, x_scales, also, st);
    return sln_mx4_product(x_codes, x_scales, w_codes, w_scales, M, N, K, scale, bias, relu, y, dtype, workspace,
                           workspace_bytes, stream);
}
