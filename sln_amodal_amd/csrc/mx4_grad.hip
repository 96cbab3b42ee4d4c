// Straight-through gradients of the 4-bit layer y = act((x^ w^T) * scale + bias), x^ and w^ rounded (gfx950):
//
//   z = gy [y > 0],   gx = (z scale) w^,   gw = scale (z^T x^),   gb = sum over the rows of z
//
// (z is 0 where y is a NaN, as under the convolutions' masks; a NaN of x^ or w^ still reaches gw or gx.)
//
// The rounding passes its gradient through unchanged, saturated values included.  w^ and x^ are what the forward
// multiplied: e2m1 values times powers of two have two significant bits, so ONE bf16 part holds them exactly, and a
// float32 gradient is exactly the sum of three bf16 parts (8 bits of its significand each, cut, not rounded).
// Products of as many parts on the bf16 matrix instructions into fp32 accumulators are therefore the float32 products:
// nothing is rounded before the sum but z * scale, to float32.  (Parts below bf16's smallest normal, 2^-126, may be lost.)
// Three parts for float32 gradients and for z * scale of any type, two where a 16-bit z is taken as it is.  (z * scale cut
// to two parts, 16 bits, costs the sums of gx up to 2^-15 of their terms, all in one direction: of 1501 x 1024 bfloat16
// results over 324 outputs 0.6 % were not the nearest; with three parts 0.014 %, a float32 product's 0.023 %.  The third part
// takes 1600 x 12544 x 1024 in bfloat16, forward and both gradients in a graph, from 229 us to 269; without scale 224.)
//
// Both products contract along rows (mfma_nt.h): gx over the outputs, so w^ is laid out [K][N]; gw over the rows of the
// batch, so z is laid out [N][M] and x^ [K][M].
#include "mx4.h"

#define MG_PITCH 65

__device__ __forceinline__ void mg_cut(float v, int parts, __bf16 *h) {
    if (!(fabsf(v) < INFINITY)) {                  // one part carries it; inf - inf would make a NaN of an infinity
        h[0] = (__bf16)v;
        for (int p = 1; p < parts; ++p) h[p] = (__bf16)0.f;
        return;
    }
    for (int p = 0; p < parts; ++p) {
        const float c = __uint_as_float(__float_as_uint(v) & 0xffff0000u);
        h[p] = (__bf16)c;
        v -= c;
    }
}
// values k ... k + 7 (k a multiple of 8) of parts row `row`
template <int P>
__device__ __forceinline__ void mg_store8(char *base, int64_t row, int64_t row_bytes, int k, const float *v) {
    char *at = base + row * row_bytes + (k >> 5) * (64 * P) + (k & 31) * 2;
    b16x8 h[P];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        __bf16 q[P];
        mg_cut(v[e], P, q);
#pragma unroll
        for (int p = 0; p < P; ++p) h[p][e] = q[p];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) *(b16x8 *)(at + p * 64) = h[p];
}
__host__ __device__ __forceinline__ int64_t mg_row_bytes(int64_t k, int parts) { return (k + 31) / 32 * 64 * parts; }

// What has to be laid out, in one launch: blocks [0, split) cut 64 x 64 tiles of gy, [split, split + turn_w) turn tiles
// of the weight's codes, the rest tiles of x's.
struct MgPrep {
    const void *gy, *y;
    const float *scale;
    int64_t stride;
    int M, N, K;
    char *rows, *cols;                   // parts of z * scale (rows M) and of z^T (rows N), or NULL
    float *bias_part;                    // one sum per 64 rows and column, or NULL
    const unsigned *w_codes, *x_codes;
    const uint8_t *w_scales, *x_scales;
    char *wt, *xt;                       // [K][N], [K][M]
    unsigned split, turn_w;
};

template <typename T, int PX, int PW>
__device__ __forceinline__ void mg_split(const MgPrep &p, unsigned b, float *z, float (*s_bias)[64]) {
    const unsigned tn = (unsigned)(p.N + 63) / 64;
    const int t = threadIdx.x, m0 = (int)(b / tn) * 64, n0 = (int)(b % tn) * 64;
    const int M = p.M, N = p.N;
    float sum = 0.f;
    for (int i = t >> 6; i < 64; i += 4) {
        const int m = m0 + i, n = n0 + (t & 63);
        float v = 0.f;
        if (m < M && n < N) {
            v = (float)((const T *)p.gy)[(int64_t)m * p.stride + n];
            if (p.y && !((float)((const T *)p.y)[(int64_t)m * N + n] > 0.f)) v = 0.f;
        }
        z[i * MG_PITCH + (t & 63)] = v;
        sum += v;
    }
    s_bias[t >> 6][t & 63] = sum;
    __syncthreads();
    if (p.bias_part && t < 64 && n0 + t < N)
        p.bias_part[(int64_t)(m0 / 64) * N + n0 + t] = (s_bias[0][t] + s_bias[1][t]) + (s_bias[2][t] + s_bias[3][t]);
    if (p.rows) {
        const int64_t rb = mg_row_bytes(N, PX);
        const int npad = (N + 31) & ~31;
        for (int e = t; e < 512; e += 256) {
            const int i = e >> 3, k = (e & 7) * 8;
            if (m0 + i >= M || n0 + k >= npad) continue;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                v[q] = z[i * MG_PITCH + k + q];
                if (p.scale && n0 + k + q < N) v[q] *= p.scale[n0 + k + q];
            }
            mg_store8<PX>(p.rows, m0 + i, rb, n0 + k, v);
        }
    }
    if (p.cols) {
        const int64_t rb = mg_row_bytes(M, PW);
        const int mpad = (M + 31) & ~31;
        for (int e = t; e < 512; e += 256) {
            const int j = e >> 3, k = (e & 7) * 8;
            if (n0 + j >= N || m0 + k >= mpad) continue;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = z[(k + q) * MG_PITCH + j];
            mg_store8<PW>(p.cols, n0 + j, rb, m0 + k, v);
        }
    }
}

// Codes [R][K] -> bf16 values as parts rows [K][R].  A block turns 64 x 64.
__device__ __forceinline__ void mg_turn(const unsigned *codes, const uint8_t *scales, int R, int K, char *out, unsigned b,
                                        float *z) {
    const unsigned tk = (unsigned)(K + 63) / 64;
    const int t = threadIdx.x, r0 = (int)(b / tk) * 64, k0 = (int)(b % tk) * 64;
    const int64_t kp = (int64_t)(K + MX_STEP - 1) / MX_STEP * MX_STEP;
    for (int e = t; e < 512; e += 256) {
        const int i = e >> 3, k = k0 + (e & 7) * 8;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (r0 + i < R) {                      // (k < kp: the padded row holds whole tiles of 64)
            const int64_t at = (int64_t)(r0 + i) * (kp / 8) + k / 8;
            mx_values8(codes[at], scales[mx_scale_at(R, r0 + i, k >> 5)], v);
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) z[i * MG_PITCH + (e & 7) * 8 + q] = v[q];
    }
    __syncthreads();
    const int64_t rb = mg_row_bytes(R, 1);
    const int rpad = (R + 31) & ~31;
    for (int e = t; e < 512; e += 256) {
        const int j = e >> 3, i = (e & 7) * 8;
        if (k0 + j >= K || r0 + i >= rpad) continue;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = z[(i + q) * MG_PITCH + j];
        mg_store8<1>(out, k0 + j, rb, r0 + i, v);
    }
}

template <typename T, int PX, int PW>
__global__ __launch_bounds__(256) void mx4_grad_prep_kernel(const MgPrep p) {
    __shared__ float z[64 * MG_PITCH];
    __shared__ float s_bias[4][64];
    if (blockIdx.x < p.split) mg_split<T, PX, PW>(p, blockIdx.x, z, s_bias);
    else if (blockIdx.x < p.split + p.turn_w) mg_turn(p.w_codes, p.w_scales, p.N, p.K, p.wt, blockIdx.x - p.split, z);
    else mg_turn(p.x_codes, p.x_scales, p.M, p.K, p.xt, blockIdx.x - p.split - p.turn_w, z);
}

// Where there are enough of them, 128 x 256 tiles of eight waves, two workgroups per CU: sixteen waves hide each other's
// loads and stores (1600 x 12544 x 1024, three parts, both gradients: 230 us; 128 x 128 tiles of four waves 285, 256 x 256
// tiles, one workgroup per CU, 281, though their k-loop alone is the fastest): 247 GFLOP of products, 1.07 PFLOP/s of the
// 1.30 that the library's bf16 product reaches.
// (Small ones: eight waves too; 1501 x 1024 x 324 bf16, both directions: 49 us without scale, with it, three parts, 52; two
// parts with four waves took 52.)
template <int P> struct MgSmall : NtShape<P, 1, 128, 128, 2, 4, 2> {};
template <int P> struct MgLarge : NtShape<P, 1, 128, 256, 2, 4, 2> {};

struct MgProduct {
    const char *a, *b;            // parts rows: a [RA] of P parts, b [RB] of one
    int RA, RB, groups, nsplit;
    unsigned tiles;               // of the launch, cuts included
    const float *row_scale;       // per row of the result, or NULL
    void *c;                      // [RA][RB]
    float *slab;                  // nsplit > 1: [nsplit][RA][RB]
};

template <typename T, typename S>
__device__ __forceinline__ void mg_product(const MgProduct &p, int at, char *smem) {
    const int ta = (p.RA + S::TA - 1) / S::TA;
    const int split = at % p.nsplit, tile = at / p.nsplit;
    const int i0 = tile % ta * S::TA, j0 = tile / ta * S::TB;
    const int64_t ra = (int64_t)p.groups * 64 * S::PA, rb = (int64_t)p.groups * 64;
    const int g0 = (int)((int64_t)p.groups * split / p.nsplit), g1 = (int)((int64_t)p.groups * (split + 1) / p.nsplit);
    f32x16 acc[S::FA][S::FB];
    nt_tile<S, b16x8, NT_EXACTB, false>(p.a + i0 * ra, ra, p.RA - i0, 0, p.b + j0 * rb, rb, p.RB - j0, g0, g1, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // a lane's elements are rows row0 + 32 i + (r & 3) + 8 (r >> 2): uniform steps from one address
    const int row0 = i0 + S::TA / S::WR * (wave / S::WC) + 4 * (lane >> 5);
    const int col0 = j0 + S::TB / S::WC * (wave % S::WC) + (lane & 31);
    const bool inside = i0 + S::TA <= p.RA && j0 + S::TB <= p.RB;                 // (uniform: no test per element)
    const int64_t first = (int64_t)row0 * p.RB + col0;
    const bool part = p.nsplit > 1;
    float *slab = part ? p.slab + (int64_t)split * p.RA * p.RB + first : nullptr;
    T *c = (T *)p.c + first;
#pragma unroll
    for (int i = 0; i < S::FA; ++i) {
        float rs[16];                              // (loads ahead of the stores, which the compiler may not pass)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            rs[r] = p.row_scale && !part ? p.row_scale[min(row0 + 32 * i + (r & 3) + 8 * (r >> 2), p.RA - 1)] : 1.f;
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int down = 32 * i + (r & 3) + 8 * (r >> 2);
                if (!inside && (row0 + down >= p.RA || col0 + 32 * j >= p.RB)) continue;
                const int64_t e = (int64_t)down * p.RB + 32 * j;
                if (part) slab[e] = acc[i][j][r];
                else c[e] = (T)(acc[i][j][r] * rs[r]);
            }
    }
}

// Both products (if their tiles are alike) and the bias sums in one launch (x: gx, w: gw; tiles = 0: not here); the tiles
// with the longer contraction first.  SX, SW: the same tile, as many parts as each first operand has.
template <typename T, typename SX, typename SW>
__global__ __launch_bounds__(SX::THREADS, 4) void mx4_grad_product_kernel(
    const MgProduct x, const MgProduct w, const float *__restrict__ bias_part, int bias_blocks, int N,
    float *__restrict__ gb) {
    static_assert(SX::THREADS == SW::THREADS, "one launch shape");
    __shared__ __attribute__((aligned(128))) char smem[SX::LDS > SW::LDS ? SX::LDS : SW::LDS];
    const bool w_first = w.groups > x.groups;
    const unsigned lead = w_first ? w.tiles : x.tiles, all = x.tiles + w.tiles;
    if (blockIdx.x < all) {
        const bool is_w = w_first == (blockIdx.x < lead);
        const int at = blockIdx.x < lead ? nt_xcd_order(blockIdx.x, lead) : nt_xcd_order(blockIdx.x - lead, all - lead);
        if (is_w) mg_product<float, SW>(w, at, smem);
        else mg_product<T, SX>(x, at, smem);
    } else {                                       // partial bias sums, added in order in double
        const int n = (blockIdx.x - all) * SX::THREADS + threadIdx.x;
        if (n >= N) return;
        double s = 0.0;
        for (int b = 0; b < bias_blocks; ++b) s += bias_part[(int64_t)b * N + n];
        gb[n] = (float)s;
    }
}

template <typename T>
__device__ __forceinline__ void mg_join(const MgProduct &p, int64_t first, int64_t step) {
    const int64_t total = (int64_t)p.RA * p.RB;
    for (int64_t e = first; e < total; e += step) {
        float v = 0.f;
        for (int k = 0; k < p.nsplit; ++k) v += p.slab[k * total + e];
        ((T *)p.c)[e] = (T)(p.row_scale ? v * p.row_scale[e / p.RB] : v);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void mx4_grad_join_kernel(const MgProduct x, const MgProduct w, unsigned blocks_x) {
    if (blockIdx.x < blocks_x) mg_join<T>(x, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)blocks_x * 256);
    else mg_join<float>(w, (int64_t)(blockIdx.x - blocks_x) * 256 + threadIdx.x, (int64_t)(gridDim.x - blocks_x) * 256);
}

// ------------------------------------------------------------------------------------------------ host side
struct MgPlan {
    int64_t z_rows, z_cols, wt, xt, bias, slab_x, slab_w, bytes;
    int gx_cuts, gw_cuts;
    bool gx_large, gw_large;
};
static inline int64_t mg_align(int64_t v) { return (v + 255) & ~(int64_t)255; }
static inline int64_t mg_tiles(int64_t RA, int64_t RB, bool large) {
    return ((RA + 127) / 128) * (large ? (RB + 255) / 256 : (RB + 127) / 128);
}
static inline bool mg_large(int64_t RA, int64_t RB) { return mg_tiles(RA, RB, true) >= 384; }   // 3/4 of the CUs' slots
static inline int mg_cuts(int64_t RA, int64_t RB, int64_t groups) {
    const int64_t tiles = mg_tiles(RA, RB, false);
    int64_t c = 512 / (tiles < 1 ? 1 : tiles);
    if (c > groups / 8) c = groups / 8;
    if (c > 32) c = 32;
    return c < 1 ? 1 : (int)c;
}
static void mg_plan(int64_t M, int64_t N, int64_t K, int px, int pw, bool gx, bool gw, bool gb, MgPlan &p) {
    int64_t at = 0;
    // (each product's own rule, whatever else is wanted: its bits do not depend on that)
    p.gx_large = mg_large(M, K);
    p.gw_large = mg_large(N, K);
    p.gx_cuts = p.gx_large ? 1 : mg_cuts(M, K, (N + 31) / 32);
    p.gw_cuts = p.gw_large ? 1 : mg_cuts(N, K, (M + 31) / 32);
    p.z_rows = at; at += gx ? mg_align(M * mg_row_bytes(N, px)) : 0;
    p.z_cols = at; at += gw ? mg_align(N * mg_row_bytes(M, pw)) : 0;
    p.wt = at; at += gx ? mg_align(K * mg_row_bytes(N, 1)) : 0;
    p.xt = at; at += gw ? mg_align(K * mg_row_bytes(M, 1)) : 0;
    p.bias = at; at += gb ? mg_align((M + 63) / 64 * N * 4) : 0;
    p.slab_x = at; at += gx && p.gx_cuts > 1 ? mg_align(p.gx_cuts * M * K * 4) : 0;
    p.slab_w = at; at += gw && p.gw_cuts > 1 ? mg_align(p.gw_cuts * N * K * 4) : 0;
    p.bytes = at;
}
// parts of z, and of z * scale
static inline int mg_parts(int dtype, bool scaled) { return dtype == SLN_DTYPE_F32 || scaled ? 3 : 2; }

extern "C" size_t sln_mx4_linear_bwd_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype, int want_gx, int want_gw,
                                                     int want_gb) {
    if (M < 1 || N < 1 || K < 1) return 0;
    MgPlan p;
    mg_plan(M, N, K, mg_parts(dtype, true), mg_parts(dtype, false), want_gx, want_gw, want_gb, p);   // with or without scale
    return (size_t)p.bytes;
}

static MgProduct mg_job(const char *a, int64_t RA, const char *b, int64_t RB, int64_t k, int cuts, bool large,
                        const float *row_scale, void *c, char *slab) {
    MgProduct p = {};
    if (!c) return p;
    p.a = a; p.b = b; p.RA = (int)RA; p.RB = (int)RB;
    p.groups = (int)((k + 31) / 32); p.nsplit = cuts;
    p.tiles = (unsigned)(mg_tiles(RA, RB, large) * cuts);
    p.row_scale = row_scale; p.c = c; p.slab = (float *)slab;
    return p;
}
static inline unsigned mg_join_blocks(const MgProduct &p) {
    if (p.tiles == 0 || p.nsplit == 1) return 0;
    const int64_t blocks = ((int64_t)p.RA * p.RB + 255) / 256;
    return (unsigned)(blocks < 4096 ? blocks : 4096);
}

template <typename T, int PX, int PW>
static void mg_run(const void *gy, int64_t stride, const void *y, const float *scale, const uint8_t *xc, const uint8_t *xs,
                   const uint8_t *wc, const uint8_t *wsc, int64_t M, int64_t N, int64_t K, void *gx, float *gw, float *gb,
                   const MgPlan &pl, char *ws, hipStream_t st) {
    MgPrep p = {};
    p.gy = gy; p.y = y; p.scale = scale; p.stride = stride;
    p.M = (int)M; p.N = (int)N; p.K = (int)K;
    p.rows = gx ? ws + pl.z_rows : nullptr;
    p.cols = gw ? ws + pl.z_cols : nullptr;
    p.bias_part = gb ? (float *)(ws + pl.bias) : nullptr;
    p.w_codes = (const unsigned *)wc; p.w_scales = wsc; p.wt = ws + pl.wt;
    p.x_codes = (const unsigned *)xc; p.x_scales = xs; p.xt = ws + pl.xt;
    const int64_t tm = (M + 63) / 64, tn = (N + 63) / 64, tk = (K + 63) / 64;
    p.split = (unsigned)(tm * tn);
    p.turn_w = gx ? (unsigned)(tk * tn) : 0u;
    hipLaunchKernelGGL((mx4_grad_prep_kernel<T, PX, PW>), dim3(p.split + p.turn_w + (gw ? (unsigned)(tk * tm) : 0u)), dim3(256),
                       0, st, p);
    const MgProduct jx = mg_job(ws + pl.z_rows, M, ws + pl.wt, K, N, pl.gx_cuts, pl.gx_large, nullptr, gx,
                                ws + pl.slab_x);
    const MgProduct jw = mg_job(ws + pl.z_cols, N, ws + pl.xt, K, M, pl.gw_cuts, pl.gw_large, scale, gw,
                                ws + pl.slab_w);
    const MgProduct none = {};
    auto launch = [&](const MgProduct &x, const MgProduct &w, bool large, float *bias) {
        const unsigned threads = MgSmall<PX>::THREADS;
        static_assert(MgSmall<PX>::THREADS == MgLarge<PX>::THREADS, "one launch shape");
        const dim3 grid(x.tiles + w.tiles + (bias ? (unsigned)(N + threads - 1) / threads : 0u));
        if (grid.x == 0) return;
        if (large)
            hipLaunchKernelGGL((mx4_grad_product_kernel<T, MgLarge<PX>, MgLarge<PW>>), grid, dim3(threads), 0, st, x, w, p.bias_part,
                               (int)tm, (int)N, bias);
        else
            hipLaunchKernelGGL((mx4_grad_product_kernel<T, MgSmall<PX>, MgSmall<PW>>), grid, dim3(threads), 0, st, x, w, p.bias_part,
                               (int)tm, (int)N, bias);
    };
    if (!gx || !gw || pl.gx_large == pl.gw_large) {
        launch(jx, jw, gx ? pl.gx_large : gw && pl.gw_large, gb);
    } else {
        launch(jx, none, pl.gx_large, gb);
        launch(none, jw, pl.gw_large, nullptr);
    }
    const unsigned bx = mg_join_blocks(jx), bw = mg_join_blocks(jw);
    if (bx + bw) hipLaunchKernelGGL((mx4_grad_join_kernel<T>), dim3(bx + bw), dim3(256), 0, st, jx, jw, bx);
}

extern "C" int sln_mx4_linear_bwd(const void *gy, int dtype, int64_t gy_stride, const void *y, const float *scale,
                                  const uint8_t *x_codes, const uint8_t *x_scales, const uint8_t *w_codes,
                                  const uint8_t *w_scales, int64_t M, int64_t N, int64_t K, void *gx, float *gw, float *gb,
                                  void *workspace, size_t workspace_bytes, sln_stream_t stream) {
    if ((dtype != SLN_DTYPE_F32 && dtype != SLN_DTYPE_BF16 && dtype != SLN_DTYPE_F16) || M < 1 || N < 1 || K < 1 ||
        gy_stride < N || !gy)
        return SLN_ERR_INVALID_ARG;
    // 128 rows below 2^32 B, and every launch below 2^31 blocks
    if (M > (1 << 21) || N > (1 << 21) || K > MX_MAX_K || (M + 63) / 64 * ((N + 63) / 64) > (1 << 28) ||
        (K + 63) / 64 * ((M + 63) / 64) > (1 << 28) || (K + 63) / 64 * ((N + 63) / 64) > (1 << 28))
        return SLN_ERR_UNSUPPORTED;
    if ((gx && (!w_codes || !w_scales)) || (gw && (!x_codes || !x_scales))) return SLN_ERR_INVALID_ARG;
    if ((gx && ((uintptr_t)w_codes & 15)) || (gw && ((uintptr_t)x_codes & 15))) return SLN_ERR_INVALID_ARG;
    MgPlan pl;
    mg_plan(M, N, K, mg_parts(dtype, scale != nullptr), mg_parts(dtype, false), gx, gw, gb, pl);
    if (pl.bytes && (!workspace || ((uintptr_t)workspace & 255))) return SLN_ERR_INVALID_ARG;
    if (workspace_bytes < (size_t)pl.bytes) return SLN_ERR_WORKSPACE;
    if (!gx && !gw && !gb) return SLN_OK;
    sln_enter();
    char *ws = (char *)workspace;
    hipStream_t st = (hipStream_t)stream;
#define MG_GO(T, PX, PW)                                                                                               \
    mg_run<T, PX, PW>(gy, gy_stride, y, scale, x_codes, x_scales, w_codes, w_scales, M, N, K, gx, gw, gb, pl, ws, st)
    if (dtype == SLN_DTYPE_F32) MG_GO(float, 3, 3);
    else if (dtype == SLN_DTYPE_BF16 && scale) MG_GO(__bf16, 3, 2);
    else if (dtype == SLN_DTYPE_BF16) MG_GO(__bf16, 2, 2);
    else if (scale) MG_GO(_Float16, 3, 2);
    else MG_GO(_Float16, 2, 2);
#undef MG_GO
    return sln_launch_status();
}
