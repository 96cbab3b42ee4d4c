// Newton-Schulz orthogonalisation of many matrices at once, and the optimiser step built on it (gfx950).
//
//   X <- G / (|G|_F + eps), on the transpose where G is taller than wide (so X is m x n, m <= n)
//   `steps` times:  A = X X^T,  P = a I + b A + c A^2,  X <- P X        (a, b, c) = (3.4445, -4.7750, 2.0315), the
//   coefficients published with the Muon optimiser
//
// maps every singular value s of X to p(s) = a s + b s^3 + c s^5, again and again: in five steps all of (0.005, 1] come
// into 0.68 ... 1.16, so X ends near the orthogonal factor U V^T of G.  p keeps [0, 1.21] inside [0, 1.21], hence
// |X|_2 <= 1.21, |A|_2 <= 1.47, |P|_2 <= 3.45 throughout and a FIXED power-of-two scale (2^14) puts every operand into
// fp16's range: an operand is two fp16 parts of value * 2^14 (22 ... 23 bits for values above 2^-17, an absolute floor of
// 2^-39 below), a product of two is three matrix instructions into an fp32 accumulator.  No pass looks for a maximum.
// Where eps outweighs |G| (|X|_F = r << 1) the operand holds X 2^h instead, h = floor(-log2 r) in the first step and two
// less in each later one (|X| grows by at most 3.45 < 4 a step): then A is held times 4^h.
//
// Launches (all matrices of a call in each of them; work lists in the workspace, made by the first launch):
//   ortho_norm_kernel    partial sums of squares in double (the optimiser: also the momentum update), the work lists
//   ortho_split_kernel   u = G / (|G| + eps) -> parts of X [m][n]
//   per step: ortho_gram_kernel    A's 128 x 128 tiles on and above the diagonal (A is symmetric), the contraction over n
//                                  cut so that one round of workgroups fills the chip; one cut: parts of A are written
//                                  (both triangles), several: fp32 partial tiles, added in order by ortho_join_kernel
//             ortho_poly_kernel    P's 64 x 64 tiles on and above the diagonal from A A^T, parts of both triangles
//             (both by ortho_square_kernel in calls with little to do)
//             ortho_apply_kernel   X <- P X; the last step writes the result, or updates the weights.
// Where the matrices are wide (ortho_pairs) two steps share their passes over X: P1 and A are symmetric and commute, so the
// second step's A is P1 A P1, and X <- (P2 P1) X once.  Three products of m^3 (ortho_poly_kernel's other kinds) instead of
// one of m^2 n and two of m^2 n.  The second A has up to a^2 = 12 times the first one's rounding errors; a pair is followed by
// a single step, five are 2 + 1 + 2: errors as without pairs, over all spectra that were tried (2 + 2 + 1 loses where half of
// the singular values are a tenth of the others: 6.7e-6, 2 + 1 + 2 1.0e-6, a float32 evaluation 1.8e-6).
// X is kept one way only, rows of n.  The Gram matrix contracts along its rows; P X contracts across them and computes
// (P X)^T with X as the first operand, read through LDS's transposing loads: the 16 accumulator values of a lane are then
// neighbours along n, and parts go straight from registers to X's rows, 16 bytes a store.
// A call whose matrices all fit one CU's LDS (ortho_small) is ONE launch instead, ortho_small_kernel: a workgroup per
// matrix runs all the steps on chip.
#include "mfma_nt.h"

#define ORTHO_BATCH 32                     // matrices per launch that takes descriptors by value
#define ORTHO_CHUNK 16384                  // elements per partial sum of squares
#define ORTHO_SCALE 16384.0f               // 2^14
#define ORTHO_UNSCALE 6.103515625e-05f     // 2^-14
#define ORTHO_A 3.4445f
#define ORTHO_B -4.7750f
#define ORTHO_C 2.0315f
#define GRAM_TILE 128

typedef NtShape<2, 2, 128, 128, 2, 4, 2> OrthoGram;
typedef NtShape<2, 2, 64, 64, 2, 2, 4> OrthoSquare;                // few workgroups: depth
typedef NtShape<2, 2, 64, 64, 2, 2, 3> OrthoPoly;                  // three on a CU (a detector's 125: 46 us; four stages 52)
typedef NtShape<2, 2, 128, 128, 2, 4, 2> OrthoApplySmall;
typedef NtShape<2, 2, 256, 256, 2, 4, 2> OrthoApplyLarge;

// What the launches are told about a matrix: by value to the first, a table in the workspace for the others.
struct OrthoProb {
    const void *g;         // rows x cols, row stride gs
    void *out;             // rows x cols, row stride os (the optimiser: the weights)
    float *buf;            // the optimiser's momentum, row stride cols; NULL: plain orthogonalisation
    int64_t gs, os, off;   // off: byte offset of this matrix's operands in the workspace
    int32_t rows, cols;
    int32_t part0, nparts; // its partial sums of squares
    int32_t split0, sym0, gram0, square0, apply0, last0, nsplit;    // first entries in the work lists, cuts of the contraction
    float lr, decay;       // update: p = p * decay - lr * X
    int32_t shift;         // h of the first step (ortho_split_kernel)
};

struct OrthoTile { int32_t prob, ij, first, cut; };        // ij = row tile << 16 | column tile; first: gram entry of cut 0

struct OrthoTable {
    OrthoProb *prob;
    OrthoTile *split, *sym, *gram, *square, *apply, *last;
    double *part;
    char *ws;
    float *slab;           // partial Gram tiles, GRAM_TILE^2 floats per gram entry
    int apply_tile;
};

struct OrthoBatch { OrthoProb p[ORTHO_BATCH]; };
struct OrthoRule {         // the optimiser's side of a call
    const double *sqnorm;
    float max_norm, momentum;
    int nesterov;
};

__host__ __device__ __forceinline__ int ortho_m(const OrthoProb &p) { return p.rows < p.cols ? p.rows : p.cols; }
__host__ __device__ __forceinline__ int ortho_n(const OrthoProb &p) { return p.rows < p.cols ? p.cols : p.rows; }
__host__ __device__ __forceinline__ int64_t ortho_row_bytes(int k) { return (int64_t)((k + 31) / 32) * 128; }
__host__ __device__ __forceinline__ int ortho_tiles(int v, int tile) { return (v + tile - 1) / tile; }

// operands of a matrix inside the workspace: X (two, in turn), A, P and, in calls that take steps in pairs, one more
struct OrthoOperands {
    char *x, *next, *a, *p, *t;                    // this turn's X, the next one's
};
__device__ __forceinline__ OrthoOperands ortho_operands(const OrthoProb &p, char *ws, int turn) {
    const int m = ortho_m(p), n = ortho_n(p);
    const int64_t bx = m * ortho_row_bytes(n);
    OrthoOperands o;
    o.x = ws + p.off + (turn & 1) * bx;
    o.next = ws + p.off + ((turn & 1) ^ 1) * bx;
    o.a = ws + p.off + 2 * bx;
    o.p = o.a + m * ortho_row_bytes(m);
    o.t = o.p + m * ortho_row_bytes(m);
    return o;
}
static int64_t ortho_operand_bytes(const OrthoProb &p, bool pairs) {
    const int m = ortho_m(p), n = ortho_n(p);
    return 2 * m * ortho_row_bytes(n) + (pairs ? 3 : 2) * m * ortho_row_bytes(m);
}

// 2^(sign h) for step `step`
__device__ __forceinline__ float ortho_shift(int shift, int step, int sign) {
    return ldexpf(1.f, sign * max(0, shift - 2 * step));
}
// h, and X = G up inv = G 2^h / (norm + eps), |G| up <= norm + eps.  (From 2^126 on 1 / (norm + eps) is no normal float32
// number and would hold too few bits: 2^64 of it goes into up.)
__device__ __forceinline__ float ortho_inverse(double sum, float eps, int &shift, float &up) {
    const double norm = sqrt(sum), r = norm / (norm + (double)eps);
    shift = 0;
    if (r > 0.0 && r < 1.0) {
        frexp(r, &shift);                          // r < 2^shift
        shift = min(max(-shift, 0), 126);
    }
    const int down = norm + (double)eps > 0x1p100 ? 64 : 0;
    up = ldexpf(1.f, shift - down);
    return (float)(ldexp(1.0, down) / (norm + (double)eps));
}

template <typename T>
__device__ __forceinline__ float ortho_load(const void *p, int64_t i) { return (float)((const T *)p)[i]; }

// The clip coefficient and the verdict of the optimiser's guard (a non-finite norm: the step is not applied).
__device__ __forceinline__ bool ortho_clip(const OrthoRule &rule, float &cf) {
    const double sq = rule.sqnorm[0];
    const double coef = (double)rule.max_norm / (sqrt(sq) + 1e-6);
    cf = coef < 1.0 ? (float)coef : 1.0f;
    return sq >= 0.0 && sq < INFINITY;
}
// One element of the momentum update (b is written if `apply`) and what is orthogonalised.
__device__ __forceinline__ float ortho_momentum(const OrthoRule &rule, float g, float cf, float &b) {
    const float gc = g * cf;
    b = rule.momentum * b + gc;
    return rule.nesterov ? gc + rule.momentum * b : b;
}
// The same from the momentum that is already updated.
__device__ __forceinline__ float ortho_update(const OrthoRule &rule, float g, float cf, float b) {
    return rule.nesterov ? g * cf + rule.momentum * b : b;
}

__device__ __forceinline__ double ortho_block_sum(double acc, double *s_red) {      // any whole number of waves
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = acc;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) s += s_red[w];
    return s;
}

// ------------------------------------------------------------------------------------------------ norms and lists
__device__ __forceinline__ void ortho_lists(const OrthoProb &p, int prob, const OrthoTable &tab) {
    const int t = threadIdx.x, m = ortho_m(p), n = ortho_n(p);
    if (t == 0) tab.prob[prob] = p;
    const int si = ortho_tiles(m, 64), sj = ortho_tiles(n, 128);
    for (int e = t; e < si * sj; e += 256) {
        const OrthoTile w = {prob, (e / sj) << 16 | (e % sj), 0, 0};
        tab.split[p.split0 + e] = w;
    }
    const int tm = ortho_tiles(m, GRAM_TILE), nsym = tm * (tm + 1) / 2;
    for (int e = t; p.nsplit > 0 && e < tm * tm; e += 256) {
        const int i = e / tm, j = e - i * tm;
        if (j < i) continue;
        const int s = i * tm - i * (i - 1) / 2 + (j - i);
        OrthoTile w = {prob, i << 16 | j, p.gram0 + s, 0};
        tab.sym[p.sym0 + s] = w;
        for (int k = 0; k < p.nsplit; ++k) {
            w.cut = k;
            tab.gram[p.gram0 + k * nsym + s] = w;
        }
    }
    const int tp = ortho_tiles(m, OrthoSquare::TA);
    for (int e = t; e < tp * tp; e += 256) {       // the whole square, or its upper triangle
        const int i = e / tp, j = e - i * tp;
        if (p.nsplit > 0 && j < i) continue;
        const OrthoTile w = {prob, i << 16 | j, 0, 0};
        tab.square[p.square0 + (p.nsplit > 0 ? i * tp - i * (i - 1) / 2 + (j - i) : e)] = w;
    }
    const int ti = ortho_tiles(m, tab.apply_tile), tj = ortho_tiles(n, tab.apply_tile);
    for (int e = t; e < ti * tj; e += 256) {       // the m tiles of one column of X run side by side
        const OrthoTile w = {prob, (e % ti) << 16 | (e / ti), 0, 0};
        tab.apply[p.apply0 + e] = w;
    }
    const int li = ortho_tiles(m, OrthoApplySmall::TB), lj = ortho_tiles(n, OrthoApplySmall::TA);
    for (int e = t; e < li * lj; e += 256) {
        const OrthoTile w = {prob, (e % li) << 16 | (e / li), 0, 0};
        tab.last[p.last0 + e] = w;
    }
}

// Block (c, i): elements [c, c + 1) * ORTHO_CHUNK of matrix i (row-major order) -> one partial sum of squares, added in a
// fixed order.  The optimiser (buf != NULL): b <- momentum b + cf g is written on the way and the sum is that of
// u = cf g + momentum b (nesterov) or u = b.  Memory-bound: 4 B read (optimiser: 8 read + 4 written) per element (63.9 M
// elements of an optimiser step, four launches: 182 us = 4.2 TB/s).
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoBatch batch, int prob0, OrthoTable tab, OrthoRule rule) {
    __shared__ double s_red[4];
    const OrthoProb &p = batch.p[blockIdx.y];
    const int t = threadIdx.x, chunk = blockIdx.x;
    if (chunk == 0) ortho_lists(p, prob0 + blockIdx.y, tab);
    if (chunk >= p.nparts) return;
    float cf = 1.f;
    bool apply = true;
    if (p.buf) apply = ortho_clip(rule, cf);
    const int64_t total = (int64_t)p.rows * p.cols, e0 = (int64_t)chunk * ORTHO_CHUNK;
    const int64_t e1 = min(total, e0 + ORTHO_CHUNK);
    double acc = 0.0;
    const bool flat = p.gs == p.cols;
    auto one = [&](float g, float *b) {
        float u = g;
        if (p.buf) {
            float nb = *b;
            u = ortho_momentum(rule, g, cf, nb);
            if (apply) *b = nb;
        }
        acc += (double)u * u;
    };
    if (flat && sizeof(T) == 2 && !((uintptr_t)p.g & 15)) {          // (never the optimiser's)
        typedef T t8 __attribute__((ext_vector_type(8)));
        const t8 *g8 = (const t8 *)p.g + (e0 >> 3);
        const int n8 = (int)((e1 - e0) >> 3);
        for (int i = t; i < n8; i += 256) {
            const t8 g = g8[i];
#pragma unroll
            for (int q = 0; q < 8; ++q) one((float)g[q], nullptr);
        }
        for (int64_t e = e0 + (int64_t)n8 * 8 + t; e < e1; e += 256) one(ortho_load<T>(p.g, e), nullptr);
    } else if (flat && sizeof(T) == 4 && !(((uintptr_t)p.g | (uintptr_t)p.buf) & 15)) {
        const float4 *g4 = (const float4 *)p.g + (e0 >> 2);
        const int n4 = (int)((e1 - e0) >> 2);
        for (int i = t; i < n4; i += 256) {
            const float4 g = g4[i];
            if (p.buf) {
                float4 *b4 = (float4 *)(p.buf + e0) + i;
                float4 b = *b4;
                one(g.x, &b.x); one(g.y, &b.y); one(g.z, &b.z); one(g.w, &b.w);
                if (apply) *b4 = b;
            } else {
                one(g.x, nullptr); one(g.y, nullptr); one(g.z, nullptr); one(g.w, nullptr);
            }
        }
        for (int64_t e = e0 + (int64_t)n4 * 4 + t; e < e1; e += 256)
            one(ortho_load<T>(p.g, e), p.buf ? p.buf + e : nullptr);
    } else {
        for (int64_t e = e0 + t; e < e1; e += 256) {
            int64_t ge = e;
            if (!flat) {
                const int64_t r = e / p.cols;
                ge = r * p.gs + (e - r * p.cols);
            }
            one(ortho_load<T>(p.g, ge), p.buf ? p.buf + e : nullptr);
        }
    }
    acc = ortho_block_sum(acc, s_red);
    if (t == 0) tab.part[p.part0 + chunk] = acc;
}

// ------------------------------------------------------------------------------------------------ parts
__device__ __forceinline__ void ortho_parts8(const float *v, f16x8 &h0, f16x8 &h1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float s = v[e] * ORTHO_SCALE;
        h0[e] = (_Float16)s;
        h1[e] = (_Float16)(s - (float)h0[e]);
    }
}
// value k ... k + 7 (k a multiple of 8) of row `row`
__device__ __forceinline__ char *ortho_at(char *base, int64_t row_bytes, int row, int k) {
    return base + row * row_bytes + (k >> 5) * 128 + (k & 31) * 2;
}
__device__ __forceinline__ void ortho_store8(char *at, const float *v) {
    f16x8 h0, h1;
    ortho_parts8(v, h0, h1);
    *(f16x8 *)at = h0;
    *(f16x8 *)(at + 64) = h1;
}

// ------------------------------------------------------------------------------------------------ G -> X
// Block = 64 x 128 of X.  Reads 4 B (optimiser: 8, u is made again from g and the new momentum), writes 4 B per element:
// bound by memory (63.9 M elements of an optimiser step: 169 us = 4.5 TB/s, a large copy's rate here 4.7).
template <typename T>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoTable tab, OrthoRule rule, float eps) {
    __shared__ float slab[64 * 129];
    __shared__ double s_red[4];
    const OrthoTile w = tab.split[blockIdx.x];
    const OrthoProb p = tab.prob[w.prob];
    const int t = threadIdx.x, m = ortho_m(p), n = ortho_n(p);
    double acc = 0.0;
    for (int i = t; i < p.nparts; i += 256) acc += tab.part[p.part0 + i];
    int shift;
    float up;
    const float inv = ortho_inverse(ortho_block_sum(acc, s_red), eps, shift, up);
    if (w.ij == 0 && t == 0) tab.prob[w.prob].shift = shift;
    float cf = 1.f;
    if (p.buf) ortho_clip(rule, cf);
    const bool tall = p.rows > p.cols;
    char *x = ortho_operands(p, tab.ws, 0).x;
    const int64_t rb = ortho_row_bytes(n);
    const int i0 = (w.ij >> 16) * 64, j0 = (w.ij & 0xffff) * 128, npad = (n + 31) & ~31;
    if (tall) {                                    // X = G^T: lanes along G's rows, turned in LDS
        for (int e = t; e < 64 * 128; e += 256) {
            const int i = e & 63, j = e >> 6;
            float v = 0.f;
            if (i0 + i < m && j0 + j < n) {
                v = ortho_load<T>(p.g, (int64_t)(j0 + j) * p.gs + i0 + i);
                if (p.buf) v = ortho_update(rule, v, cf, p.buf[(int64_t)(j0 + j) * p.cols + i0 + i]);
            }
            slab[i * 129 + j] = v * up * inv;
        }
        __syncthreads();
    }
    for (int e = t; e < 64 * 16; e += 256) {
        const int i = e >> 4, k = j0 + (e & 15) * 8;
        if (i0 + i >= m || k >= npad) continue;
        float v[8];
        if (tall) {
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = slab[i * 129 + (e & 15) * 8 + q];
        } else {
            const int64_t at = (int64_t)(i0 + i) * p.gs + k, bt = (int64_t)(i0 + i) * p.cols + k;
            float g[8], b[8];
            const bool wide = sizeof(T) == 4 && k + 8 <= n && !(((uintptr_t)((const float *)p.g + at)) & 15) &&
                              !(p.buf && ((uintptr_t)(p.buf + bt) & 15));
            typedef T t8 __attribute__((ext_vector_type(8)));
            if (sizeof(T) == 2 && k + 8 <= n && !(((uintptr_t)((const T *)p.g + at)) & 15)) {
                const t8 a = *(const t8 *)((const T *)p.g + at);
#pragma unroll
                for (int q = 0; q < 8; ++q) { g[q] = (float)a[q]; b[q] = 0.f; }
            } else if (wide) {
                *(float4 *)g = *(const float4 *)((const float *)p.g + at);
                *(float4 *)(g + 4) = *(const float4 *)((const float *)p.g + at + 4);
                if (p.buf) {
                    *(float4 *)b = *(const float4 *)(p.buf + bt);
                    *(float4 *)(b + 4) = *(const float4 *)(p.buf + bt + 4);
                }
            } else {
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    g[q] = k + q < n ? ortho_load<T>(p.g, at + q) : 0.f;
                    b[q] = p.buf && k + q < n ? p.buf[bt + q] : 0.f;
                }
            }
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = (p.buf ? ortho_update(rule, g[q], cf, b[q]) : g[q]) * up * inv;
        }
        ortho_store8(ortho_at(x, rb, i0 + i, k), v);
    }
}

// ------------------------------------------------------------------------------------------------ symmetric tiles
// A R x TILE slab (rows i0 ..., columns j0 ... of an m x m matrix) from LDS to parts of the matrix and, where `mirror`, of
// its transpose.  Values behind the last column (row) are the zeros that pad the contraction.  The pitch TILE + 5 is odd
// and 8 pitches are 40 mod 64: neither way of reading meets more than two lanes on a bank.
template <int R, int TILE, int THREADS>
__device__ __forceinline__ void ortho_store_sym(const float *slab, int i0, int j0, int m, char *dst, bool mirror) {
    const int t = threadIdx.x, mpad = (m + 31) & ~31;
    const int64_t rb = ortho_row_bytes(m);
    for (int e = t; e < R * (TILE / 8); e += THREADS) {
        const int r = e / (TILE / 8), c8 = e % (TILE / 8) * 8, k = j0 + c8;
        if (i0 + r >= m || k >= mpad) continue;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = k + q < m ? slab[r * (TILE + 5) + c8 + q] : 0.f;
        ortho_store8(ortho_at(dst, rb, i0 + r, k), v);
    }
    if (!mirror) return;
    for (int e = t; e < TILE * (R / 8); e += THREADS) {
        const int c = e / (R / 8), r8 = e % (R / 8) * 8, k = i0 + r8;
        if (j0 + c >= m || k >= mpad) continue;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = k + q < m ? slab[(r8 + q) * (TILE + 5) + c] : 0.f;
        ortho_store8(ortho_at(dst, rb, j0 + c, k), v);
    }
}

// Accumulators of slab h (the waves that hold rows TILE / 2 h ...) to LDS, in units of the values.
template <typename S>
__device__ __forceinline__ void ortho_slab_from_acc(float *slab, const f32x16 (&acc)[S::FA][S::FB], int h, float unscale) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave / S::WC != h) return;
#pragma unroll
    for (int i = 0; i < S::FA; ++i)
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                slab[(32 * i + nt_acc_row(r, lane)) * (S::TB + 5) + S::TB / S::WC * (wave % S::WC) + 32 * j + (lane & 31)] =
                    acc[i][j][r] * unscale;
}

// ------------------------------------------------------------------------------------------------ A = X X^T
// Bound by the matrix instructions and by LDS together: a k-step of 128 x 128 takes 768 clocks of products, and 96 KB of
// fragments and 32 KB of DMA at 128 B a clock 1024; the two workgroups of a CU cover each other's waits.  125 matrices of
// a detector (97 GFLOP of products, m (m + 1) n for every matrix and part product): 147 us = 660 TFLOP/s, whole tiles 830;
// four waves per tile (64 KB of fragments, half the waves) took 5 % of the optimiser step more.
__global__ __launch_bounds__(OrthoGram::THREADS, 4) void ortho_gram_kernel(OrthoTable tab, int turn, int ntiles) {
    typedef OrthoGram S;
    __shared__ __attribute__((aligned(128))) char smem[S::LDS];
    static_assert(64 * (S::TB + 5) * 4 <= S::LDS, "epilogue slab must fit the operand stages");
    const int at = nt_xcd_runs(blockIdx.x, ntiles);
    const OrthoTile w = tab.gram[at];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws, turn);
    const int m = ortho_m(p), n = ortho_n(p);
    const int i0 = (w.ij >> 16) * GRAM_TILE, j0 = (w.ij & 0xffff) * GRAM_TILE;
    const int64_t rb = ortho_row_bytes(n);
    const int groups = (n + 31) / 32;
    const int g0 = (int)((int64_t)groups * w.cut / p.nsplit), g1 = (int)((int64_t)groups * (w.cut + 1) / p.nsplit);
    f32x16 acc[S::FA][S::FB];
    nt_tile<S, f16x8, NT_SPLIT2, false>(o.x + i0 * rb, rb, m - i0, 0, o.x + j0 * rb, rb, m - j0, g0, g1, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (p.nsplit > 1) {
        float *slab = tab.slab + (int64_t)at * GRAM_TILE * GRAM_TILE;
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int j = 0; j < S::FB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    slab[(64 * (wave / S::WC) + 32 * i + nt_acc_row(r, lane)) * GRAM_TILE + 32 * (wave % S::WC) + 32 * j +
                         (lane & 31)] = acc[i][j][r];
        return;
    }
    for (int h = 0; h < 2; ++h) {
        if (i0 + 64 * h >= m) break;
        __syncthreads();
        ortho_slab_from_acc<S>((float *)smem, acc, h, ORTHO_UNSCALE * ORTHO_UNSCALE);
        __syncthreads();
        ortho_store_sym<64, GRAM_TILE, S::THREADS>((const float *)smem, i0 + 64 * h, j0, m, o.a, i0 != j0);
    }
}

// The cuts of a Gram tile, added in order.  Block = 32 rows of one tile.
__global__ __launch_bounds__(256) void ortho_join_kernel(OrthoTable tab) {
    __shared__ float slab[32 * (GRAM_TILE + 5)];
    const OrthoTile w = tab.sym[blockIdx.x >> 2];
    const int h = blockIdx.x & 3;
    const OrthoProb p = tab.prob[w.prob];
    const int m = ortho_m(p), tm = ortho_tiles(m, GRAM_TILE), nsym = tm * (tm + 1) / 2;
    const int i0 = (w.ij >> 16) * GRAM_TILE + 32 * h, j0 = (w.ij & 0xffff) * GRAM_TILE;
    if (p.nsplit == 1 || i0 >= m) return;
    const float4 *src = (const float4 *)(tab.slab + (int64_t)w.first * GRAM_TILE * GRAM_TILE + 32 * h * GRAM_TILE);
    const int64_t next = (int64_t)nsym * (GRAM_TILE * GRAM_TILE / 4);
#pragma unroll
    for (int e4 = 0; e4 < 4; ++e4) {
        const int e = e4 * 256 + threadIdx.x;
        float4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = 0; k < p.nsplit; ++k) {
            const float4 v = src[k * next + e];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        float *d = slab + (e >> 5) * (GRAM_TILE + 5) + (e & 31) * 4;
        const float u = ORTHO_UNSCALE * ORTHO_UNSCALE;
        d[0] = s.x * u; d[1] = s.y * u; d[2] = s.z * u; d[3] = s.w * u;
    }
    __syncthreads();
    ortho_store_sym<32, GRAM_TILE, 256>(slab, i0, j0, m, ortho_operands(p, tab.ws, 0).a, (w.ij >> 16) != (w.ij & 0xffff));
}

// ------------------------------------------------------------------------------------------------ P = a I + b A + c A^2
// Short contractions (8 to 32 k-steps): many small tiles and three workgroups per CU hide their latency.  125 matrices of a
// detector (18 GFLOP of products) 46 us, 128 x 128 tiles of eight waves 51; 21 matrices 25 and 36.
//
// The kinds of a pair of steps (all symmetric, all from the tiles on and above the diagonal): B = P1 A, A <- P1 B (held
// times 4^h of the second step), P2 from the new A, and P2 P1, held as a quarter (its norm is up to 3.45^2).
enum OrthoKind { PAIR_P, PAIR_B, PAIR_A, PAIR_P2, PAIR_PP };
template <OrthoKind KIND>
__global__ __launch_bounds__(256, 3) void ortho_poly_kernel(OrthoTable tab, int ntiles, int step) {
    typedef OrthoPoly S;
    constexpr int TILE = S::TA, R = TILE / 2;
    __shared__ __attribute__((aligned(128))) char smem[S::LDS];
    static_assert(R * (TILE + 5) * 4 <= S::LDS, "epilogue slab must fit the operand stages");
    const OrthoTile w = tab.square[nt_xcd_runs(blockIdx.x, ntiles)];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws, 0);
    const int m = ortho_m(p);
    const int i0 = (w.ij >> 16) * TILE, j0 = (w.ij & 0xffff) * TILE;
    const int64_t rb = ortho_row_bytes(m);
    f32x16 acc[S::FA][S::FB];
    constexpr bool POLY = KIND == PAIR_P || KIND == PAIR_P2;
    const char *u = POLY ? o.a : KIND == PAIR_PP ? o.t : o.p;
    const char *v = POLY || KIND == PAIR_B ? o.a : KIND == PAIR_A ? o.t : o.p;
    char *out = KIND == PAIR_P ? o.p : KIND == PAIR_B || KIND == PAIR_P2 ? o.t : o.a;
    nt_tile<S, f16x8, NT_SPLIT2, false>(u + i0 * rb, rb, m - i0, 0, v + j0 * rb, rb, m - j0, 0, (m + 31) / 32, smem, acc);
    const int t = threadIdx.x;
    float *slab = (float *)smem;
    const float down = ortho_shift(p.shift, step, -1), down2 = down * down;
    const int fewer = max(0, p.shift - 2 * step) - max(0, p.shift - 2 * (step + 1));        // of h, in the next step
    const float scale = POLY ? ORTHO_C * (down2 * down2) : KIND == PAIR_A ? ldexpf(1.f, -2 * fewer)
                                                         : KIND == PAIR_PP ? 0.25f : 1.f;
    for (int h = 0; h < 2; ++h) {
        const int r0 = i0 + R * h;
        if (r0 >= m) break;
        __syncthreads();
        ortho_slab_from_acc<S>(slab, acc, h, scale * (ORTHO_UNSCALE * ORTHO_UNSCALE));
        __syncthreads();
        for (int e = t; POLY && e < R * (TILE / 8); e += 256) {     // + b A + a I, in place
            const int r = e / (TILE / 8), c8 = e % (TILE / 8) * 8, k = j0 + c8;
            if (r0 + r >= m || k >= m) continue;
            const char *at = ortho_at(o.a, rb, r0 + r, k);
            const f16x8 h0 = *(const f16x8 *)at, h1 = *(const f16x8 *)(at + 64);
            float *d = slab + r * (TILE + 5) + c8;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float av = ((float)h0[q] + (float)h1[q]) * (ORTHO_UNSCALE * down2);
                d[q] += ORTHO_B * av + (r0 + r == k + q ? ORTHO_A : 0.f);
            }
        }
        __syncthreads();
        ortho_store_sym<R, TILE, 256>(slab, r0, j0, m, out, i0 != j0);
    }
}

// ------------------------------------------------------------------------------------------------ square products
// A = X X^T and P (POLY) of calls with little to do: every tile of the square, both triangles.  A lane's eight neighbours
// down a column are eight neighbours along the row of the transpose, and the product is symmetric: parts go from registers
// to that row.  Twice the products of the triangle, but no cuts, no turn through LDS and no second store (where there is
// enough work the triangles win: P of the heads' 21 matrices 24 us against 31, of all 125 46 against 69).
template <bool POLY>
__global__ __launch_bounds__(256, 2) void ortho_square_kernel(OrthoTable tab, int ntiles, int step) {
    typedef OrthoSquare S;
    __shared__ __attribute__((aligned(128))) char smem[S::LDS];
    const OrthoTile w = tab.square[nt_xcd_runs(blockIdx.x, ntiles)];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws, step);
    const int m = ortho_m(p), k = POLY ? m : ortho_n(p);
    const int i0 = (w.ij >> 16) * S::TA, j0 = (w.ij & 0xffff) * S::TB;
    const int64_t rb = ortho_row_bytes(k), rm = ortho_row_bytes(m);
    const char *y = POLY ? o.a : o.x;
    f32x16 acc[S::FA][S::FB];
    nt_tile<S, f16x8, NT_SPLIT2, false>(y + i0 * rb, rb, m - i0, 0, y + j0 * rb, rb, m - j0, 0, (k + 31) / 32, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c0 = i0 + S::TA / S::WR * (wave / S::WC), r0 = j0 + S::TB / S::WC * (wave % S::WC) + (lane & 31);
    const float down = POLY ? ortho_shift(p.shift, step, -1) : 1.f, down2 = down * down;
    const float un2 = ORTHO_UNSCALE * ORTHO_UNSCALE, fc = POLY ? ORTHO_C * (down2 * down2) * un2 : un2;
    const float fb = ORTHO_B * down2 * ORTHO_UNSCALE;
    char *dst = POLY ? o.p : o.a;
    const int mpad = (m + 31) & ~31;
#pragma unroll
    for (int j = 0; j < S::FB; ++j)
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                nt_acc_rows8(acc[i][j], h, v);
                const int row = r0 + 32 * j, c = c0 + 32 * i + 16 * h + 8 * (lane >> 5);
                if (row >= m || c >= mpad) continue;
                if (POLY) {
                    const char *at = ortho_at(o.a, rm, row, c);
                    const f16x8 h0 = *(const f16x8 *)at, h1 = *(const f16x8 *)(at + 64);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        v[q] = fc * v[q] + fb * ((float)h0[q] + (float)h1[q]) + (row == c + q ? ORTHO_A : 0.f);
                } else {
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] *= fc;
                }
#pragma unroll
                for (int q = 0; q < 8; ++q)
                    if (c + q >= m) v[q] = 0.f;    // (copies of the last row: what pads the contraction is zero)
                ortho_store8(ortho_at(dst, rm, row, c), v);
            }
}

// ------------------------------------------------------------------------------------------------ X <- P X
// One 32 (n, from k0) x 32 (m, from r0) block of (P X)^T held by a wave.  Wide matrices: a lane's element (h, q) is column
// k0 + 16 h + 8 (lane >> 5) + q of row r0 + (lane & 31); tall ones: element r is row k0 + nt_acc_row(r), column r0 + (lane
// & 31), lanes side by side.  ortho_old: the weights of a block, fetched ahead of the stores of the one before.
__device__ __forceinline__ void ortho_old(const OrthoProb &p, int k0, int r0, int m, int n, float *old) {
    const int lane = threadIdx.x & 63, row = r0 + (lane & 31);
    const float *w = (const float *)p.out;
    if (p.rows > p.cols) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int k = k0 + nt_acc_row(r, lane);
            old[r] = row < m && k < n ? w[(int64_t)k * p.os + row] : 0.f;
        }
        return;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = k0 + 16 * h + 8 * (lane >> 5);
        const float *d = w + (int64_t)row * p.os + k;
        if (row < m && k + 8 <= n && !((uintptr_t)d & 15)) {
            *(float4 *)(old + 8 * h) = *(const float4 *)d;
            *(float4 *)(old + 8 * h + 4) = *(const float4 *)(d + 4);
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) old[8 * h + q] = row < m && k + q < n ? d[q] : 0.f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void ortho_result(const OrthoProb &p, const f32x16 &acc, int k0, int r0, int m, int n,
                                             float unscale, const float *old) {
    const int lane = threadIdx.x & 63, row = r0 + (lane & 31);
    if (row >= m) return;
    if (p.rows > p.cols) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int k = k0 + nt_acc_row(r, lane);
            if (k >= n) continue;
            const int64_t at = (int64_t)k * p.os + row;
            const float v = acc[r] * unscale;
            if (p.buf) ((float *)p.out)[at] = old[r] * p.decay - p.lr * v;
            else ((T *)p.out)[at] = (T)v;
        }
        return;
    }
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[8];
        nt_acc_rows8(acc, h, v);
        const int k = k0 + 16 * h + 8 * (lane >> 5);
        const int64_t at = (int64_t)row * p.os + k;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            v[q] *= unscale;
            if (p.buf) v[q] = old[8 * h + q] * p.decay - p.lr * v[q];
        }
        T *d = (T *)p.out + at;                    // (the optimiser: T is float)
        if (k + 8 <= n && !((uintptr_t)d & (4 * sizeof(T) - 1))) {
            t4 a, b;
#pragma unroll
            for (int q = 0; q < 4; ++q) { a[q] = (T)v[q]; b[q] = (T)v[4 + q]; }
            *(t4 *)d = a;
            *(t4 *)(d + 4) = b;
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q)
                if (k + q < n) d[q] = (T)v[q];
        }
    }
}

struct OrthoTurn { int turn, step, pair; };         // passes over X before this one; the (first) step it makes; of two
// LAST: the result instead of the next step's X.  Bound as the Gram products are, and by its stores: 125 matrices of a
// detector (193 GFLOP of products) 227 us = 850 TFLOP/s with 256 x 256 tiles, the library's fp16 product 1390.
template <typename T, typename S, bool LAST>
__global__ __launch_bounds__(S::THREADS, S::TA == 128 ? 4 : 2) void ortho_apply_kernel(OrthoTable tab,
                                                                                         const OrthoTile *list, int ntiles,
                                                                                         OrthoTurn turn, OrthoRule rule) {
    __shared__ __attribute__((aligned(128))) char smem[S::LDS];
    const OrthoTile w = list[nt_xcd_runs(blockIdx.x, ntiles)];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws, turn.turn);
    const int m = ortho_m(p), n = ortho_n(p);
    const int i0 = (w.ij >> 16) * S::TB, j0 = (w.ij & 0xffff) * S::TA;
    const int64_t rx = ortho_row_bytes(n), rp = ortho_row_bytes(m);
    const int groups = (n + 31) / 32;
    f32x16 acc[S::FA][S::FB];
    nt_tile<S, f16x8, NT_SPLIT2, true>(o.x + (j0 / 32) * 128, rx, groups - j0 / 32, m, (turn.pair ? o.a : o.p) + i0 * rp, rp, m - i0, 0,
                                       (m + 31) / 32, smem, acc);
    if (LAST && p.buf) {
        const double sq = rule.sqnorm[0];
        if (!(sq >= 0.0 && sq < INFINITY)) return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int k0 = j0 + S::TA / S::WR * (wave / S::WC), r0 = i0 + S::TB / S::WC * (wave % S::WC);
    const float unscale = ORTHO_UNSCALE * ORTHO_UNSCALE * (turn.pair ? 4.f : 1.f) * ortho_shift(p.shift, turn.step, -1) *
                          (LAST ? 1.f : ortho_shift(p.shift, turn.step + 1 + turn.pair, 1));
    if (LAST) {
        float old[2][16];
        if (p.buf) ortho_old(p, k0, r0, m, n, old[0]);
#pragma unroll
        for (int b = 0; b < S::FA * S::FB; ++b) {
            const int i = b % S::FA, j = b / S::FA, i2 = (b + 1) % S::FA, j2 = (b + 1) / S::FA;
            if (p.buf && b + 1 < S::FA * S::FB) ortho_old(p, k0 + 32 * i2, r0 + 32 * j2, m, n, old[(b + 1) & 1]);
            ortho_result<T>(p, acc[i][j], k0 + 32 * i, r0 + 32 * j, m, n, unscale, old[b & 1]);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < S::FB; ++j)
#pragma unroll
        for (int i = 0; i < S::FA; ++i) {
            const int row = r0 + 32 * j + (lane & 31);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                nt_acc_rows8(acc[i][j], h, v);
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] *= unscale;
                const int k = k0 + 32 * i + 16 * h + 8 * (lane >> 5);
                if (row < m && k < groups * 32) ortho_store8(ortho_at(o.next, rx, row, k), v);
            }
        }
}

// ------------------------------------------------------------------------------------------------ one launch
// A matrix whose shorter side is at most 32 (MB = 1) or 64 (MB = 2) and whose parts of X fit 144 KB of LDS, by one
// workgroup of eight waves.  X rows of G groups of 128 B; S: 16 KB for the joined sums of the Gram matrix, then A, then P
// (rows of MB groups).  16-byte chunks are XORed with bits of the row (f) so that both ways of reading -- sixteen rows of
// one chunk, four rows of four chunks -- meet at most two lanes on a bank.
//   Gram: wave (block, part of the contraction); the parts meet in S; the block's sums stay in registers for b A.
//   Apply: a wave takes a group of 32 columns, reads all of its X, and writes P X in its place.
// Latency-bound: 64 x 576 takes 54 us, 13 to read, norm and lay out, 8.3 a step (clock counts: the Gram products 2.4 us,
// what is between them and P X 3, P X 3: three rounds of groups, 24 matrix instructions and 220 others each).
#define SMALL_X 147456
#define SMALL_S 16384
__host__ __device__ static inline bool ortho_small(int m, int n) {
    return m <= 64 && (int64_t)(m <= 32 ? 32 : 64) * ortho_row_bytes(n) <= SMALL_X;
}
__device__ __forceinline__ int small_swizzle(int row, int c) { return c ^ (((row & 1) << 2) | ((row >> 1) & 3)); }
// byte of chunk c (0 ... 7; part 1 from 4 on) of group g of row `row`
__device__ __forceinline__ int small_at(int row, int pitch, int g, int c) {
    return row * pitch + g * 128 + small_swizzle(row, c) * 16;
}
__device__ __forceinline__ void small_products(const f16x8 *a, const f16x8 *b, f32x16 &acc, f32x16 &cor) {
    cor = nt_mfma<f16x8>(a[1], b[0], cor);
    acc = nt_mfma<f16x8>(a[0], b[0], acc);
    cor = nt_mfma<f16x8>(a[0], b[1], cor);
}

template <typename T, int MB>
__global__ __launch_bounds__(512) void ortho_small_kernel(OrthoBatch batch, OrthoRule rule, int steps, float eps) {
    __shared__ __attribute__((aligned(128))) char smem[SMALL_X + SMALL_S];
    constexpr int MP = 32 * MB, CUTS = MB == 2 ? 2 : 4, SP = MB * 128;      // contraction cuts, pitch of S
    char *lx = smem, *ls = smem + SMALL_X;
    const OrthoProb p = batch.p[blockIdx.x];
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int m = ortho_m(p), n = ortho_n(p), groups = (n + 31) / 32, pitch = groups * 128;
    const bool tall = p.rows > p.cols;
    float cf = 1.f;
    bool apply = true;
    if (p.buf) apply = ortho_clip(rule, cf);
    // ---- u (and the momentum) and its norm: a thread holds up to nine runs of eight neighbours along n
    constexpr int RUNS = SMALL_X / 4 / 8 / 512;
    float u[RUNS][8];
    // f(s, row, run of eight): runs t + 512 s, lanes along G's rows; stepped, not divided
    const int width = tall ? MP : groups * 4, dq = 512 / width, dr = 512 - dq * width, b0 = t / width, a0 = t - b0 * width;
    auto each = [&](auto f) {
        int a = a0, b = b0;
#pragma unroll
        for (int s = 0; s < RUNS; ++s) {
            f(s, tall ? a : b, tall ? b : a);
            a += dr; b += dq;
            if (a >= width) { a -= width; ++b; }
        }
    };
    const bool vec = !tall && sizeof(T) == 4 && (n & 3) == 0 && (p.gs & 3) == 0 &&
                     !(((uintptr_t)p.g | (uintptr_t)p.buf) & 15);
    // eight neighbours along n, side by side or ld apart (tall); zeros outside.  (One branch around all the loads: none
    // waits for another.)
    auto fetch = [&](auto *base, int64_t ld, float (&v)[RUNS][8]) {
        if (vec)
            each([&](int s, int i, int k8) {
                const float *at = (const float *)base + (int64_t)i * ld + k8 * 8;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float4 x = {0.f, 0.f, 0.f, 0.f};
                    if (i < m && k8 * 8 + 4 * h < n) x = *(const float4 *)(at + 4 * h);
                    *(float4 *)(v[s] + 4 * h) = x;
                }
            });
        else
            each([&](int s, int i, int k8) {
                const auto *at = base + (tall ? (int64_t)k8 * 8 * ld + i : (int64_t)i * ld + k8 * 8);
                const int64_t next = tall ? ld : 1;
#pragma unroll
                for (int q = 0; q < 8; ++q) v[s][q] = i < m && k8 * 8 + q < n ? (float)at[q * next] : 0.f;
            });
    };
    fetch((const T *)p.g, p.gs, u);
    if (p.buf) {
        float b[RUNS][8];
        fetch((const float *)p.buf, p.cols, b);
        each([&](int s, int i, int k8) {
            float *d = p.buf + (tall ? (int64_t)k8 * 8 * p.cols + i : (int64_t)i * p.cols + k8 * 8);
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                u[s][q] = ortho_momentum(rule, u[s][q], cf, b[s][q]);
                if (apply && i < m && k8 * 8 + q < n) d[tall ? (int64_t)q * p.cols : q] = b[s][q];
            }
        });
    }
    double sum = 0.0;
#pragma unroll
    for (int s = 0; s < RUNS; ++s)
#pragma unroll
        for (int q = 0; q < 8; ++q) sum += (double)u[s][q] * u[s][q];
    int shift;
    float up;
    const float inv = ortho_inverse(ortho_block_sum(sum, (double *)ls), eps, shift, up);
    // ---- X
    each([&](int s, int i, int k8) {
        if (t + 512 * s >= MP * groups * 4) return;
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = u[s][q] * up * inv;
        f16x8 h0, h1;
        ortho_parts8(v, h0, h1);
        *(f16x8 *)(lx + small_at(i, pitch, k8 >> 2, k8 & 3)) = h0;
        *(f16x8 *)(lx + small_at(i, pitch, k8 >> 2, 4 + (k8 & 3))) = h1;
    });
    __syncthreads();
    const int blk = wave % (MB * MB), cut = wave / (MB * MB), bi = blk / MB, bj = blk % MB;
    const float un2 = ORTHO_UNSCALE * ORTHO_UNSCALE;
    for (int step = 0; step < steps; ++step) {
        // (opaque: addresses that follow from the lane are made where they are used; kept over all the phases they spill)
        int lane = t & 63;
        asm volatile("" : "+v"(lane));
        const int frow = lane & 31, fhalf = lane >> 5;
        // ---- A = X X^T: block (bi, bj), groups of this cut
        f32x16 ga, gb;                             // a0 b0; the corrections
#pragma unroll
        for (int r = 0; r < 16; ++r) ga[r] = gb[r] = 0.f;
        if (cut < CUTS) {
            auto take = [&](int g, f16x8 (&fa)[2][2], f16x8 (&fb)[2][2]) {
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        fa[kk][q] = *(const f16x8 *)(lx + small_at(32 * bi + frow, pitch, g, 4 * q + 2 * kk + fhalf));
                        fb[kk][q] = *(const f16x8 *)(lx + small_at(32 * bj + frow, pitch, g, 4 * q + 2 * kk + fhalf));
                    }
            };
            auto multiply = [&](const f16x8 (&fa)[2][2], const f16x8 (&fb)[2][2]) {
                small_products(fa[0], fb[0], ga, gb);
                small_products(fa[1], fb[1], ga, gb);
            };
            int g = groups * cut / CUTS;
            const int end = groups * (cut + 1) / CUTS;
            f16x8 fa[2][2][2], fb[2][2][2];
            if (g < end) take(g, fa[0], fb[0]);
            for (; g + 2 < end; g += 2) {          // the next group's reads behind this one's products
                take(g + 1, fa[1], fb[1]);
                multiply(fa[0], fb[0]);
                take(g + 2, fa[0], fb[0]);
                multiply(fa[1], fb[1]);
            }
            if (g + 1 < end) take(g + 1, fa[1], fb[1]);
            if (g < end) multiply(fa[0], fb[0]);
            if (g + 1 < end) multiply(fa[1], fb[1]);
#pragma unroll
            for (int r = 0; r < 16; ++r) ga[r] += gb[r];
            if (cut > 0) {
                float *d = (float *)ls + ((cut - 1) * MB * MB + blk) * 1024 + lane;
#pragma unroll
                for (int r = 0; r < 16; ++r) d[r * 64] = ga[r];
            }
        }
        __syncthreads();
        if (cut == 0) {
#pragma unroll
            for (int c = 1; c < CUTS; ++c) {
                const float *s = (const float *)ls + ((c - 1) * MB * MB + blk) * 1024 + lane;
#pragma unroll
                for (int r = 0; r < 16; ++r) ga[r] += s[r * 64];
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) ga[r] *= un2;      // A 4^h
        }
        __syncthreads();
        // a block is symmetric to its mirror image: eight neighbours of column lane & 31 are eight neighbours of that row
        auto store_block = [&](const f32x16 &b) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v[8];
                nt_acc_rows8(b, h, v);
                f16x8 h0, h1;
                ortho_parts8(v, h0, h1);
                const int row = 32 * bj + frow, c = 2 * h + fhalf;
                *(f16x8 *)(ls + small_at(row, SP, bi, c)) = h0;
                *(f16x8 *)(ls + small_at(row, SP, bi, 4 + c)) = h1;
            }
        };
        if (cut == 0) store_block(ga);
        __syncthreads();
        // ---- P = a I + b A + c A^2
        const float down = ortho_shift(shift, step, -1), down2 = down * down;
        f32x16 pa;
        if (cut == 0) {
#pragma unroll
            for (int r = 0; r < 16; ++r) pa[r] = gb[r] = 0.f;
#pragma unroll
            for (int g = 0; g < MB; ++g)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    f16x8 fa[2], fb[2];
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        fa[q] = *(const f16x8 *)(ls + small_at(32 * bi + frow, SP, g, 4 * q + 2 * kk + fhalf));
                        fb[q] = *(const f16x8 *)(ls + small_at(32 * bj + frow, SP, g, 4 * q + 2 * kk + fhalf));
                    }
                    small_products(fa, fb, pa, gb);
                }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                pa[r] = ORTHO_C * (down2 * down2) * un2 * (pa[r] + gb[r]) + ORTHO_B * down2 * ga[r] +
                        (32 * bi + nt_acc_row(r, lane) == 32 * bj + frow ? ORTHO_A : 0.f);
        }
        __syncthreads();
        if (cut == 0) store_block(pa);
        __syncthreads();
        // ---- X <- P X, as (P X)^T: rows n of group g, columns m
        const bool last = step + 1 == steps;
        const float unscale = un2 * down * (last ? 1.f : ortho_shift(shift, step + 1, 1));
        f16x8 fp[MB][MB][2][2];                    // P's rows: [block of m][k group][kk][part]
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int kg = 0; kg < MB; ++kg)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int q = 0; q < 2; ++q)
                        fp[b][kg][kk][q] = *(const f16x8 *)(ls + small_at(32 * b + frow, SP, kg, 4 * q + 2 * kk + fhalf));
        for (int g = wave; g < groups; g += 8) {
            f16x8 fx[MB][2][2];                    // [k group][kk][part]
#pragma unroll
            for (int kg = 0; kg < MB; ++kg)
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        union { s16x4 h[2]; f16x8 v; } u;
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int k = 32 * kg + 16 * kk + 8 * fhalf + 4 * e + ((lane >> 2) & 3);
                            const char *at2 = lx + small_at(k, pitch, g, 4 * q + 2 * (frow >> 4) + ((lane & 3) >> 1)) +
                                              (lane & 1) * 8;
                            u.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at2);
                        }
                        fx[kg][kk][q] = u.v;
                    }
            f32x16 y[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) y[b][r] = 0.f;
#pragma unroll
                for (int kg = 0; kg < MB; ++kg)
#pragma unroll
                    for (int kk = 0; kk < 2; ++kk) small_products(fx[kg][kk], fp[b][kg][kk], y[b], y[b]);
            }
            if (last) {
                if (apply)
#pragma unroll
                    for (int b = 0; b < MB; ++b) {
                        float old[16];
                        if (p.buf) ortho_old(p, 32 * g, 32 * b, m, n, old);
                        ortho_result<T>(p, y[b], 32 * g, 32 * b, m, n, unscale, old);
                    }
                continue;
            }
#pragma unroll
            for (int b = 0; b < MB; ++b)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[8];
                    nt_acc_rows8(y[b], h, v);
#pragma unroll
                    for (int q = 0; q < 8; ++q) v[q] *= unscale;
                    f16x8 h0, h1;
                    ortho_parts8(v, h0, h1);
                    const int row = 32 * b + frow, c = 2 * h + fhalf;
                    *(f16x8 *)(lx + small_at(row, pitch, g, c)) = h0;
                    *(f16x8 *)(lx + small_at(row, pitch, g, 4 + c)) = h1;
                }
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ host side
// Everything about a call that follows from its shapes.
struct OrthoPlan {
    int64_t prob, split, sym, gram, square, apply, last, part, slab, operands, bytes;
    int nsplit, nsym, ngram, nsquare, napply, nlast, nparts, cut, apply_tile, empty;
    int64_t gram_at[17];             // first entry of each class of Gram items, the long ones first
    bool joined, small, squares;     // squares: short Gram products, not cut
    bool pairs;                      // two steps per pass over X
};

// Cuts of a matrix with k columns and their class (0: the longest sixteenth): the launch ends together if it begins with
// the long ones (125 matrices of a detector, c = 79: 147 us instead of 179 in the order of their rows).
static inline int64_t ortho_cuts(const OrthoPlan &pl, int64_t k) { return pl.squares ? 0 : ((k + 31) / 32 + pl.cut - 1) / pl.cut; }
static inline int ortho_gram_class(const OrthoPlan &pl, int64_t k) {
    const int64_t g = (k + 31) / 32, cuts = (g + pl.cut - 1) / pl.cut;
    return 15 - (int)(((g + cuts - 1) / cuts - 1) * 16 / pl.cut);
}

static inline int64_t ortho_align(int64_t v) { return (v + 255) & ~(int64_t)255; }

template <typename D>
static void ortho_sides(const D &d, int64_t &m, int64_t &n) {
    m = d.rows < d.cols ? d.rows : d.cols;
    n = d.rows < d.cols ? d.cols : d.rows;
}

// Cuts of the Gram contraction: the longest run of k-steps that one item gets.  A workgroup alone on its CU takes 0.65 us
// a k-step, one of two 1.13; an item costs about six steps more than it has, and a partial tile a sixteenth of a step to
// store and to join (all launches together).  In quarters of a step: items that each have a CU end after 4 (c + 6), two on
// a CU after 7 (c + 6); W k-steps in more items take about 7 (W + 6 items) / 512, the last ones ending half a cut apart.
// The c, in steps of an eighth, that makes this least.  Measured per step of the iteration, relative to a shorter cut: 23
// matrices of 256 x 2304, c = 24 (207 items) 9 us less than 12, 36 6 more, 72 24 more; 21 of 2 x 256 to 1024 x 12544, c =
// 40 (493 items) 11 us less than 24, 72 15 more; 125 of a whole detector, c = 100 (636) 16 us less than 32, 200 29 more.
template <typename D>
static int64_t ortho_gram_cut(const D *d, int n) {
    int64_t best = 8, least = INT64_MAX, steps = 0, longest = 0;
    for (int i = 0; i < n; ++i) {
        int64_t m, k;
        ortho_sides(d[i], m, k);
        const int64_t t = (m + GRAM_TILE - 1) / GRAM_TILE, g = (k + 31) / 32;
        steps += t * (t + 1) / 2 * g;
        if (g > longest) longest = g;
    }
    for (int64_t c = steps / 1024 > 8 ? steps / 1024 : 8;; c += c / 8 + 1) {
        int64_t items = 0;
        for (int i = 0; i < n; ++i) {
            int64_t m, k;
            ortho_sides(d[i], m, k);
            const int64_t t = (m + GRAM_TILE - 1) / GRAM_TILE;
            items += t * (t + 1) / 2 * (((k + 31) / 32 + c - 1) / c);
        }
        const int64_t most = c < longest ? c : longest;
        const int64_t cost = items / 4 + (items <= 256 ? 4 * (most + 6) : items <= 512 ? 7 * (most + 6)
                                                                                       : 7 * (steps + 6 * items) / 512 + 2 * most);
        if (cost < least) { least = cost; best = c; }
        if (items <= 256 || c >= longest) break;
    }
    return best;
}

// A pair of steps saves three times m^2 n and costs three times m^3, in short products that run at half the rate.  Five
// steps, 2 + 1 + 2, against single ones, measured in turn: 23 matrices of 256 x 2304 315 us and 372, 21 of the heads (m^2 n
// 6.6 times m^3, an optimiser step) 958 and 1133, 125 of a detector (5.2 times) 2096 and 2484.  Around the limit: 16 of 512 x
// 768 442 and 422, x 1024 452 and 449, x 1536 522 and 564; 4 of 1024 x 1536 611 and 604, x 2048 641 and 655.
static inline bool ortho_pairs(double wide, double cubes) { return wide > 2. * cubes; }

template <typename D>
static int ortho_plan(const D *d, int n, OrthoPlan &pl) {
    pl = OrthoPlan();
    pl.small = true;
    int64_t square64 = 0, apply256 = 0, live = 0, longest = 0;
    double wide = 0., cubes = 0.;                  // m^2 n and m^3 over the matrices
    for (int i = 0; i < n; ++i) {
        if (d[i].rows < 0 || d[i].cols < 0 || d[i].rows > (1 << 22) || d[i].cols > (1 << 22)) return SLN_ERR_INVALID_ARG;
        int64_t m, k;
        ortho_sides(d[i], m, k);
        if (m > 65535) return SLN_ERR_UNSUPPORTED;
        if (m == 0) continue;
        ++live;
        pl.small = pl.small && ortho_small((int)m, (int)k);
        square64 += ((m + 63) / 64) * ((m + 63) / 64);
        if ((k + 31) / 32 > longest) longest = (k + 31) / 32;
        wide += (double)m * m * k;
        cubes += (double)m * m * m;
        apply256 += ((m + 255) / 256) * ((k + 255) / 256);
    }
    pl.empty = live == 0;
    if (pl.empty || pl.small) return SLN_OK;
    pl.cut = (int)ortho_gram_cut(d, n);
    // Tiles: large ones where they fill the chip, else smaller ones.  Few and short Gram products (up to one tile of 64 x 64
    // per CU, up to 80 k-steps) go without cuts, partial tiles and the launch that joins them.
    // (the large ones where the rounds of 256 they make are three quarters full: alone on its CU a workgroup's stores are
    // not covered by another's loads; the optimiser's last step, which also reads the weights, takes the small ones)
    pl.apply_tile = 4 * apply256 >= 3 * ((apply256 + 255) / 256 * 256) ? 256 : 128;
    pl.squares = square64 <= 256 && longest <= 80;
    pl.pairs = !pl.squares && ortho_pairs(wide, cubes);
    int64_t nsplit = 0, nsym = 0, ngram = 0, nsquare = 0, napply = 0, nlast = 0, nparts = 0, operands = 0;
    for (int i = 0; i < n; ++i) {
        if (d[i].rows == 0 || d[i].cols == 0) continue;
        OrthoProb p = {};
        p.rows = d[i].rows; p.cols = d[i].cols;
        const int64_t m = ortho_m(p), k = ortho_n(p);
        const int64_t tm = (m + GRAM_TILE - 1) / GRAM_TILE, cuts = ortho_cuts(pl, k);
        const int64_t tp = (m + OrthoSquare::TA - 1) / OrthoSquare::TA;
        pl.joined |= cuts > 1;
        nsplit += ((m + 63) / 64) * ((k + 127) / 128);
        if (!pl.squares) {
            nsym += tm * (tm + 1) / 2;
            ngram += tm * (tm + 1) / 2 * cuts;
            pl.gram_at[ortho_gram_class(pl, k) + 1] += tm * (tm + 1) / 2 * cuts;
        }
        nsquare += pl.squares ? tp * tp : tp * (tp + 1) / 2;
        napply += ((m + pl.apply_tile - 1) / pl.apply_tile) * ((k + pl.apply_tile - 1) / pl.apply_tile);
        nlast += ((m + 127) / 128) * ((k + 127) / 128);
        nparts += ((int64_t)p.rows * p.cols + ORTHO_CHUNK - 1) / ORTHO_CHUNK;
        operands += ortho_align(ortho_operand_bytes(p, pl.pairs));
        const int64_t most = 1 << 28;
        if (nsplit > most || ngram > most || nsquare > most || nlast > most || nparts > most) return SLN_ERR_UNSUPPORTED;
    }
    for (int i = 1; i < 17; ++i) pl.gram_at[i] += pl.gram_at[i - 1];
    int64_t at = 0;
    pl.prob = at; at += ortho_align(live * (int64_t)sizeof(OrthoProb));
    pl.split = at; at += ortho_align(nsplit * (int64_t)sizeof(OrthoTile));
    pl.sym = at; at += ortho_align(nsym * (int64_t)sizeof(OrthoTile));
    pl.gram = at; at += ortho_align(ngram * (int64_t)sizeof(OrthoTile));
    pl.square = at; at += ortho_align(nsquare * (int64_t)sizeof(OrthoTile));
    pl.apply = at; at += ortho_align(napply * (int64_t)sizeof(OrthoTile));
    pl.last = at; at += ortho_align(nlast * (int64_t)sizeof(OrthoTile));
    pl.part = at; at += ortho_align(nparts * (int64_t)sizeof(double));
    pl.slab = at; at += pl.joined ? ortho_align(ngram * (int64_t)(GRAM_TILE * GRAM_TILE * 4)) : 0;
    pl.operands = at; at += operands;
    pl.bytes = at;
    pl.nsplit = (int)nsplit; pl.nsym = (int)nsym; pl.ngram = (int)ngram; pl.nsquare = (int)nsquare; pl.napply = (int)napply;
    pl.nlast = (int)nlast;
    pl.nparts = (int)nparts;
    return SLN_OK;
}

static void ortho_desc(const sln_ortho_desc_t &d, OrthoProb &p) {
    p = OrthoProb();
    p.g = d.g; p.out = d.out;
    p.gs = d.g_stride; p.os = d.out_stride;
    p.rows = d.rows; p.cols = d.cols;
    p.decay = 1.f;
}
static void ortho_desc(const sln_muon_desc_t &d, OrthoProb &p) {
    p = OrthoProb();
    p.g = d.grad; p.out = d.param; p.buf = d.momentum;
    p.gs = p.os = d.cols;
    p.rows = d.rows; p.cols = d.cols;
    p.lr = d.lr; p.decay = d.decay;
}

template <typename T, typename D, int MB>
static void ortho_run_small(const D *d, int n, int steps, float eps, const OrthoRule &rule, hipStream_t stream) {
    OrthoBatch batch;
    int inb = 0;
    for (int i = 0; i < n; ++i) {
        int64_t m, k;
        ortho_sides(d[i], m, k);
        if (m > 0 && (m <= 32) == (MB == 1)) ortho_desc(d[i], batch.p[inb++]);
        if (inb == ORTHO_BATCH || (inb > 0 && i + 1 == n)) {
            hipLaunchKernelGGL((ortho_small_kernel<T, MB>), dim3(inb), dim3(512), 0, stream, batch, rule, steps, eps);
            inb = 0;
        }
    }
}

template <typename T, typename S>
static void ortho_apply(const OrthoTable &tab, const OrthoTile *list, int n, OrthoTurn turn, bool last, const OrthoRule &rule,
                        hipStream_t stream) {
    if (last)
        hipLaunchKernelGGL((ortho_apply_kernel<T, S, true>), dim3(n), dim3(S::THREADS), 0, stream, tab, list, n, turn, rule);
    else
        hipLaunchKernelGGL((ortho_apply_kernel<T, S, false>), dim3(n), dim3(S::THREADS), 0, stream, tab, list, n, turn, rule);
}

template <typename T, typename D>
static int ortho_run(const D *d, int n, int steps, float eps, const OrthoRule &rule, void *workspace, size_t ws_bytes,
                     hipStream_t stream) {
    OrthoPlan pl;
    const int rc = ortho_plan(d, n, pl);
    if (rc != SLN_OK) return rc;
    if (pl.empty) return SLN_OK;
    if (pl.bytes && (!workspace || ((uintptr_t)workspace & 255))) return SLN_ERR_INVALID_ARG;
    if (ws_bytes < (size_t)pl.bytes) return SLN_ERR_WORKSPACE;
    sln_enter();
    if (pl.small) {
        ortho_run_small<T, D, 1>(d, n, steps, eps, rule, stream);
        ortho_run_small<T, D, 2>(d, n, steps, eps, rule, stream);
        return sln_launch_status();
    }
    char *ws = (char *)workspace;
    const OrthoTable tab = {(OrthoProb *)(ws + pl.prob), (OrthoTile *)(ws + pl.split), (OrthoTile *)(ws + pl.sym),
                            (OrthoTile *)(ws + pl.gram), (OrthoTile *)(ws + pl.square), (OrthoTile *)(ws + pl.apply),
                            (OrthoTile *)(ws + pl.last), (double *)(ws + pl.part), ws, (float *)(ws + pl.slab), pl.apply_tile};
    OrthoBatch batch;
    int prob0 = 0, inb = 0, parts = 1, part0 = 0, split0 = 0, sym0 = 0, square0 = 0, apply0 = 0, last0 = 0;
    int64_t off = pl.operands;
    for (int i = 0; i <= n; ++i) {
        if (inb == ORTHO_BATCH || (inb > 0 && i == n)) {
            hipLaunchKernelGGL((ortho_norm_kernel<T>), dim3(parts, inb), dim3(256), 0, stream, batch, prob0, tab, rule);
            prob0 += inb; inb = 0; parts = 1;
        }
        if (i == n || d[i].rows == 0 || d[i].cols == 0) continue;
        OrthoProb &p = batch.p[inb++];
        ortho_desc(d[i], p);
        const int m = ortho_m(p), k = ortho_n(p);
        const int tm = ortho_tiles(m, GRAM_TILE), tp = ortho_tiles(m, OrthoSquare::TA);
        p.off = off; off += ortho_align(ortho_operand_bytes(p, pl.pairs));
        p.nsplit = (int)ortho_cuts(pl, k);
        p.part0 = part0; p.nparts = sln_div_up((long)p.rows * p.cols, ORTHO_CHUNK); part0 += p.nparts;
        p.split0 = split0; split0 += ortho_tiles(m, 64) * ortho_tiles(k, 128);
        p.sym0 = sym0; sym0 += pl.squares ? 0 : tm * (tm + 1) / 2;
        if (!pl.squares) {
            int64_t &g0 = pl.gram_at[ortho_gram_class(pl, k)];
            p.gram0 = (int)g0; g0 += tm * (tm + 1) / 2 * p.nsplit;
        }
        p.square0 = square0; square0 += pl.squares ? tp * tp : tp * (tp + 1) / 2;
        p.apply0 = apply0; apply0 += ortho_tiles(m, pl.apply_tile) * ortho_tiles(k, pl.apply_tile);
        p.last0 = last0; last0 += ortho_tiles(m, 128) * ortho_tiles(k, 128);
        if (p.nparts > parts) parts = p.nparts;
    }
    hipLaunchKernelGGL((ortho_split_kernel<T>), dim3(pl.nsplit), dim3(256), 0, stream, tab, rule, eps);
    OrthoTurn turn = {0, 0, 0};
    for (; turn.step < steps; turn.step += 1 + turn.pair, ++turn.turn) {
        const int s = turn.step;
        turn.pair = pl.pairs && s % 3 == 0 && s + 1 < steps;
        if (pl.squares) {
            hipLaunchKernelGGL((ortho_square_kernel<false>), dim3(pl.nsquare), dim3(256), 0, stream, tab, pl.nsquare, s);
            hipLaunchKernelGGL((ortho_square_kernel<true>), dim3(pl.nsquare), dim3(256), 0, stream, tab, pl.nsquare, s);
        } else {
            const dim3 tri(pl.nsquare), block(256);
            hipLaunchKernelGGL(ortho_gram_kernel, dim3(pl.ngram), dim3(OrthoGram::THREADS), 0, stream, tab, turn.turn, pl.ngram);
            if (pl.joined) hipLaunchKernelGGL(ortho_join_kernel, dim3(4 * pl.nsym), block, 0, stream, tab);
            hipLaunchKernelGGL((ortho_poly_kernel<PAIR_P>), tri, block, 0, stream, tab, pl.nsquare, s);
            if (turn.pair) {
                hipLaunchKernelGGL((ortho_poly_kernel<PAIR_B>), tri, block, 0, stream, tab, pl.nsquare, s);
                hipLaunchKernelGGL((ortho_poly_kernel<PAIR_A>), tri, block, 0, stream, tab, pl.nsquare, s);
                hipLaunchKernelGGL((ortho_poly_kernel<PAIR_P2>), tri, block, 0, stream, tab, pl.nsquare, s + 1);
                hipLaunchKernelGGL((ortho_poly_kernel<PAIR_PP>), tri, block, 0, stream, tab, pl.nsquare, s);
            }
        }
        const bool last = s + 1 + turn.pair == steps, weights = last && rule.sqnorm;
        if (pl.apply_tile == 256 && !weights) ortho_apply<T, OrthoApplyLarge>(tab, tab.apply, pl.napply, turn, last, rule, stream);
        else if (weights) ortho_apply<T, OrthoApplySmall>(tab, tab.last, pl.nlast, turn, last, rule, stream);
        else ortho_apply<T, OrthoApplySmall>(tab, tab.apply, pl.napply, turn, last, rule, stream);
    }
    return sln_launch_status();
}

extern "C" size_t sln_orthogonalize_workspace_bytes(const sln_ortho_desc_t *descs, int n) {
    OrthoPlan pl;
    if (n < 0 || (n > 0 && !descs) || ortho_plan(descs, n, pl) != SLN_OK) return 0;
    return (size_t)pl.bytes;
}

extern "C" int sln_orthogonalize(const sln_ortho_desc_t *descs, int n, int dtype, int steps, float eps, void *workspace,
                                 size_t workspace_bytes, sln_stream_t stream) {
    if (n < 0 || (n > 0 && !descs) || steps < 1 || steps > 64 || !(eps >= 1e-30f)) return SLN_ERR_INVALID_ARG;
    for (int i = 0; i < n; ++i) {
        const sln_ortho_desc_t &d = descs[i];
        if (d.rows == 0 || d.cols == 0) continue;
        if (!d.g || !d.out || d.g_stride < d.cols || d.out_stride < d.cols) return SLN_ERR_INVALID_ARG;
    }
    const OrthoRule rule = {nullptr, 0.f, 0.f, 0};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case SLN_DTYPE_F32: return ortho_run<float>(descs, n, steps, eps, rule, workspace, workspace_bytes, s);
        case SLN_DTYPE_BF16: return ortho_run<__bf16>(descs, n, steps, eps, rule, workspace, workspace_bytes, s);
        case SLN_DTYPE_F16: return ortho_run<_Float16>(descs, n, steps, eps, rule, workspace, workspace_bytes, s);
        default: return SLN_ERR_INVALID_ARG;
    }
}

extern "C" size_t sln_muon_step_workspace_bytes(const sln_muon_desc_t *descs, int n) {
    OrthoPlan pl;
    if (n < 0 || (n > 0 && !descs) || ortho_plan(descs, n, pl) != SLN_OK) return 0;
    return (size_t)pl.bytes;
}

extern "C" int sln_muon_step_f32(const sln_muon_desc_t *descs, int n, int steps, float eps, const double *sqnorm,
                                 float max_norm, float momentum, int nesterov, void *workspace, size_t workspace_bytes,
                                 sln_stream_t stream) {
    if (n < 0 || (n > 0 && !descs) || steps < 1 || steps > 64 || !(eps >= 1e-30f) || !sqnorm) return SLN_ERR_INVALID_ARG;
    for (int i = 0; i < n; ++i) {
        const sln_muon_desc_t &d = descs[i];
        if (d.rows == 0 || d.cols == 0) continue;
        if (!d.grad || !d.param || !d.momentum) return SLN_ERR_INVALID_ARG;
    }
    const OrthoRule rule = {sqnorm, max_norm, momentum, nesterov};
    return ortho_run<float>(descs, n, steps, eps, rule, workspace, workspace_bytes, (hipStream_t)stream);
}
