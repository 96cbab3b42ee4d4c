// Newton-Schulz orthogonalisation of many matrices at once, and the optimiser step built on it (gfx950).
//
//   X <- G / (|G|_F + eps), on the transpose where G is taller than wide (so X is m x n, m <= n)
//   `steps` times:  A = X X^T,  P = a I + b A + c A^2,  X <- P X        (a, b, c) = (3.4445, -4.7750, 2.0315)
//
// maps every singular value s of X to p(s) = a s + b s^3 + c s^5, again and again: in five steps all of (0.005, 1] come
// into 0.68 ... 1.14, so X ends near the orthogonal factor U V^T of G.  p keeps [0, 1.21] inside [0, 1.21], hence
// |X|_2 <= 1.21, |A|_2 <= 1.47, |P|_2 <= 3.45 throughout and a FIXED power-of-two scale (2^14) puts every operand into
// fp16's range: an operand is two fp16 parts of value * 2^14 (22 ... 23 bits for values above 2^-17, an absolute floor of
// 2^-39 below), a product of two is three matrix instructions into an fp32 accumulator.  No pass looks for a maximum.
// Where eps outweighs |G| (|X|_F = r << 1) the operand holds X 2^h instead, h = floor(-log2 r) in the first step and two
// less in each later one (|X| grows by at most 3.45 < 4 a step): then A is held times 4^h.
//
// Launches (all matrices of a call in each of them; a work list in the workspace, made by the first launch):
//   ortho_norm_kernel    partial sums of squares in double (the optimiser: also the momentum update), the work lists
//   ortho_split_kernel   u = G / (|G| + eps) -> parts of X [m][n] and of X^T [n][m]
//   per step: ortho_gram_kernel    A's tiles on and above the diagonal (A is symmetric), the contraction over n cut so that
//                                  the launch fills the chip; one cut: parts of A are written (both triangles), several:
//                                  fp32 partial tiles, added in order by ortho_join_kernel
//             ortho_poly_kernel    P's tiles on and above the diagonal from A A^T, parts of both triangles
//             ortho_apply_kernel   X <- P X from P's rows and X^T's rows: parts of X (next step's Gram matrix) and of X^T
//                                  (next step's product); the last step writes the result, or updates the weights.
// Every contraction runs along rows of both operands: that is why X is kept both ways.
#include "mfma_nt.h"

#define ORTHO_BATCH 32                     // matrices per ortho_norm_kernel launch (descriptors travel by value)
#define ORTHO_CHUNK 16384                  // elements per partial sum of squares
#define ORTHO_SCALE 16384.0f               // 2^14
#define ORTHO_UNSCALE 6.103515625e-05f     // 2^-14
#define ORTHO_PITCH 133                    // floats per row of the 64-row epilogue slab: odd, 8 * 133 = 40 mod 64
#define ORTHO_LDS (2 * NtShape<2, 2>::STAGE)

static_assert(64 * ORTHO_PITCH * 4 <= ORTHO_LDS, "epilogue slab must fit the operand stages");

// What one launch of ortho_norm_kernel is told about a matrix (by value), and the entry it leaves in the table.
struct OrthoProb {
    const void *g;         // rows x cols, row stride gs
    void *out;             // rows x cols, row stride os (the optimiser: the weights)
    float *buf;            // the optimiser's momentum, row stride cols; NULL: plain orthogonalisation
    int64_t gs, os, off;   // off: byte offset of this matrix's operands in the workspace
    int32_t rows, cols;
    int32_t part0, nparts; // its partial sums of squares
    int32_t sym0, gram0, apply0, nsplit;   // first entries in the work lists, cuts of the Gram contraction
    float lr, decay;       // update: p = p * decay - lr * X
    int32_t shift;         // h of the first step (ortho_split_kernel)
};

struct OrthoTile { int32_t prob, ij, first, split; };   // ij = row tile << 16 | column tile; first: gram entry of cut 0

struct OrthoTable {
    OrthoProb *prob;
    OrthoTile *sym, *gram, *apply;
    double *part;
    char *ws;
    float *slab;           // partial Gram tiles, NT_TILE^2 floats per gram entry
};

struct OrthoBatch { OrthoProb p[ORTHO_BATCH]; };

__host__ __device__ __forceinline__ int ortho_m(const OrthoProb &p) { return p.rows < p.cols ? p.rows : p.cols; }
__host__ __device__ __forceinline__ int ortho_n(const OrthoProb &p) { return p.rows < p.cols ? p.cols : p.rows; }
__host__ __device__ __forceinline__ int64_t ortho_row_bytes(int k) { return (int64_t)((k + 31) / 32) * 128; }

// operands of a matrix inside the workspace: X, X^T (two, in turn), A, P
struct OrthoOperands { char *x, *xt[2], *a, *p; };
__device__ __forceinline__ OrthoOperands ortho_operands(const OrthoProb &p, char *ws) {
    const int m = ortho_m(p), n = ortho_n(p);
    const int64_t bx = m * ortho_row_bytes(n), bt = n * ortho_row_bytes(m), bs = m * ortho_row_bytes(m);
    OrthoOperands o;
    o.x = ws + p.off;
    o.xt[0] = o.x + bx;
    o.xt[1] = o.xt[0] + bt;
    o.a = o.xt[1] + bt;
    o.p = o.a + bs;
    return o;
}
static int64_t ortho_operand_bytes(const OrthoProb &p) {
    const int m = ortho_m(p), n = ortho_n(p);
    return m * ortho_row_bytes(n) + 2 * n * ortho_row_bytes(m) + 2 * m * ortho_row_bytes(m);
}

// 2^(sign h) for step `step`
__device__ __forceinline__ float ortho_shift(const OrthoProb &p, int step, int sign) {
    return ldexpf(1.f, sign * max(0, p.shift - 2 * step));
}

template <typename T>
__device__ __forceinline__ float ortho_load(const void *p, int64_t i) { return (float)((const T *)p)[i]; }

// The clip coefficient and the verdict of the optimiser's guard (a non-finite norm: the step is not applied).
__device__ __forceinline__ bool ortho_clip(const double *sqnorm, float max_norm, float &cf) {
    const double sq = sqnorm[0];
    const double coef = (double)max_norm / (sqrt(sq) + 1e-6);
    cf = coef < 1.0 ? (float)coef : 1.0f;
    return sq >= 0.0 && sq < INFINITY;
}

// ------------------------------------------------------------------------------------------------ norms and lists
// Block (c, i): elements [c, c + 1) * ORTHO_CHUNK of matrix i (row-major order) -> one partial sum of squares, added in a
// fixed order.  The optimiser (buf != NULL): b <- momentum b + cf g is written on the way and the sum is that of
// u = cf g + momentum b (nesterov) or u = b.  Memory-bound: 4 B read (optimiser: 8 read + 4 written) per element.
template <typename T>
__global__ __launch_bounds__(256) void ortho_norm_kernel(OrthoBatch batch, int prob0, OrthoTable tab,
                                                         const double *__restrict__ sqnorm, float max_norm,
                                                         float momentum, int nesterov) {
    __shared__ double s_red[4];
    const OrthoProb &p = batch.p[blockIdx.y];
    const int t = threadIdx.x, chunk = blockIdx.x;
    const int m = ortho_m(p), n = ortho_n(p);
    const int tm = (m + NT_TILE - 1) / NT_TILE, tn = (n + NT_TILE - 1) / NT_TILE;
    if (chunk == 0) {
        if (t == 0) tab.prob[prob0 + blockIdx.y] = p;
        const int prob = prob0 + blockIdx.y, nsym = tm * (tm + 1) / 2;
        for (int e = t; e < tm * tm; e += 256) {
            const int i = e / tm, j = e - i * tm;
            if (j < i) continue;
            const int s = i * tm - i * (i - 1) / 2 + (j - i);
            const OrthoTile tile = {prob, i << 16 | j, p.gram0 + s, p.nsplit};
            tab.sym[p.sym0 + s] = tile;
            for (int k = 0; k < p.nsplit; ++k) {
                const OrthoTile cut = {prob, i << 16 | j, p.gram0 + s, k};
                tab.gram[p.gram0 + k * nsym + s] = cut;
            }
        }
        for (int e = t; e < tm * tn; e += 256) {
            const int j = e / tm, i = e - j * tm;
            const OrthoTile tile = {prob, i << 16 | j, 0, 0};
            tab.apply[p.apply0 + e] = tile;
        }
    }
    if (chunk >= p.nparts) return;
    float cf = 1.f;
    bool apply = true;
    if (p.buf) apply = ortho_clip(sqnorm, max_norm, cf);
    const int64_t total = (int64_t)p.rows * p.cols, e0 = (int64_t)chunk * ORTHO_CHUNK;
    const int64_t e1 = min(total, e0 + ORTHO_CHUNK);
    double acc = 0.0;
    const bool flat = p.gs == p.cols;
    auto one = [&](float g, float *b) {
        float u = g;
        if (p.buf) {
            const float gc = g * cf, nb = momentum * *b + gc;
            if (apply) *b = nb;
            u = nesterov ? gc + momentum * nb : nb;
        }
        acc += (double)u * u;
    };
    if (flat && sizeof(T) == 4 && !(((uintptr_t)p.g | (uintptr_t)p.buf) & 15)) {
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
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if ((t & 63) == 0) s_red[t >> 6] = acc;
    __syncthreads();
    if (t == 0) tab.part[p.part0 + chunk] = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
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

// A 64 x 128 slab (rows i0 ..., columns j0 ... of an R x C matrix) from LDS to parts of the matrix (`dst`: R rows of
// C values) and of its transpose (`dst_t`: C rows of R values); either may be NULL.  Values behind the last column (row)
// are the zeros that pad the contraction: `keep` of a lane's values says so.
__device__ __forceinline__ void ortho_store_slab(const float *slab, int i0, int j0, int R, int C, char *dst, char *dst_t) {
    const int t = threadIdx.x;
    if (dst) {
        const int64_t rb = ortho_row_bytes(C);
        const int cpad = (C + 31) & ~31;
        for (int e = t; e < 64 * 16; e += 256) {
            const int r = e >> 4, k = j0 + (e & 15) * 8;
            if (i0 + r >= R || k >= cpad) continue;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = k + q < C ? slab[r * ORTHO_PITCH + (e & 15) * 8 + q] : 0.f;
            ortho_store8(ortho_at(dst, rb, i0 + r, k), v);
        }
    }
    if (dst_t) {
        const int64_t rb = ortho_row_bytes(R);
        const int rpad = (R + 31) & ~31;
        for (int e = t; e < 128 * 8; e += 256) {
            const int c = e >> 3, k = i0 + (e & 7) * 8;
            if (j0 + c >= C || k >= rpad) continue;
            float v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) v[q] = k + q < R ? slab[((e & 7) * 8 + q) * ORTHO_PITCH + c] : 0.f;
            ortho_store8(ortho_at(dst_t, rb, j0 + c, k), v);
        }
    }
}

// Accumulators of slab h (the two waves that hold rows 64 h ... 64 h + 63) to LDS, in units of the values.
__device__ __forceinline__ void ortho_slab_from_acc(float *slab, const f32x16 (&acc)[2][2], int h, float unscale) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((wave >> 1) != h) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                slab[(32 * i + nt_acc_row(r, lane)) * ORTHO_PITCH + 64 * (wave & 1) + 32 * j + (lane & 31)] =
                    acc[i][j][r] * unscale;
}

// ------------------------------------------------------------------------------------------------ G -> X, X^T
// Block = one 128 x 128 tile of X in two 64-row slabs.  Reads 4 B (optimiser: 8, u is made again from g and the new
// momentum), writes 8 B per element.
template <typename T>
__global__ __launch_bounds__(256) void ortho_split_kernel(OrthoTable tab, const double *__restrict__ sqnorm,
                                                          float max_norm, float momentum, int nesterov, float eps) {
    __shared__ float slab[64 * ORTHO_PITCH];
    __shared__ double s_red[4];
    const OrthoTile w = tab.apply[blockIdx.x];
    const OrthoProb p = tab.prob[w.prob];
    const int t = threadIdx.x, m = ortho_m(p), n = ortho_n(p);
    double acc = 0.0;
    for (int i = t; i < p.nparts; i += 256) acc += tab.part[p.part0 + i];
    for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o);
    if ((t & 63) == 0) s_red[t >> 6] = acc;
    __syncthreads();
    const double norm = sqrt((s_red[0] + s_red[1]) + (s_red[2] + s_red[3]));
    const float inv = (float)(1.0 / (norm + (double)eps));
    const double r = norm / (norm + (double)eps);
    int shift = 0;
    if (r > 0.0 && r < 1.0) {
        frexp(r, &shift);                          // r < 2^shift
        shift = min(max(-shift, 0), 126);
    }
    if (w.ij == 0 && t == 0) tab.prob[w.prob].shift = shift;
    const float up = ldexpf(1.f, shift);           // |g| up <= norm + eps
    float cf = 1.f;
    if (p.buf) ortho_clip(sqnorm, max_norm, cf);
    const bool tall = p.rows > p.cols;
    const OrthoOperands o = ortho_operands(p, tab.ws);
    const int i0 = (w.ij >> 16) * NT_TILE, j0 = (w.ij & 0xffff) * NT_TILE;
    auto value = [&](int r, int c) {               // of G, original orientation
        const float g = ortho_load<T>(p.g, (int64_t)r * p.gs + c);
        if (!p.buf) return g * up * inv;
        const float b = p.buf[(int64_t)r * p.cols + c];
        return (nesterov ? g * cf + momentum * b : b) * up * inv;
    };
    for (int h = 0; h < 2; ++h) {
        const int r0 = i0 + 64 * h;
        if (r0 >= m) break;
        __syncthreads();
        for (int e = t; e < 64 * 128; e += 256) {
            int i, j;                               // of the slab; the faster one runs along G's rows
            if (tall) { i = e & 63; j = e >> 6; } else { j = e & 127; i = e >> 7; }
            const bool in = r0 + i < m && j0 + j < n;
            slab[i * ORTHO_PITCH + j] = in ? (tall ? value(j0 + j, r0 + i) : value(r0 + i, j0 + j)) : 0.f;
        }
        __syncthreads();
        ortho_store_slab(slab, r0, j0, m, n, o.x, o.xt[0]);
    }
}

// ------------------------------------------------------------------------------------------------ A = X X^T
__global__ __launch_bounds__(256, 2) void ortho_gram_kernel(OrthoTable tab, int ntiles) {
    __shared__ __attribute__((aligned(128))) char smem[ORTHO_LDS];
    const int at = nt_xcd_order(blockIdx.x, ntiles);
    const OrthoTile w = tab.gram[at];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws);
    const int m = ortho_m(p), n = ortho_n(p);
    const int i0 = (w.ij >> 16) * NT_TILE, j0 = (w.ij & 0xffff) * NT_TILE;
    const int64_t rb = ortho_row_bytes(n);
    const int groups = (n + 31) / 32;
    const int g0 = (int)((int64_t)groups * w.split / p.nsplit), g1 = (int)((int64_t)groups * (w.split + 1) / p.nsplit);
    f32x16 acc[2][2];
    nt_tile<f16x8, 2, 2, NT_SPLIT2>(o.x + i0 * rb, rb, m - i0, o.x + j0 * rb, rb, m - j0, g0, g1, smem, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (p.nsplit > 1) {
        float *slab = tab.slab + (int64_t)at * NT_TILE * NT_TILE;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    slab[(64 * (wave >> 1) + 32 * i + nt_acc_row(r, lane)) * NT_TILE + 64 * (wave & 1) + 32 * j +
                         (lane & 31)] = acc[i][j][r];
        return;
    }
    for (int h = 0; h < 2; ++h) {
        if (i0 + 64 * h >= m) break;
        __syncthreads();
        ortho_slab_from_acc((float *)smem, acc, h, ORTHO_UNSCALE * ORTHO_UNSCALE);
        __syncthreads();
        ortho_store_slab((const float *)smem, i0 + 64 * h, j0, m, m, o.a, i0 == j0 ? nullptr : o.a);
    }
}

// The cuts of a Gram tile, added in order.  Block = 64 rows of one tile.
__global__ __launch_bounds__(256) void ortho_join_kernel(OrthoTable tab) {
    __shared__ float slab[64 * ORTHO_PITCH];
    const OrthoTile w = tab.sym[blockIdx.x >> 1];
    const int h = blockIdx.x & 1;
    const OrthoProb p = tab.prob[w.prob];
    const int m = ortho_m(p), tm = (m + NT_TILE - 1) / NT_TILE, nsym = tm * (tm + 1) / 2;
    const int i0 = (w.ij >> 16) * NT_TILE + 64 * h, j0 = (w.ij & 0xffff) * NT_TILE;
    if (p.nsplit == 1 || i0 >= m) return;
    const OrthoOperands o = ortho_operands(p, tab.ws);
    const float4 *src = (const float4 *)(tab.slab + (int64_t)w.first * NT_TILE * NT_TILE + 64 * h * NT_TILE);
    for (int e = threadIdx.x; e < 64 * 32; e += 256) {
        float4 s = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < p.nsplit; ++k) {
            const float4 v = src[(int64_t)k * nsym * (NT_TILE * NT_TILE / 4) + e];
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        float *d = slab + (e >> 5) * ORTHO_PITCH + (e & 31) * 4;
        const float u = ORTHO_UNSCALE * ORTHO_UNSCALE;
        d[0] = s.x * u; d[1] = s.y * u; d[2] = s.z * u; d[3] = s.w * u;
    }
    __syncthreads();
    ortho_store_slab(slab, i0, j0, m, m, o.a, (w.ij >> 16) == (w.ij & 0xffff) ? nullptr : o.a);
}

// ------------------------------------------------------------------------------------------------ P = a I + b A + c A^2
__global__ __launch_bounds__(256, 2) void ortho_poly_kernel(OrthoTable tab, int ntiles, int step, float ca, float cb,
                                                            float cc) {
    __shared__ __attribute__((aligned(128))) char smem[ORTHO_LDS];
    const OrthoTile w = tab.sym[nt_xcd_order(blockIdx.x, ntiles)];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws);
    const int m = ortho_m(p);
    const int i0 = (w.ij >> 16) * NT_TILE, j0 = (w.ij & 0xffff) * NT_TILE;
    const int64_t rb = ortho_row_bytes(m);
    f32x16 acc[2][2];
    nt_tile<f16x8, 2, 2, NT_SPLIT2>(o.a + i0 * rb, rb, m - i0, o.a + j0 * rb, rb, m - j0, 0, (m + 31) / 32, smem, acc);
    const int t = threadIdx.x;
    float *slab = (float *)smem;
    const float down = ortho_shift(p, step, -1), down2 = down * down;
    for (int h = 0; h < 2; ++h) {
        const int r0 = i0 + 64 * h;
        if (r0 >= m) break;
        __syncthreads();
        ortho_slab_from_acc(slab, acc, h, cc * (down2 * down2) * (ORTHO_UNSCALE * ORTHO_UNSCALE));
        __syncthreads();
        for (int e = t; e < 64 * 16; e += 256) {     // + b A + a I, in place
            const int r = e >> 4, k = j0 + (e & 15) * 8;
            if (r0 + r >= m || k >= m) continue;
            const char *at = ortho_at(o.a, rb, r0 + r, k);
            const f16x8 h0 = *(const f16x8 *)at, h1 = *(const f16x8 *)(at + 64);
            float *d = slab + r * ORTHO_PITCH + (e & 15) * 8;
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float av = ((float)h0[q] + (float)h1[q]) * (ORTHO_UNSCALE * down2);
                d[q] += cb * av + (r0 + r == k + q ? ca : 0.f);
            }
        }
        __syncthreads();
        ortho_store_slab(slab, r0, j0, m, m, o.p, i0 == j0 ? nullptr : o.p);
    }
}

// ------------------------------------------------------------------------------------------------ X <- P X
// LAST: write the result in T (or update the weights: buf != NULL) instead of the next step's operands.
template <typename T, bool LAST>
__global__ __launch_bounds__(256, 2) void ortho_apply_kernel(OrthoTable tab, int ntiles, int step,
                                                             const double *__restrict__ sqnorm) {
    __shared__ __attribute__((aligned(128))) char smem[ORTHO_LDS];
    const OrthoTile w = tab.apply[nt_xcd_order(blockIdx.x, ntiles)];
    const OrthoProb p = tab.prob[w.prob];
    const OrthoOperands o = ortho_operands(p, tab.ws);
    const int m = ortho_m(p), n = ortho_n(p);
    const int i0 = (w.ij >> 16) * NT_TILE, j0 = (w.ij & 0xffff) * NT_TILE;
    const int64_t rb = ortho_row_bytes(m);
    f32x16 acc[2][2];
    nt_tile<f16x8, 2, 2, NT_SPLIT2>(o.p + i0 * rb, rb, m - i0, o.xt[step & 1] + j0 * rb, rb, n - j0, 0, (m + 31) / 32,
                                    smem, acc);
    const int t = threadIdx.x;
    const float *slab = (const float *)smem;
    const float unscale = ORTHO_UNSCALE * ORTHO_UNSCALE * ortho_shift(p, step, -1) * (LAST ? 1.f : ortho_shift(p, step + 1, 1));
    if (LAST && p.buf) {
        const double sq = sqnorm[0];
        if (!(sq >= 0.0 && sq < INFINITY)) return;
    }
    for (int h = 0; h < 2; ++h) {
        const int r0 = i0 + 64 * h;
        if (r0 >= m) break;
        __syncthreads();
        ortho_slab_from_acc((float *)smem, acc, h, unscale);
        __syncthreads();
        if (!LAST) {
            ortho_store_slab(slab, r0, j0, m, n, o.x, o.xt[(step & 1) ^ 1]);
            continue;
        }
        const bool tall = p.rows > p.cols;
        for (int e = t; e < 64 * 128; e += 256) {
            int i, j;
            if (tall) { i = e & 63; j = e >> 6; } else { j = e & 127; i = e >> 7; }
            if (r0 + i >= m || j0 + j >= n) continue;
            const int64_t at = tall ? (int64_t)(j0 + j) * p.os + r0 + i : (int64_t)(r0 + i) * p.os + j0 + j;
            const float v = slab[i * ORTHO_PITCH + j];
            if (p.buf) {
                float *d = (float *)p.out + at;
                *d = *d * p.decay - p.lr * v;
            } else {
                ((T *)p.out)[at] = (T)v;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
// Positions of everything in the workspace: a pure function of the shapes.
struct OrthoPlan {
    int64_t prob, sym, gram, apply, part, slab, operands, bytes;
    int nsym, ngram, napply, nparts, max_parts, joined;
};

static inline int64_t ortho_align(int64_t v) { return (v + 255) & ~(int64_t)255; }

// Cuts of the Gram contraction: enough work items that a launch over all matrices gives every CU its two workgroups, but
// no cut shorter than 8 k-steps (below that its partial tile costs more to write and add than it saves).
static inline int ortho_cut_groups(int64_t tile_groups) {
    const int64_t g = (tile_groups + 511) / 512;
    return g < 8 ? 8 : (g > (1 << 20) ? 1 << 20 : (int)g);
}

template <typename D>
static int ortho_plan(const D *d, int n, OrthoPlan &pl) {
    int64_t tile_groups = 0;
    for (int i = 0; i < n; ++i) {
        if (d[i].rows < 0 || d[i].cols < 0 || d[i].rows > (1 << 22) || d[i].cols > (1 << 22)) return SLN_ERR_INVALID_ARG;
        const int64_t m = d[i].rows < d[i].cols ? d[i].rows : d[i].cols, k = d[i].rows < d[i].cols ? d[i].cols : d[i].rows;
        if (m > 65535) return SLN_ERR_UNSUPPORTED;
        const int64_t tm = (m + NT_TILE - 1) / NT_TILE;
        tile_groups += tm * (tm + 1) / 2 * ((k + 31) / 32);
    }
    const int cut = ortho_cut_groups(tile_groups);
    int64_t nsym = 0, ngram = 0, napply = 0, nparts = 0, max_parts = 0, operands = 0, nprob = 0;
    bool joined = false;
    for (int i = 0; i < n; ++i) {
        if (d[i].rows == 0 || d[i].cols == 0) continue;
        OrthoProb p = {};
        p.rows = d[i].rows; p.cols = d[i].cols;
        const int64_t m = ortho_m(p), k = ortho_n(p);
        const int64_t tm = (m + NT_TILE - 1) / NT_TILE, tn = (k + NT_TILE - 1) / NT_TILE;
        const int64_t groups = (k + 31) / 32, nsplit = (groups + cut - 1) / cut;
        joined |= nsplit > 1;
        ++nprob;
        nsym += tm * (tm + 1) / 2;
        ngram += tm * (tm + 1) / 2 * nsplit;
        napply += tm * tn;
        const int64_t parts = ((int64_t)p.rows * p.cols + ORTHO_CHUNK - 1) / ORTHO_CHUNK;
        nparts += parts;
        if (parts > max_parts) max_parts = parts;
        operands += ortho_align(ortho_operand_bytes(p));
        if (tn > 65535 || nsym > (1 << 28) || ngram > (1 << 28) || napply > (1 << 28) || nparts > (1 << 28) ||
            max_parts > (1 << 24))
            return SLN_ERR_UNSUPPORTED;
    }
    int64_t at = 0;
    pl.prob = at; at += ortho_align(nprob * (int64_t)sizeof(OrthoProb));
    pl.sym = at; at += ortho_align(nsym * (int64_t)sizeof(OrthoTile));
    pl.gram = at; at += ortho_align(ngram * (int64_t)sizeof(OrthoTile));
    pl.apply = at; at += ortho_align(napply * (int64_t)sizeof(OrthoTile));
    pl.part = at; at += ortho_align(nparts * (int64_t)sizeof(double));
    pl.slab = at; at += joined ? ortho_align(ngram * (int64_t)(NT_TILE * NT_TILE * 4)) : 0;
    pl.operands = at; at += operands;
    pl.bytes = at;
    pl.nsym = (int)nsym; pl.ngram = (int)ngram; pl.napply = (int)napply;
    pl.nparts = (int)nparts; pl.max_parts = (int)max_parts; pl.joined = joined;
    return SLN_OK;
}

struct OrthoStep { const double *sqnorm; float max_norm, momentum; int nesterov; };

static void ortho_desc(const sln_ortho_desc_t &d, OrthoProb &p) {
    p.g = d.g; p.out = d.out; p.buf = nullptr;
    p.gs = d.g_stride; p.os = d.out_stride;
    p.lr = 0.f; p.decay = 1.f;
}
static void ortho_desc(const sln_muon_desc_t &d, OrthoProb &p) {
    p.g = d.grad; p.out = d.param; p.buf = d.momentum;
    p.gs = p.os = d.cols;
    p.lr = d.lr; p.decay = d.decay;
}

template <typename T, typename D>
static int ortho_run(const D *d, int n, int steps, float eps, const OrthoStep &st, void *workspace, size_t ws_bytes,
                     hipStream_t stream) {
    OrthoPlan pl;
    const int rc = ortho_plan(d, n, pl);
    if (rc != SLN_OK) return rc;
    if (pl.napply == 0) return SLN_OK;
    if (!workspace || ((uintptr_t)workspace & 255)) return SLN_ERR_INVALID_ARG;
    if (ws_bytes < (size_t)pl.bytes) return SLN_ERR_WORKSPACE;
    char *ws = (char *)workspace;
    const OrthoTable tab = {(OrthoProb *)(ws + pl.prob), (OrthoTile *)(ws + pl.sym), (OrthoTile *)(ws + pl.gram),
                            (OrthoTile *)(ws + pl.apply), (double *)(ws + pl.part), ws, (float *)(ws + pl.slab)};
    int64_t tile_groups = 0;
    for (int i = 0; i < n; ++i) {
        const int64_t m = d[i].rows < d[i].cols ? d[i].rows : d[i].cols, k = d[i].rows < d[i].cols ? d[i].cols : d[i].rows;
        const int64_t tm = (m + NT_TILE - 1) / NT_TILE;
        tile_groups += tm * (tm + 1) / 2 * ((k + 31) / 32);
    }
    const int cut = ortho_cut_groups(tile_groups);
    sln_enter();
    OrthoBatch batch;
    int prob0 = 0, inb = 0, batch_parts = 1, part0 = 0, sym0 = 0, gram0 = 0, apply0 = 0;
    int64_t off = pl.operands;
    auto flush = [&]() {
        if (inb == 0) return;
        hipLaunchKernelGGL((ortho_norm_kernel<T>), dim3(batch_parts, inb), dim3(256), 0, stream, batch, prob0, tab,
                           st.sqnorm, st.max_norm, st.momentum, st.nesterov);
        prob0 += inb; inb = 0; batch_parts = 1;
    };
    for (int i = 0; i < n; ++i) {
        if (d[i].rows == 0 || d[i].cols == 0) continue;
        OrthoProb &p = batch.p[inb];
        ortho_desc(d[i], p);
        p.rows = d[i].rows; p.cols = d[i].cols;
        const int m = ortho_m(p), k = ortho_n(p);
        const int tm = sln_div_up(m, NT_TILE), tn = sln_div_up(k, NT_TILE);
        p.off = off; off += ortho_align(ortho_operand_bytes(p));
        p.nsplit = ((k + 31) / 32 + cut - 1) / cut;
        p.part0 = part0; p.nparts = sln_div_up((long)p.rows * p.cols, ORTHO_CHUNK); part0 += p.nparts;
        p.sym0 = sym0; sym0 += tm * (tm + 1) / 2;
        p.gram0 = gram0; gram0 += tm * (tm + 1) / 2 * p.nsplit;
        p.apply0 = apply0; apply0 += tm * tn;
        if (p.nparts > batch_parts) batch_parts = p.nparts;
        if (++inb == ORTHO_BATCH) flush();
    }
    flush();
    hipLaunchKernelGGL((ortho_split_kernel<T>), dim3(pl.napply), dim3(256), 0, stream, tab, st.sqnorm, st.max_norm,
                       st.momentum, st.nesterov, eps);
    for (int s = 0; s < steps; ++s) {
        hipLaunchKernelGGL(ortho_gram_kernel, dim3(pl.ngram), dim3(256), 0, stream, tab, pl.ngram);
        if (pl.joined) hipLaunchKernelGGL(ortho_join_kernel, dim3(2 * pl.nsym), dim3(256), 0, stream, tab);
        hipLaunchKernelGGL(ortho_poly_kernel, dim3(pl.nsym), dim3(256), 0, stream, tab, pl.nsym, s, 3.4445f,
                           -4.7750f, 2.0315f);
        if (s + 1 < steps)
            hipLaunchKernelGGL((ortho_apply_kernel<T, false>), dim3(pl.napply), dim3(256), 0, stream, tab, pl.napply, s,
                               st.sqnorm);
        else
            hipLaunchKernelGGL((ortho_apply_kernel<T, true>), dim3(pl.napply), dim3(256), 0, stream, tab, pl.napply, s,
                               st.sqnorm);
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
    const OrthoStep st = {nullptr, 0.f, 0.f, 0};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case SLN_DTYPE_F32: return ortho_run<float>(descs, n, steps, eps, st, workspace, workspace_bytes, s);
        case SLN_DTYPE_BF16: return ortho_run<__bf16>(descs, n, steps, eps, st, workspace, workspace_bytes, s);
        case SLN_DTYPE_F16: return ortho_run<_Float16>(descs, n, steps, eps, st, workspace, workspace_bytes, s);
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
    const OrthoStep st = {sqnorm, max_norm, momentum, nesterov};
    return ortho_run<float>(descs, n, steps, eps, st, workspace, workspace_bytes, (hipStream_t)stream);
}
