// C = A B^T on the 16-bit matrix instructions for operands that exist as one, two or three 16-bit parts per value
// (gfx950): the core of the Newton-Schulz products (ortho.hip) and of the 4-bit layer's gradients (mx4_grad.hip).
//
// Operand layout ("parts rows"): row r of a matrix with P parts is a run of k groups; a group holds 32 values of the
// contraction, part 0's 32 words, then part 1's, ... = 64 P bytes.  One k-step of one row is therefore ONE piece of 64 P
// contiguous bytes: the LDS DMA pays per 128-B line it touches, not per byte, and with two parts a row's step is a line.
// The contraction is padded to whole groups with zeros; rows need no padding (rows behind the last one are read as
// copies of it and their results dropped).
//
// Tile 128 x 128, four waves of 64 x 64 (2 x 2 accumulators of v_mfma_f32_32x32x16), k-step 32, two LDS stages (64 KB
// with two parts each: two workgroups per CU, one's loads beside the other's products).  Per step and wave: 12 products
// of 32 cycles per 16 values of k for 8 fragment reads -- the matrix pipe is the bound, LDS (two thirds of it) is not.
#pragma once
#include "common.h"

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

#define NT_TILE 128
#define NT_GROUP 32                      // values of the contraction per group

// which part products make up a * b
#define NT_SPLIT2 0   // two parts each: a1 b0 + a0 b1 + a0 b0 (a1 b1 is below the last bit of a0 b0's sum)
#define NT_EXACTB 1   // any number of parts of a, b exact in one part: sum over the parts of a, smallest first
#define NT_PLAIN 2    // one part each; two groups per step (the "parts" are neighbouring groups)

template <typename V>
__device__ __forceinline__ f32x16 nt_mfma(V a, V b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 nt_mfma<f16x8>(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 nt_mfma<b16x8>(b16x8 a, b16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// Position of 16-B chunk c of row `row` among the row's 4 P chunks in LDS: an XOR that puts the same chunk of eight
// neighbouring rows into eight different 16-B columns of the banks.
template <int P>
__device__ __forceinline__ int nt_swizzle(int row, int c) {
    if (P == 2) return c ^ (row & 7);
    return (c & ~3) | ((c & 3) ^ ((row >> 1) & 3));
}

template <int PA, int PB>
struct NtShape {
    static constexpr int A_BYTES = NT_TILE * 64 * PA, B_BYTES = NT_TILE * 64 * PB;
    static constexpr int STAGE = A_BYTES + B_BYTES;
};

// Byte offsets (within the operand, relative to its first row of the tile) of the pieces that this lane fetches.
template <int P>
__device__ __forceinline__ void nt_piece_offsets(int rows_left, long row_bytes, int wave, int lane, unsigned *off) {
#pragma unroll
    for (int q = 0; q < 2 * P; ++q) {
        const int slot = (q * 4 + wave) * 64 + lane;
        const int row = slot / (4 * P), c = slot - row * (4 * P);
        off[q] = (unsigned)((long)min(row, rows_left - 1) * row_bytes + nt_swizzle<P>(row, c) * 16);
    }
}

// acc[i][j]: this wave's 32 x 32 blocks of the tile (rows 64 (wave >> 1) + 32 i, columns 64 (wave & 1) + 32 j), summed
// over the k groups [g0, g1) (NT_PLAIN: pairs of groups).  `a` / `b`: first byte of the tile's first row; a_rows /
// b_rows: rows that exist from there on (> 0).  128 row_bytes must fit 32 bits.  Ends with every LDS read done but no
// barrier.
template <typename V, int PA, int PB, int MODE>
__device__ __forceinline__ void nt_tile(const char *a, long a_row_bytes, int a_rows, const char *b, long b_row_bytes,
                                        int b_rows, int g0, int g1, char *smem, f32x16 (&acc)[2][2]) {
    typedef __attribute__((address_space(3))) void lds_void;
    typedef __attribute__((address_space(1))) const void glb_void;
    typedef NtShape<PA, PB> S;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wr = wave >> 1, wc = wave & 1;
    unsigned aoff[2 * PA], boff[2 * PB];
    nt_piece_offsets<PA>(a_rows, a_row_bytes, wave, lane, aoff);
    nt_piece_offsets<PB>(b_rows, b_row_bytes, wave, lane, boff);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    auto issue = [&](int g, int stage) {
        const char *ga = a + (long)g * (64 * PA), *gb = b + (long)g * (64 * PB);
        char *l = smem + stage * S::STAGE + wave * 1024;
#pragma unroll
        for (int q = 0; q < 2 * PA; ++q)
            __builtin_amdgcn_global_load_lds((glb_void *)(ga + aoff[q]), (lds_void *)(l + q * 4096), 16, 0, 0);
#pragma unroll
        for (int q = 0; q < 2 * PB; ++q)
            __builtin_amdgcn_global_load_lds((glb_void *)(gb + boff[q]), (lds_void *)(l + S::A_BYTES + q * 4096), 16, 0,
                                             0);
    };
    const int frow = lane & 31, fhalf = lane >> 5;
    if (g0 < g1) issue(g0, 0);
    for (int g = g0; g < g1; ++g) {
        // this wave's pieces of the stage have landed, then everyone's; and everyone is done reading the other stage
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int stage = (g - g0) & 1;
        const char *la = smem + stage * S::STAGE, *lb = la + S::A_BYTES;
        if (g + 1 < g1) issue(g + 1, stage ^ 1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            V fa[2][PA], fb[2][PB];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int ra = 64 * wr + 32 * i + frow, rb = 64 * wc + 32 * i + frow;
#pragma unroll
                for (int p = 0; p < PA; ++p)
                    fa[i][p] = *(const V *)(la + ra * (64 * PA) + nt_swizzle<PA>(ra, 4 * p + 2 * kk + fhalf) * 16);
#pragma unroll
                for (int p = 0; p < PB; ++p)
                    fb[i][p] = *(const V *)(lb + rb * (64 * PB) + nt_swizzle<PB>(rb, 4 * p + 2 * kk + fhalf) * 16);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (MODE == NT_SPLIT2) {
                        acc[i][j] = nt_mfma<V>(fa[i][1], fb[j][0], acc[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][1], acc[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][0], acc[i][j]);
                    } else if constexpr (MODE == NT_EXACTB) {
#pragma unroll
                        for (int p = PA - 1; p >= 0; --p) acc[i][j] = nt_mfma<V>(fa[i][p], fb[j][0], acc[i][j]);
                    } else {
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][0], acc[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][1], fb[j][1], acc[i][j]);
                    }
                }
        }
    }
}

// Row (0 ... 31) of accumulator element r of a 32 x 32 block; the column is lane & 31.
__device__ __forceinline__ int nt_acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// Workgroups are dealt to the eight XCDs in turn: give each XCD (and its L2) one contiguous run of the work list.
__device__ __forceinline__ int nt_xcd_order(int bid, int n) {
    const int q = n >> 3, r = n & 7, x = bid & 7;
    return x * q + min(x, r) + (bid >> 3);
}
