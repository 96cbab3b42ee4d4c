// C = A B^T on the 16-bit matrix instructions for operands that exist as one, two or three 16-bit parts per value
// (gfx950): the core of the Newton-Schulz products (ortho.hip) and of the 4-bit layer's gradients (mx4_grad.hip).
//
// Operand layout ("parts rows"): row r of a matrix with P parts is a run of groups; a group holds 32 neighbouring values,
// part 0's 32 words, then part 1's, ... = 64 P bytes.  A row is padded to whole groups with zeros.  Where the contraction
// runs along the rows, one k-step of one row is ONE piece of 64 P contiguous bytes: the LDS DMA pays per 128-B line it
// touches, not per byte, and with two parts a row's step is a line.  The first operand may also be read across its rows
// (TRA: the matrix is [k][a], two parts): a stage is then 32 rows of TA / 32 groups, and the fragments come out of LDS
// through the transposing read.  Rows (TRA: groups) behind the last one are read as copies of it; what they give is dropped.
//
// Tile TA x TB, WR x WC waves, k-step 32, NST LDS stages filled by DMA, NST - 1 of them in flight.  v_mfma_f32_32x32x16:
// 32 cycles for a k of 16; a wave of 64 x 64 reads 8 fragments for 12 products (two parts each), one of 128 x 64 12 for 24.
// Measured alone (4096^3, two parts each, random values): 128 x 128, two workgroups per CU: 1089 TFLOP/s of products;
// 256 x 256, one of eight waves: 1305, which is what the library's fp16 product reaches on this card (1390 at 8192^3).
// The DMA goes through buffer descriptors: base and step in scalar registers, one 32-bit offset per piece and lane (with
// flat addresses the loop carries a 64-bit pointer per piece, and the 256 x 256 tile spills).
#pragma once
#include "common.h"

typedef __attribute__((address_space(3))) void nt_lds;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t nt_buffer(const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, (int)(unsigned)(bytes < 0xffffffffll ? bytes : 0xffffffffll),
                                             0x00020000);
}

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// which part products make up a * b
#define NT_SPLIT2 0   // two parts each: a1 b0 + a0 b1 + a0 b0 (a1 b1 is below the last bit of a0 b0's sum); without TRA, a
                      // wave of up to two blocks sums the corrections apart: the large sum is rounded once per 16 values, not
                      // three times (with TRA, P X, the roundings differ from element to element and average out)
#define NT_EXACTB 1   // any number of parts of a, b exact in one part: sum over the parts of a, smallest first

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

// Position of 16-B chunk c of row `row` among the row's 4 P chunks in LDS: an XOR that puts the same chunk of sixteen
// neighbouring rows -- the sixteen lanes that a 16-byte LDS read serves at a time -- into the sixteen 16-B columns of the
// 64 banks.
template <int P>
__device__ __forceinline__ int nt_swizzle(int row, int c) {
    if (P == 2) return c ^ ((row >> 1) & 7);
    return (c & ~3) | ((c & 3) ^ ((row >> 2) & 3));
}

template <int PA_, int PB_, int TA_, int TB_, int WR_, int WC_, int NST_>
struct NtShape {
    static constexpr int PA = PA_, PB = PB_, TA = TA_, TB = TB_, WR = WR_, WC = WC_, NST = NST_;
    static constexpr int NW = WR * WC, THREADS = NW * 64;
    static constexpr int A_BYTES = TA * 64 * PA, B_BYTES = TB * 64 * PB, STAGE = A_BYTES + B_BYTES, LDS = NST * STAGE;
    static constexpr int QA = A_BYTES / 1024 / NW, QB = B_BYTES / 1024 / NW;      // pieces of 1 KiB per wave and stage
    static constexpr int FA = TA / WR / 32, FB = TB / WC / 32;                    // 32 x 32 blocks per wave
    static_assert(QA * NW * 1024 == A_BYTES && QB * NW * 1024 == B_BYTES, "whole pieces per wave");
    static_assert(FA * WR * 32 == TA && FB * WC * 32 == TB, "whole blocks per wave");
    static_assert((QA + QB) * (NST - 2 > 0 ? NST - 2 : 0) < 64, "waits count to 63");
};

// Byte offsets (within the operand, relative to its first row of the tile) of the pieces that this lane fetches.
template <int P, int Q, int NW>
__device__ __forceinline__ void nt_piece_offsets(int rows_left, int64_t row_bytes, int wave, int lane, unsigned *off) {
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        const int slot = (q * NW + wave) * 64 + lane;
        const int row = slot / (4 * P), c = slot - row * (4 * P);
        off[q] = (unsigned)((int64_t)min(row, rows_left - 1) * row_bytes + nt_swizzle<P>(row, c) * 16);
    }
}

// Transposing reads of a 16-value step for FA blocks of 32 columns, two parts each: sixteen lanes turn a 4 (k) x 16 block,
// lane l addressing 8 B of row l / 4 and receiving column l.  f[i][p]: the fragment.  at[q]: byte of part (q & 1) of the
// blocks with i & 1 == q >> 1; STEP: bytes to row k + 4 and, times four, KK steps of 16 rows.  One asm block that ends with
// its own wait: behind the builtin the compiler waits for the DMA that is in flight, too.
template <int FA, int STEP, int KK, typename V>
__device__ __forceinline__ void nt_read_turned(const unsigned (&at)[4], V (&f)[FA][2]) {
    static_assert(FA == 2 || FA == 4, "blocks per wave");
    union { s16x4 h[2]; V v; } u[FA][2];
    constexpr int K0 = 4 * STEP * KK, K1 = K0 + STEP;
    if constexpr (FA == 2) {
        asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                     "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(u[0][0].h[0]), "=&v"(u[0][0].h[1]), "=&v"(u[0][1].h[0]), "=&v"(u[0][1].h[1]),
                       "=&v"(u[1][0].h[0]), "=&v"(u[1][0].h[1]), "=&v"(u[1][1].h[0]), "=&v"(u[1][1].h[1])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(K0), "n"(K1)
                     : "memory");
    } else {
        asm volatile("ds_read_b64_tr_b16 %0, %16 offset:%20\n\tds_read_b64_tr_b16 %1, %16 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %2, %17 offset:%20\n\tds_read_b64_tr_b16 %3, %17 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %4, %18 offset:%20\n\tds_read_b64_tr_b16 %5, %18 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %6, %19 offset:%20\n\tds_read_b64_tr_b16 %7, %19 offset:%21\n\t"
                     "ds_read_b64_tr_b16 %8, %16 offset:%22\n\tds_read_b64_tr_b16 %9, %16 offset:%23\n\t"
                     "ds_read_b64_tr_b16 %10, %17 offset:%22\n\tds_read_b64_tr_b16 %11, %17 offset:%23\n\t"
                     "ds_read_b64_tr_b16 %12, %18 offset:%22\n\tds_read_b64_tr_b16 %13, %18 offset:%23\n\t"
                     "ds_read_b64_tr_b16 %14, %19 offset:%22\n\tds_read_b64_tr_b16 %15, %19 offset:%23\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(u[0][0].h[0]), "=&v"(u[0][0].h[1]), "=&v"(u[0][1].h[0]), "=&v"(u[0][1].h[1]),
                       "=&v"(u[1][0].h[0]), "=&v"(u[1][0].h[1]), "=&v"(u[1][1].h[0]), "=&v"(u[1][1].h[1]),
                       "=&v"(u[2][0].h[0]), "=&v"(u[2][0].h[1]), "=&v"(u[2][1].h[0]), "=&v"(u[2][1].h[1]),
                       "=&v"(u[3][0].h[0]), "=&v"(u[3][0].h[1]), "=&v"(u[3][1].h[0]), "=&v"(u[3][1].h[1])
                     : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(K0), "n"(K1), "n"(K0 + 256), "n"(K1 + 256)
                     : "memory");
    }
#pragma unroll
    for (int i = 0; i < FA; ++i) { f[i][0] = u[i][0].v; f[i][1] = u[i][1].v; }
}

// acc[i][j]: this wave's 32 x 32 blocks of the tile (rows TA / WR * (wave / WC) + 32 i, columns TB / WC * (wave % WC) +
// 32 j), summed over the k groups [g0, g1).  `a` / `b`: first byte of the tile's first row; a_left / b_left: rows that
// exist from there on (> 0); TA (TB) rows must span less than 2^32 bytes.  TRA: `a` is the first byte of the tile's first
// group in row 0, a_left the groups that exist from there on, a_rows the rows.  Ends with every LDS read done but no
// barrier.
template <typename S, typename V, int MODE, bool TRA>
__device__ __forceinline__ void nt_tile(const char *a, int64_t a_row_bytes, int a_left, int a_rows, const char *b,
                                        int64_t b_row_bytes, int b_left, int g0, int g1, char *smem,
                                        f32x16 (&acc)[S::FA][S::FB]) {
#ifdef __HIP_DEVICE_COMPILE__                      // (the host pass knows no buffer descriptors in templates)
    constexpr int PA = S::PA, PB = S::PB, QA = S::QA, QB = S::QB, NW = S::NW;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wr = wave / S::WC, wc = wave % S::WC;
    unsigned aoff[QA], boff[QB];
    if constexpr (!TRA) {
        nt_piece_offsets<PA, QA, NW>(a_left, a_row_bytes, wave, lane, aoff);
    } else {                                       // row of the stage, offset within it
#pragma unroll
        for (int q = 0; q < QA; ++q) {
            const int slot = (q * NW + wave) * 64 + lane, k = slot / (S::TA / 4), p = slot % (S::TA / 4);
            const int unit = (p >> 2) ^ (k & 3);
            aoff[q] = (unsigned)(k * a_row_bytes + min(unit >> 1, a_left - 1) * 128 + (unit & 1) * 64 + (p & 3) * 16);
        }
    }
    nt_piece_offsets<PB, QB, NW>(b_left, b_row_bytes, wave, lane, boff);
#pragma unroll
    for (int i = 0; i < S::FA; ++i)
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    constexpr bool APART = MODE == NT_SPLIT2 && !TRA && S::FA * S::FB <= 2;
    f32x16 cor[APART ? S::FA : 1][APART ? S::FB : 1];
    if constexpr (APART) {
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int j = 0; j < S::FB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) cor[i][j][r] = 0.f;
    }

    const __amdgpu_buffer_rsrc_t bb = nt_buffer(b, INT64_MAX), ba0 = nt_buffer(a, INT64_MAX);
    auto issue = [&](int g) {
        char *l = smem + (g - g0) % S::NST * S::STAGE + wave * 1024;
        // (TRA: rows behind the last one lie outside the descriptor and arrive as zeros)
        const __amdgpu_buffer_rsrc_t ba =
            TRA ? nt_buffer(a + 32 * (int64_t)g * a_row_bytes, (int64_t)(a_rows - 32 * g) * a_row_bytes) : ba0;
#pragma unroll
        for (int q = 0; q < QA; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ba, (nt_lds *)(l + q * (NW * 1024)), 16, aoff[q],
                                                     TRA ? 0u : (unsigned)g * (64 * PA), 0, 0);
#pragma unroll
        for (int q = 0; q < QB; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(bb, (nt_lds *)(l + S::A_BYTES + q * (NW * 1024)), 16, boff[q],
                                                     (unsigned)g * (64 * PB), 0, 0);
    };
    const int frow = lane & 31, fhalf = lane >> 5;
    unsigned tr_off[4];
    if constexpr (TRA) {                           // row k of the first step, part q & 1 of block q >> 1 (of this wave)
        const int k = 8 * fhalf + ((lane >> 2) & 3), unit = S::TA / S::WR / 16 * wr;
#pragma unroll
        for (int q = 0; q < 4; ++q)
            tr_off[q] = k * (S::TA * 4) + ((unit + q) ^ (k & 3)) * 64 + (frow >> 4) * 32 + (lane & 3) * 8;
    }
#pragma unroll
    for (int s = 0; s < S::NST - 1; ++s)
        if (g0 + s < g1) issue(g0 + s);
    for (int g = g0; g < g1; ++g) {
        // this wave's pieces of the stage have landed (later stages' may be in flight), then everyone's; and everyone is
        // done reading the stage before, whose buffer the next DMA fills
        if (S::NST > 2 && g + S::NST - 2 < g1)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((QA + QB) * (S::NST > 2 ? S::NST - 2 : 0)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const char *la = smem + (g - g0) % S::NST * S::STAGE, *lb = la + S::A_BYTES;
        if (g + S::NST - 1 < g1) issue(g + S::NST - 1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            V fa[S::FA][PA], fb[S::FB][PB];
#pragma unroll
            for (int j = 0; j < S::FB; ++j) {
                const int row = S::TB / S::WC * wc + 32 * j + frow;
#pragma unroll
                for (int p = 0; p < PB; ++p)
                    fb[j][p] = *(const V *)(lb + row * (64 * PB) + nt_swizzle<PB>(row, 4 * p + 2 * kk + fhalf) * 16);
            }
            if constexpr (TRA) {
                unsigned at[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) at[q] = (unsigned)(uintptr_t)(nt_lds *)la + tr_off[q];
                if (kk == 0) nt_read_turned<S::FA, 4 * (S::TA * 4), 0>(at, fa);
                else nt_read_turned<S::FA, 4 * (S::TA * 4), 1>(at, fa);
            } else {
#pragma unroll
                for (int i = 0; i < S::FA; ++i) {
                    const int row = S::TA / S::WR * wr + 32 * i + frow;
#pragma unroll
                    for (int p = 0; p < PA; ++p)
                        fa[i][p] = *(const V *)(la + row * (64 * PA) + nt_swizzle<PA>(row, 4 * p + 2 * kk + fhalf) * 16);
                }
            }
#pragma unroll
            for (int i = 0; i < S::FA; ++i)
#pragma unroll
                for (int j = 0; j < S::FB; ++j) {
                    if constexpr (APART) {
                        cor[i][j] = nt_mfma<V>(fa[i][1], fb[j][0], cor[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][0], acc[i][j]);
                        cor[i][j] = nt_mfma<V>(fa[i][0], fb[j][1], cor[i][j]);
                    } else if constexpr (MODE == NT_SPLIT2) {
                        acc[i][j] = nt_mfma<V>(fa[i][1], fb[j][0], acc[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][1], acc[i][j]);
                        acc[i][j] = nt_mfma<V>(fa[i][0], fb[j][0], acc[i][j]);
                    } else {
#pragma unroll
                        for (int p = PA - 1; p >= 0; --p) acc[i][j] = nt_mfma<V>(fa[i][p], fb[j][0], acc[i][j]);
                    }
                }
        }
    }
    if constexpr (APART) {
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int j = 0; j < S::FB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] += cor[i][j][r];
    }
#endif
}

// Row (0 ... 31) of accumulator element r of a 32 x 32 block; the column is lane & 31.
__device__ __forceinline__ int nt_acc_row(int r, int lane) { return (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5); }

// Rows 16 h + 8 (lane >> 5) ... + 7 of column lane & 31 of a 32 x 32 block: the two halves of the wave trade four values,
// so that a lane's eight are neighbours (one 16-byte store of 16-bit words).
__device__ __forceinline__ void nt_acc_rows8(const f32x16 &acc, int h, float *v) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[8 * h + e]), __float_as_uint(acc[8 * h + 4 + e]),
                                                         false, false);
        v[e] = __uint_as_float(s[0]);
        v[4 + e] = __uint_as_float(s[1]);
    }
}

// The same where the list holds items of different lengths, the long ones first: runs of four in turn.
__device__ __forceinline__ int nt_xcd_runs(int bid, int n) {
    const int k = bid >> 3, at = ((k >> 2) * 8 + (bid & 7)) * 4 + (k & 3);
    return n - bid <= n % 32 ? bid : at;           // (the last n % 32 items stay where they are)
}

// Workgroups are dealt to the eight XCDs in turn: give each XCD (and its L2) one contiguous run of the work list.
__device__ __forceinline__ int nt_xcd_order(int bid, int n) {
    const int q = n >> 3, r = n & 7, x = bid & 7;
    return x * q + min(x, r) + (bid >> 3);
}
