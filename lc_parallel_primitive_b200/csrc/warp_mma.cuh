// Warp-level products of 16-bit tiles in shared memory (ldmatrix, mma.sync
// m16n8k16 bf16), and the split of float32 values into two bf16 parts.
//
// A tile has rows of COLS bf16 elements (64 or 128); its 16-byte pieces are
// permuted within a row by the row's number modulo 8, so that 8 rows at the
// same column lie in different banks.
#pragma once
#include <cuda_bf16.h>
#include "bulk.cuh"
#include "common.cuh"

namespace lcpp {

template <int COLS>
__device__ __forceinline__ uint32_t tile_at(uint32_t tile, int row, int piece) {
    return tile + row * (COLS * 2) + ((piece ^ (row & 7)) << 4);
}
// The pair of elements (row, col), (row, col + 1), col even.
template <int COLS>
__device__ __forceinline__ uint32_t tile_word(uint32_t tile, int row, int col) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(tile_at<COLS>(tile, row, col >> 3) + (col & 7) * 2));
    return v;
}

// 16-byte copy to shared memory; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// rows x COLS elements from rows `stride` elements apart; zeros beyond `have_rows` and `have_cols` (a multiple of 8).
template <int COLS>
__device__ __forceinline__ void tile_load(uint32_t tile, const __nv_bfloat16* from, uint64_t stride, int rows, int have_rows,
                                          int have_cols, int thread, int threads) {
    for (int i = thread; i < rows * (COLS / 8); i += threads) {
        const int r = i / (COLS / 8), c = i % (COLS / 8);
        const bool have = r < have_rows && c * 8 < have_cols;
        cp_async16_fill(tile_at<COLS>(tile, r, c), have ? from + r * stride + c * 8 : from, have ? 16 : 0);
    }
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// 16 x 16 pieces of a tile as operands.  (row, piece): the first row and 16-byte piece of the block.
// A fragment (m16 k16): a stored [m][k], a_t stored [k][m].
template <int COLS>
__device__ __forceinline__ void load_a(uint32_t (&r)[4], uint32_t tile, int row, int piece, int lane) {
    ldmatrix4(r, tile_at<COLS>(tile, row + (lane & 15), piece + (lane >> 4)));
}
template <int COLS>
__device__ __forceinline__ void load_a_t(uint32_t (&r)[4], uint32_t tile, int row, int piece, int lane) {
    ldmatrix4_t(r, tile_at<COLS>(tile, row + (lane & 7) + (lane >> 4) * 8, piece + ((lane >> 3) & 1)));
}
// Two B fragments (k16 n8 each: r[0], r[1] and r[2], r[3]): b stored [n][k], b_t stored [k][n].
template <int COLS>
__device__ __forceinline__ void load_b(uint32_t (&r)[4], uint32_t tile, int row, int piece, int lane) {
    ldmatrix4(r, tile_at<COLS>(tile, row + (lane & 7) + (lane >> 4) * 8, piece + ((lane >> 3) & 1)));
}
template <int COLS>
__device__ __forceinline__ void load_b_t(uint32_t (&r)[4], uint32_t tile, int row, int piece, int lane) {
    ldmatrix4_t(r, tile_at<COLS>(tile, row + (lane & 15), piece + (lane >> 4)));
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// (x, y) as pairs of bf16: hi the roundings, lo what they leave, itself rounded (the sum is off by 2^-18 at most).
__device__ __forceinline__ void split_bf16(float x, float y, uint32_t& hi, uint32_t& lo) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(y), "f"(x));
    const float rx = x - __uint_as_float(hi << 16), ry = y - __uint_as_float(hi & 0xffff0000u);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(lo) : "f"(ry), "f"(rx));
}
__device__ __forceinline__ float bf16_low(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float bf16_high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
// Accumulators of two neighbouring 16 x 8 tiles as the fragment of the 16 x 16 block they are: as A (m = rows), and as
// two B fragments with n = rows: (f[0], f[2]) rows 0-7, (f[1], f[3]) rows 8-15.
__device__ __forceinline__ void split_block(const float (&c0)[4], const float (&c1)[4], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    split_bf16(c0[0], c0[1], hi[0], lo[0]);
    split_bf16(c0[2], c0[3], hi[1], lo[1]);
    split_bf16(c1[0], c1[1], hi[2], lo[2]);
    split_bf16(c1[2], c1[3], hi[3], lo[3]);
}

}  // namespace lcpp
