// Warp-level products of float16 tiles in shared memory (ldmatrix, mma.sync m16n8k16) and float32 values as pairs of
// float16.
//
// Tiles are made of blocks with rows of 64 elements (128 bytes); the 16-byte pieces of a row are permuted by the row's
// number modulo 8, so that 8 rows at the same column lie in different banks.  The same image lies in global memory, so
// that a block is one bulk copy.
//
// A float32 value x enters a product as hi + lo: hi = f16(x s), lo = f16(x s - hi), with a power of two s that brings
// the largest value of the matrix to 2^14 .. 2^15.  That leaves 2^-23 of a value, or 2^-39 of the largest where lo is
// subnormal; hi hi + hi lo + lo hi leaves out 2^-22.  bf16 pairs would need no scale, but leave 2^-17.
#pragma once
#include <cuda_fp16.h>
#include "bulk.cuh"
#include "common.cuh"

namespace lcpp {

constexpr int BLOCK_COLS = 64, BLOCK_ROW = 128;  // elements and bytes of a row

// Byte of element (row, col) within a block.
__host__ __device__ __forceinline__ uint32_t block_at(uint32_t row, uint32_t col) {
    return row * BLOCK_ROW + ((((col >> 3) ^ row) & 7) << 4) + (col & 7) * 2;
}

// What a lane adds to a block's address and its first row's for 16 x 16 elements at columns 16 j (j = 0 .. 3).
struct LaneOffsets {
    uint32_t rows[4];   // a stored [m][k], b stored [k][n] (transposed on the way)
    uint32_t cols[4];   // b stored [n][k], a stored [k][m] (transposed on the way)
    __device__ __forceinline__ explicit LaneOffsets(int lane) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            rows[j] = (((2 * j + (lane >> 4)) ^ (lane & 7)) << 4) + (lane & 15) * BLOCK_ROW;
            cols[j] = (((2 * j + ((lane >> 3) & 1)) ^ (lane & 7)) << 4) + ((lane & 7) + (lane >> 4) * 8) * BLOCK_ROW;
        }
    }
};

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
// Fragments of the 16 x 16 elements at (row, 16 j) of a block: A (m16 k16), or two of B (k16 n8 each: r[0], r[1] and
// r[2], r[3]); _t where the block holds the operand's transpose.
__device__ __forceinline__ void load_a(uint32_t (&r)[4], uint32_t block, int row, int j, const LaneOffsets& o) {
    ldmatrix4(r, block + row * BLOCK_ROW + o.rows[j]);
}
__device__ __forceinline__ void load_a_t(uint32_t (&r)[4], uint32_t block, int row, int j, const LaneOffsets& o) {
    ldmatrix4_t(r, block + row * BLOCK_ROW + o.cols[j]);
}
__device__ __forceinline__ void load_b(uint32_t (&r)[4], uint32_t block, int row, int j, const LaneOffsets& o) {
    ldmatrix4(r, block + row * BLOCK_ROW + o.cols[j]);
}
__device__ __forceinline__ void load_b_t(uint32_t (&r)[4], uint32_t block, int row, int j, const LaneOffsets& o) {
    ldmatrix4_t(r, block + row * BLOCK_ROW + o.rows[j]);
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Both halves of a pair of B fragments.
__device__ __forceinline__ void mma_f16_2(float (&c0)[4], float (&c1)[4], const uint32_t (&a)[4], const uint32_t (&b)[4]) {
    mma_f16(c0, a, b[0], b[1]);
    mma_f16(c1, a, b[2], b[3]);
}

// ---- scales ------------------------------------------------------------------------------------------
// A power of two and its inverse.
struct Scale {
    float by, back;
};
// 1 / v for a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float power_inverse(float v) { return __int_as_float(0x7f000000 - __float_as_int(v)); }
// For the largest absolute value `most`: most * by is in [2^14, 2^15), by <= 2^LIMIT (1 for zeros).  The limits keep
// products of two scales, and a scale times a value that is not of its own matrix, within float32.  An infinity among the values
// would leave nothing of the others: all become NaN.
__device__ __forceinline__ Scale scale_of_field(int e, int field) {
    if (e == 255) return Scale{__int_as_float(0x7fffffff), __int_as_float(0x7fffffff)};
    if (e == 0) field = 127;
    return Scale{__int_as_float(field << 23), __int_as_float((254 - field) << 23)};
}
template <int LIMIT = 80>
__device__ __forceinline__ Scale scale_for(float most) {
    const int e = __float_as_int(most) >> 23 & 255;
    return scale_of_field(e, min(268 - e, 127 + LIMIT));
}
// The scale, or `by` if that is less.
__device__ __forceinline__ Scale scale_up_to(Scale s, float by) { return s.by > by ? Scale{by, power_inverse(by)} : s; }
// Of values that are `back` times smaller or larger than they stand here (a power of two): by / back is a power of 2^8, so that
// matrices of like size share it, and most * by is in [2^7, 2^15).
__device__ __forceinline__ Scale coarse_scale_for(float most, float back = 1.0f) {
    const int e = __float_as_int(most) >> 23 & 255, own = (__float_as_int(back) >> 23 & 255) - 127;
    return scale_of_field(e, own + ((min(141 - e, 80) - own) >> 3) * 8 + 127);
}
// The inverse scale of what is kept as float16: 0 of nothing (or of what is below float32's normal numbers, of which by = 1
// leaves nothing), which says nothing of the sizes beside it.
__device__ __forceinline__ float kept_back(float most, float back) { return most < 1.17549435e-38f ? 0.0f : back; }
__device__ __forceinline__ float warp_max(float v) {  // of values >= 0
    return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}
__device__ __forceinline__ float max3_abs(float m, float x, float y) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(x)), "f"(fabsf(y)));
    return r;
}
template <int N>
__device__ __forceinline__ float max_abs(const float (&c)[N][4]) {  // of the warp's accumulators
    float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) m0 = max3_abs(m0, c[n][0], c[n][1]), m1 = max3_abs(m1, c[n][2], c[n][3]);
    return warp_max(fmaxf(m0, m1));
}

// ---- two float32 at a time -------------------------------------------------------------------------
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void pair_split(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_sub(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// (x, y) *= (a, b)
__device__ __forceinline__ void scale_pair(float& x, float& y, uint64_t by) { pair_split(pair_mul(pair_of(x, y), by), x, y); }
template <int N>
__device__ __forceinline__ void scale_all(float (&c)[N][4], float by) {
    const uint64_t b = pair_of(by, by);
#pragma unroll
    for (int n = 0; n < N; ++n) scale_pair(c[n][0], c[n][1], b), scale_pair(c[n][2], c[n][3], b);
}

__device__ __forceinline__ uint32_t pack_f16(float x, float y) {
    uint32_t v;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(v) : "f"(y), "f"(x));
    return v;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) { return __half22float2(*(const __half2*)&v); }
__device__ __forceinline__ void split_f16(float x, float y, float s, uint32_t& hi, uint32_t& lo) {
    const uint64_t v = pair_mul(pair_of(x, y), pair_of(s, s));  // exact but where it is far below the largest
    float a, b;
    pair_split(v, a, b);
    hi = pack_f16(a, b);
    const float2 h = unpack_f16(hi);
    pair_split(pair_sub(v, pair_of(h.x, h.y)), a, b);
    lo = pack_f16(a, b);
}
// Accumulators of two neighbouring 16 x 8 tiles as the fragment of the 16 x 16 block they are: as A (m = rows), and as
// two B fragments with n = rows: (f[0], f[2]) rows 0-7, (f[1], f[3]) rows 8-15.
__device__ __forceinline__ void split_block(const float (&c0)[4], const float (&c1)[4], float s, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    split_f16(c0[0], c0[1], s, hi[0], lo[0]);
    split_f16(c0[2], c0[3], s, hi[1], lo[1]);
    split_f16(c1[0], c1[1], s, hi[2], lo[2]);
    split_f16(c1[2], c1[3], s, hi[3], lo[3]);
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
// 16-byte asynchronous copy to shared memory; `bytes` 0 writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

}  // namespace lcpp
