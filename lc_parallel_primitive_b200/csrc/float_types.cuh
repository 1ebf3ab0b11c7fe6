// 2- and 4-byte floating element types of the sequence operators.  Arithmetic
// is always float32; an element is widened when it is loaded and rounded to
// nearest even once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <utility>
#include "common.cuh"

namespace lcpp {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Dispatch a functor over the three floating element types.
template <typename F>
inline lcpp_status dispatch_float(int dtype, F&& f) {
    switch (dtype) {
        case LCPP_F32: return f((float)0);
        case LCPP_F16: return f(__half());
        case LCPP_BF16: return f(__nv_bfloat16());
        default: return LCPP_ERR_INVALID_ARG;
    }
}

inline bool is_float_dtype(int dtype) { return dtype == LCPP_F32 || dtype == LCPP_F16 || dtype == LCPP_BF16; }

// Every pointer is a whole number of elements (of 2 bytes for the half types, else 4).
template <typename... P>
inline bool elements_aligned(int dtype, const P*... p) {
    return ((uintptr_t)0 | ... | (uintptr_t)p) % (dtype == LCPP_F16 || dtype == LCPP_BF16 ? 2 : 4) == 0;
}

// Memory that a call reads or writes: `rows` pieces of `bytes` bytes, `stride` bytes from one to the next.
struct Region {
    uintptr_t at;
    uint64_t rows, stride, bytes;
    Region(const void* p, uint64_t n) : Region(p, 1, n, n) {}
    Region(const void* p, uint64_t r, uint64_t s, uint64_t b)
        : at((uintptr_t)p), rows(p && b ? r : 0), stride(r > 1 ? s : b), bytes(b) {}
    // One piece lies on the other's, each row on its own.
    bool same(const Region& o) const { return at == o.at && rows == o.rows && stride == o.stride && bytes == o.bytes; }
    // Whether they have a byte in common.  Exact for one piece or equal strides (columns of one buffer, say); two
    // matrices of different strides within each other's bounds count as overlapping.
    bool meets(const Region& o) const {
        if (!rows || !o.rows) return false;
        Region a = joined(), b = o.joined();
        if (b.at < a.at) std::swap(a, b);
        const uint64_t d = b.at - a.at;
        if (d >= (a.rows - 1) * a.stride + a.bytes) return false;
        if (a.rows == 1 || (b.rows > 1 && b.stride != a.stride) || !a.stride) return true;
        return d % a.stride < a.bytes || (d % a.stride + b.bytes > a.stride && d / a.stride + 1 < a.rows);
    }
    template <typename... R>
    bool apart(const R&... others) const { return (!meets(others) && ...); }
    template <typename... R>
    bool apart_or_same(const R&... others) const { return ((same(others) || !meets(others)) && ...); }

  private:
    Region joined() const {  // rows without gaps are one piece
        Region r = *this;
        if (r.stride == r.bytes) r.bytes *= r.rows, r.stride = r.bytes, r.rows = 1;
        return r;
    }
};

}  // namespace lcpp
