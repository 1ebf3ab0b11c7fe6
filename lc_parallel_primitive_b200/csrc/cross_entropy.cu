// Softmax cross entropy over a vocabulary from hidden states (DeviceCrossEntropy), without the logits in memory.
//
//   z = H W^T,  logsum_i = log sum_v exp(z_iv),  loss_i = logsum_i - z_i,target(i)
//   G_iv = grad_loss_i (exp(z_iv - logsum_i) - [v = target(i)]),  dH = G W,  dW = G^T H
//
// Rows with a negative target take no part: the others are packed together first (ce_plan_kernel, ce_pack_kernel), so
// that neither their work nor what their hidden states hold reaches anything.
//
// Four matrix products carry the work: the logits (ce_gemm_kernel<CE_LOGSUM>, whose epilogue leaves a maximum and a
// sum for each row and 128 columns), and, for a piece of the vocabulary at a time, the logits again with G as the
// epilogue's result (CE_GRAD), G W (CE_HIDDEN) and G^T H (CE_WEIGHT).
//
// Times: 8192 rows of 4096 bf16 channels over 128000 tokens, 7373 of which take part (29 tiles): logits 5.8 ms (1.34 PFLOP/s of
// what the tiles take), and 5.9, 6.5 and 6.1 ms in four pieces for the gradients; 31 TFLOP in 23.4 ms, 1.33 PFLOP/s, with
// the power limit's clocks.  The logits are computed twice, a quarter of the work: kept for the backward pass they would take
// 2 bytes each (2.1 GB here), and rounded to 8 bits they would be off by more than the probabilities may be.
#include "float_types.cuh"
#include "tcgen05.cuh"
#include "warp_mma.cuh"

namespace lcpp {

bool make_tensor_map(CUtensorMap* map, bool bf16, const void* base, uint64_t inner, uint64_t rows, uint64_t planes,
                     uint64_t row_bytes, uint64_t plane_bytes, uint32_t box_rows) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            fn = nullptr;
        }
        return (Encode)fn;
    }();
    if (!encode) return false;
    const cuuint64_t dims[3] = {inner, rows, planes}, strides[2] = {row_bytes, plane_bytes};
    const cuuint32_t box[3] = {64, box_rows, 1}, step[3] = {1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
                  dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int CE_BM = 256, CE_BN = 256, CE_BK = 64;  // tile of a pair of CTAs, and its step along K
constexpr int CE_STAGES = 6;
constexpr int CE_HALF_BYTES = 128 * CE_BK * 2;       // one CTA's half of an operand's step
constexpr int CE_STAGE_BYTES = 2 * CE_HALF_BYTES;    // both operands
constexpr int CE_EPILOGUE_WARPS = 8;
constexpr int CE_THREADS = 64 + 32 * CE_EPILOGUE_WARPS;  // a loading warp, a warp that issues products, the epilogue
constexpr uint32_t CE_DRAIN_LIMIT = 1u << 14;  // polls of at most a microsecond that a CTA waits for its own copies in the end
constexpr float CE_LOG2E = 1.44269504088896f;
// G is kept for gradients of the loss as shares of the largest, which the sums are multiplied by in the end: for a mean's
// equal gradients the shares are 1, and an entry's rounding is that of the probability alone (-1 for an unlikely target is
// exact, where rounding 1 / rows would be off the same way in all rows).  float16 times 2^14, or small probabilities
// would vanish.
template <typename T>
constexpr float CE_GAIN = std::is_same_v<T, __half> ? 16384.0f : 1.0f;

enum { CE_LOGSUM, CE_GRAD, CE_HIDDEN, CE_WEIGHT };

// The next kernel may start; the one before has ended.
__device__ __forceinline__ void ce_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void ce_wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What the rows that take part are, in packed order; written by ce_plan_kernel.
struct CePlan {
    uint32_t* count;   // rows that take part
    float* largest;    // largest finite |grad_loss| of them
    int32_t* slot;     // of a row, or -1
    uint32_t* row;     // of a slot
    int32_t* target;
    float *logsum, *gain;
};

struct CeGemm {
    CePlan plan;
    const float *hidden_back, *weight_back;  // logits of float32: inverse scales by slot and token
    uint32_t vocab0, vocab;   // the piece [vocab0, vocab0 + vocab)
    uint32_t channels;
    uint32_t padded;          // rows of the packed buffers
    uint32_t splits;          // CE_HIDDEN: parts of K, each with its own sum
    uint32_t row0, row_end;   // CE_WEIGHT: the slots to sum over, of those that there are
    uint32_t add;             // add to what is there
    float2* part;             // CE_LOGSUM: (maximum, sum of exp(z - maximum)) by 128 columns and slot
    float* right;             // CE_LOGSUM: the targets' logits by slot
    void* grad;               // CE_GRAD: G (planes, padded, grad_stride)
    uint64_t grad_stride;
    float* sums;              // CE_HIDDEN: (splits, padded, sum_stride)
    uint64_t sum_stride;
    void* out;                // CE_WEIGHT: gradient of the weight
    uint64_t out_stride;
    uint32_t grad_wide, out_wide;  // bytes that the rows of G and out start on: 32, 16 or 1
};

struct CeBarriers {
    uint64_t full[CE_STAGES], empty[CE_STAGES], sum_full[2], sum_empty[2];
    uint32_t tmem;
};

// Float32 operands are sums of 16-bit planes.  Logits: two of float16, with a scale for each row, which leave 2^-23 of a
// value (2^-39 of its row's largest where that is more): 3 products (2^-22 is left out).  Gradients: three of bf16, 6 products to
// about 2^-24; G has probabilities of any size, and what a row of G or a column of it has in common is no scale of a sum
// over it.  With 6 products for the logits too, loss and gradients of 2048 x 512 x 32000 took 1352 us
// instead of 1160.
template <typename T, int EPI>
constexpr int CE_PAIRS = sizeof(T) == 2 ? 1 : EPI == CE_LOGSUM || EPI == CE_GRAD ? 3 : 6;
template <typename T, int EPI>
constexpr bool CE_BF16 = sizeof(T) == 4 ? CE_PAIRS<T, EPI> == 6 : !std::is_same_v<T, __half>;
// The planes of a's and b's i-th product, small products first.
template <int PAIRS>
__device__ __forceinline__ void ce_pair(uint32_t i, uint32_t* a, uint32_t* b) {
    if constexpr (PAIRS == 3) *a = i == 1, *b = i == 0;  // (0,1) (1,0) (0,0)
    else if constexpr (PAIRS == 6) *a = 0x010120 >> (4 * i) & 15, *b = 0x001102 >> (4 * i) & 15;  // (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
    else *a = *b = 0;
}

template <int EPI>
struct CeTiles {
    uint32_t m, n, parts, steps;  // tiles along M and N, parts of K, steps along the whole K (of one pair of planes)
    __device__ __forceinline__ CeTiles(const CeGemm& p, uint32_t count) : parts(1) {
        if constexpr (EPI == CE_LOGSUM || EPI == CE_GRAD) {
            m = (count + CE_BM - 1) / CE_BM, n = (p.vocab + CE_BN - 1) / CE_BN, steps = (p.channels + CE_BK - 1) / CE_BK;
        } else if constexpr (EPI == CE_HIDDEN) {
            m = (count + CE_BM - 1) / CE_BM, n = (p.channels + CE_BN - 1) / CE_BN, steps = (p.vocab + CE_BK - 1) / CE_BK;
            parts = p.splits;
        } else {
            m = (p.vocab + CE_BM - 1) / CE_BM, n = (p.channels + CE_BN - 1) / CE_BN;
            const uint32_t end = min(count, p.row_end);
            steps = end > p.row0 ? (end - p.row0 + CE_BK - 1) / CE_BK : 0;
        }
    }
    __device__ __forceinline__ uint64_t units() const { return (uint64_t)m * n * parts; }
    // Bands of 8 tiles along M, M fastest, part after part: the tiles under way share operands in L2 (a
    // tile's parts one after the other read 3.1 GB instead of 1.5 for 4096 x 2048 by 65536, of 0.8 that there are).
    __device__ __forceinline__ void at(uint64_t unit, uint32_t* mt, uint32_t* nt, uint32_t* first, uint32_t* end) const {
        const uint64_t tile = unit - (uint64_t)part(unit) * m * n;
        // 64-bit division takes a thread some hundred cycles
        const uint32_t band = tile >> 32 || n >> 29 ? (uint32_t)(tile / (8ull * n)) : (uint32_t)tile / (8 * n), height = min(8u, m - band * 8);
        const uint32_t in = (uint32_t)(tile - band * 8ull * n);
        *mt = band * 8 + in % height, *nt = in / height;
        range(part(unit), first, end);
    }
    __device__ __forceinline__ uint32_t part(uint64_t unit) const {
        if (parts == 1) return 0;
        return unit >> 32 ? (uint32_t)(unit / ((uint64_t)m * n)) : (uint32_t)unit / (m * n);  // m n < 2^28
    }
    // Steps along K of a part; parts <= CE_MAX_SPLITS and steps <= 2^24.
    __device__ __forceinline__ void range(uint32_t part, uint32_t* first, uint32_t* end) const {
        *first = steps * part / parts, *end = steps * (part + 1) / parts;
    }
};

template <typename T>
__device__ __forceinline__ uint32_t ce_pack2(float a, float b) {
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 v = __floats2half2_rn(a, b);
        return *(const uint32_t*)&v;
    } else {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *(const uint32_t*)&v;
    }
}
__device__ __forceinline__ float ce_exp2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// v = exp(v - shift): the difference is taken first, so that a row's largest logit gives exactly 1.
__device__ __forceinline__ void ce_exp32(float (&v)[32], float shift) {
    const uint64_t s = pair_of(shift, shift), by = pair_of(CE_LOG2E, CE_LOG2E);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        pair_split(pair_mul(pair_sub(pair_of(v[i], v[i + 1]), s), by), v[i], v[i + 1]);
        v[i] = ce_exp2(v[i]), v[i + 1] = ce_exp2(v[i + 1]);
    }
}

// 32 bytes, a whole sector, on a 32-byte boundary.
__device__ __forceinline__ void ce_store_sector(void* to, const uint32_t (&v)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7])
                 : "memory");
}
__device__ __forceinline__ void ce_load_sector(uint32_t (&v)[8], const void* from) {
    asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "l"(from)
                 : "memory");
}
// 32 values of a row, `width` of which exist; rows start on `wide` bytes.  A lane has a row of its own, so that a warp's
// store meets 32 rows: whole sectors are half the transactions of 16-byte stores.
template <typename T>
__device__ __forceinline__ void ce_store32(T* to, const float (&v)[32], uint32_t width, uint32_t wide) {
    if (wide >= 32 && width >= 32) {
        constexpr int E = 32 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 32 / E; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[i * E + j]);
                else w[j] = ce_pack2<T>(v[i * E + 2 * j], v[i * E + 2 * j + 1]);
            }
            ce_store_sector(to + i * E, w);
        }
    } else if (wide >= 16 && width >= 32) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 8; ++i) ((float4*)to)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                ((uint4*)to)[i] = make_uint4(ce_pack2<T>(v[8 * i], v[8 * i + 1]), ce_pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                                             ce_pack2<T>(v[8 * i + 4], v[8 * i + 5]), ce_pack2<T>(v[8 * i + 6], v[8 * i + 7]));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < width) to[i] = narrow<T>(v[i]);
    }
}

// v += the row's
__device__ __forceinline__ void ce_add32(float (&v)[32], const float* from, uint32_t width, uint32_t wide) {
    if (wide >= 32 && width >= 32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[8];
            ce_load_sector(w, from + i * 8);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i * 8 + j] += __uint_as_float(w[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < width) v[i] += from[i];
    }
}

// Logits of float32 out of their scales: the row's, and those of 32 tokens from `back` on.
template <typename T>
__device__ __forceinline__ void ce_unscale(float (&v)[32], float row, const float* back) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            const float4 b = *(const float4*)(back + i);
            v[i] *= row * b.x, v[i + 1] *= row * b.y, v[i + 2] *= row * b.z, v[i + 3] *= row * b.w;
        }
    }
}

// T: the element type of hidden states and weight.
template <typename T, int EPI>
__device__ __forceinline__ void ce_epilogue(const CeGemm& p, uint32_t tmem, uint32_t lane_row, uint32_t count, uint32_t mt,
                                            uint32_t nt, uint32_t half, bool empty, uint32_t part) {
    const uint32_t m = mt * CE_BM + lane_row;              // this thread's row of the tile
    const uint32_t n0 = nt * CE_BN + half * (CE_BN / 2);   // and its first column
    float v[32];
    if constexpr (EPI == CE_LOGSUM) {
        float top = -INFINITY, sum = 0.0f, right = 0.0f;
        const bool live = m < count;
        const int64_t target = live ? (int64_t)p.plan.target[m] - (int64_t)p.vocab0 - n0 : -1;
        const float back = sizeof(T) == 4 && live ? p.hidden_back[m] : 0.0f;
#pragma unroll 1
        for (int c = 0; c < CE_BN / 2; c += 32) {
            tmem_load32(tmem + c, v);
            ce_unscale<T>(v, back, p.weight_back + n0 + c);
            const int width = (int)p.vocab - (int)n0 - c;
            if (width < 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i >= width) v[i] = -INFINITY;
            }
            if (target >= c && target < c + 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (target == c + i) right = v[i];
            }
            float most = v[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) most = fmaxf(most, v[i]);
            const float base = fmaxf(top, most), shift = base == -INFINITY ? 0.0f : base;
            float s[4] = {0, 0, 0, 0};
            ce_exp32(v, shift);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[i & 3] += v[i];
            sum = sum * ce_exp2((top - shift) * CE_LOG2E) + ((s[0] + s[1]) + (s[2] + s[3]));
            top = base;
        }
        if (live) {
            p.part[(uint64_t)(nt * 2 + half) * p.padded + m] = make_float2(top, sum);
            if (target >= 0 && target < CE_BN / 2) p.right[m] = right;
        }
    } else if constexpr (EPI == CE_GRAD) {
        using E = std::conditional_t<std::is_same_v<T, __half>, __half, __nv_bfloat16>;
        const bool live = m < count;
        const int64_t target = live ? (int64_t)p.plan.target[m] - (int64_t)p.vocab0 - n0 : -1;
        const float logsum = live ? p.plan.logsum[m] : 0.0f;
        float gain = live ? p.plan.gain[m] : 0.0f;
        if (live && gain != 0.0f) gain = gain / *p.plan.largest * CE_GAIN<T>;
        const float back = sizeof(T) == 4 && live ? p.hidden_back[m] : 0.0f;
        E* const to = (E*)p.grad + (uint64_t)m * p.grad_stride + n0;
#pragma unroll 1
        for (int c = 0; c < CE_BN / 2; c += 32) {
            tmem_load32(tmem + c, v);
            const int width = (int)p.grad_stride - (int)n0 - c;
            if (width <= 0) break;
            ce_unscale<T>(v, back, p.weight_back + p.vocab0 + n0 + c);
            ce_exp32(v, logsum);
            if (target >= c && target < c + 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (target == c + i) v[i] -= 1.0f;
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = live ? v[i] * gain : 0.0f;
            const int real = (int)p.vocab - (int)n0 - c;
            if (real < 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (i >= real) v[i] = 0.0f;
            }
            if constexpr (sizeof(T) == 2) {
                ce_store32<E>(to + c, v, width, p.grad_wide);
            } else {  // three parts of 8 bits
#pragma unroll
                for (int plane = 0; plane < 3; ++plane) {
                    ce_store32<E>(to + plane * (uint64_t)p.padded * p.grad_stride + c, v, width, p.grad_wide);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] -= widen(narrow<E>(v[i]));
                }
            }
        }
    } else if constexpr (EPI == CE_HIDDEN) {
        float* const to = p.sums + ((uint64_t)part * p.padded + m) * p.sum_stride + n0;
#pragma unroll 1
        for (int c = 0; c < CE_BN / 2; c += 32) {
            tmem_load32(tmem + c, v);
            const int width = (int)p.sum_stride - (int)n0 - c;
            if (width <= 0) break;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = empty ? 0.0f : v[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (8 * i >= width) break;
                uint32_t w[8];
                if (p.add) {
                    ce_load_sector(w, to + c + 8 * i);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[8 * i + j] += __uint_as_float(w[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[8 * i + j]);
                ce_store_sector(to + c + 8 * i, w);
            }
        }
    } else {
        const bool live = m < p.vocab;
        const float unit = *p.plan.largest / CE_GAIN<T>;
        T* const to = (T*)p.out + (uint64_t)(p.vocab0 + m) * p.out_stride + n0;
#pragma unroll 1
        for (int c = 0; c < CE_BN / 2; c += 32) {
            tmem_load32(tmem + c, v);
            const int width = (int)p.channels - (int)n0 - c;
            if (width <= 0) break;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = empty ? 0.0f : v[i] * unit;
            if constexpr (sizeof(T) == 4) {
                if (p.add && live) ce_add32(v, to + c, width, p.out_wide);
            }
            if (live) ce_store32<T>(to + c, v, width, p.out_wide);
        }
    }
}

// Bound by the tensor cores: 4096 rows (3686 that take part) x 2048 x 65536 bf16, tensor pipe 95 % of the cycles for the logits and for G, 94 % for
// G^T H, 87 % for G W with its 1.7 waves of tiles and parts; DRAM 11 to 20 % (G W 30 %), L2 50 %.  Long runs of it meet the power limit,
// so that bytes not moved are time too.  2 CTAs a tile halve what shared memory and L2 pass on for the same products.
// One pair of CTAs makes tiles of 256 x 256: each CTA holds 128 rows of A and 128 rows of B (as K-major) and has 128
// rows of the sum in its tensor memory, twice, so that the epilogue of a tile runs under the next one's products.
template <typename T, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(CE_THREADS, 1)
ce_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
               const __grid_constant__ CeGemm p) {
    constexpr bool A_MN = EPI == CE_WEIGHT, B_MN = EPI == CE_HIDDEN || EPI == CE_WEIGHT;
    constexpr uint32_t PAIRS = CE_PAIRS<T, EPI>;
    extern __shared__ uint8_t ce_smem[];
    __shared__ CeBarriers bar;
    const uint32_t tiles = (smem_u32(ce_smem) + 1023) & ~1023u;  // swizzled boxes start on 1024 bytes
    const uint32_t warp = threadIdx.x >> 5, rank = cluster_rank();
    const uint32_t limit = g_spin_limit;  // polls of at most a microsecond
    if (warp == 0 && elect_one()) {
        tma_prefetch_map(&map_a);
        tma_prefetch_map(&map_b);
        for (int i = 0; i < CE_STAGES; ++i) mbar_init(&bar.full[i], 1), mbar_init(&bar.empty[i], 1);
        for (int i = 0; i < 2; ++i) mbar_init(&bar.sum_full[i], 1), mbar_init(&bar.sum_empty[i], 2 * CE_EPILOGUE_WARPS);
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&bar.tmem, 512);
    tmem_fence_before();
    __syncthreads();
    cluster_sync();
    tmem_fence_after();
    const uint32_t tmem = bar.tmem;
    ce_let_next_start();
    ce_wait_for_last();
    const uint32_t count = *p.plan.count;
    const CeTiles<EPI> tl(p, count);
    const uint32_t groups = gridDim.x / 2, group = blockIdx.x / 2;
    bool ok = true;

    if (warp == 0) {
        if (elect_one()) {
            uint32_t it = 0;  // steps so far
            for (uint64_t unit = group; ok && unit < tl.units(); unit += groups) {
                uint32_t mt, nt, first, end;
                tl.at(unit, &mt, &nt, &first, &end);
                for (uint32_t pair = 0; ok && pair < PAIRS; ++pair) {
                    uint32_t pa, pb;
                    ce_pair<PAIRS>(pair, &pa, &pb);
                    for (uint32_t k = first; k < end; ++k, ++it) {
                        const uint32_t s = it % CE_STAGES;
                        if (it >= CE_STAGES && !mbar_poll(&bar.empty[s], (it / CE_STAGES - 1) & 1, limit)) {
                            ok = false;
                            break;
                        }
                        const uint32_t a = tiles + s * CE_STAGE_BYTES, b = a + CE_HALF_BYTES;
                        if (rank == 0) mbar_arrive_expect_tx(&bar.full[s], 2 * CE_STAGE_BYTES);
                        const uint32_t full = cluster_smem(smem_u32(&bar.full[s]), 0);
                        const int m0 = mt * CE_BM + rank * 128, n0 = nt * CE_BN + rank * 128, k0 = k * CE_BK;
                        if constexpr (A_MN) {
                            tma_load_3d(&map_a, a, full, m0, p.row0 + k0, pa);
                            tma_load_3d(&map_a, a + CE_HALF_BYTES / 2, full, m0 + 64, p.row0 + k0, pa);
                        } else {
                            tma_load_3d(&map_a, a, full, k0, m0, pa);
                        }
                        if constexpr (B_MN) {
                            const int y = k0 + (EPI == CE_HIDDEN ? p.vocab0 : p.row0);
                            tma_load_3d(&map_b, b, full, n0, y, pb);
                            tma_load_3d(&map_b, b + CE_HALF_BYTES / 2, full, n0 + 64, y, pb);
                        } else {
                            tma_load_3d(&map_b, b, full, k0, p.vocab0 + n0, pb);
                        }
                    }
                }
            }
            // Every copy has landed before the CTA may leave: its stage was read.  Stages that nothing reads any more, since a
            // wait gave up, are waited for as long as a copy can take.
            for (uint32_t back = 0; back < CE_STAGES && back < it; ++back) {
                const uint32_t last = it - 1 - back;
                if (!mbar_poll(&bar.empty[last % CE_STAGES], (last / CE_STAGES) & 1, CE_DRAIN_LIMIT)) break;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            constexpr uint32_t instruction = mma_instruction(CE_BF16<T, EPI>, A_MN, B_MN, CE_BM, CE_BN);
            constexpr uint32_t lead_a = A_MN ? CE_HALF_BYTES / 2 : 16, lead_b = B_MN ? CE_HALF_BYTES / 2 : 16;
            constexpr uint32_t step_a = A_MN ? 2048 : 32, step_b = B_MN ? 2048 : 32;  // bytes of 16 along K
            uint32_t it = 0, sums = 0;
            for (uint64_t unit = group; ok && unit < tl.units(); unit += groups, ++sums) {
                uint32_t first, end;
                tl.range(tl.part(unit), &first, &end);
                const uint32_t d = sums & 1;
                if (sums >= 2 && !mbar_poll(&bar.sum_empty[d], (sums / 2 - 1) & 1, limit)) {
                    ok = false;
                    break;
                }
                tmem_fence_after();
                const uint32_t steps = (end - first) * PAIRS;
                for (uint32_t k = 0; k < steps; ++k, ++it) {
                    const uint32_t s = it % CE_STAGES;
                    if (!mbar_poll(&bar.full[s], (it / CE_STAGES) & 1, limit)) {
                        ok = false;
                        break;
                    }
                    tmem_fence_after();
                    const uint32_t a = tiles + s * CE_STAGE_BYTES, b = a + CE_HALF_BYTES;
#pragma unroll
                    for (uint32_t i = 0; i < CE_BK / 16; ++i)
                        mma_f16_pair(tmem + d * CE_BN, mma_descriptor(a + i * step_a, lead_a, 1024),
                                     mma_descriptor(b + i * step_b, lead_b, 1024), instruction, k || i);
                    mma_commit_pair(&bar.empty[s]);
                }
                if (ok) mma_commit_pair(&bar.sum_full[d]);
            }
            // and so have the products' last arrivals, also where the epilogue does not wait for them any more
            if (sums) mbar_poll(&bar.sum_full[(sums - 1) & 1], ((sums - 1) / 2) & 1, CE_DRAIN_LIMIT);
        }
        __syncwarp();
    } else {
        const uint32_t quarter = warp & 3, half = (warp - 2) >> 2;  // a warp reaches the lanes of its number modulo 4
        uint32_t sums = 0;
        for (uint64_t unit = group; unit < tl.units(); unit += groups, ++sums) {
            uint32_t mt, nt, first, end;
            tl.at(unit, &mt, &nt, &first, &end);
            const uint32_t d = sums & 1;
            ok = __all_sync(0xffffffffu, mbar_poll(&bar.sum_full[d], (sums / 2) & 1, limit));
            if (!ok) break;
            tmem_fence_after();
            ce_epilogue<T, EPI>(p, tmem + d * CE_BN + half * (CE_BN / 2) + (quarter * 32 << 16),
                                rank * 128 + quarter * 32 + (threadIdx.x & 31), count, mt, nt, half, first == end,
                                tl.part(unit));
            tmem_fence_before();
            __syncwarp();
            if (elect_one()) mbar_arrive_cluster(cluster_smem(smem_u32(&bar.sum_empty[d]), 0));
        }
    }
    if (!ok) set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
    tmem_fence_before();
    __syncthreads();
    cluster_sync();
    tmem_fence_after();
    if (warp == 1) tmem_free(tmem, 512);
}

// ---- before and after the products ------------------------------------------------------------------
constexpr int CE_PLAN_THREADS = 1024;
// One CTA: which rows take part, in order, with their targets, gradients and sums.
__global__ void __launch_bounds__(CE_PLAN_THREADS)
ce_plan_kernel(const int32_t* targets, const float* grad_loss, uint64_t grad_stride, const float* logsum, uint32_t rows,
               uint32_t vocab, CePlan plan) {
    __shared__ uint32_t sums[32];
    __shared__ float tops[32];
    ce_let_next_start();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t base = 0;
    float most = 0.0f;
    for (uint64_t r0 = 0; r0 < rows; r0 += CE_PLAN_THREADS * 4) {  // 128 rows a warp
        int32_t t[4];
        uint32_t ballot[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t r = r0 + warp * 128 + i * 32 + lane;
            t[i] = r < rows ? targets[r] : -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (t[i] >= 0 && (uint32_t)t[i] >= vocab) {
                set_error(LCPP_ERR_INVALID_ARG);
                t[i] = -1;
            }
            ballot[i] = __ballot_sync(0xffffffffu, t[i] >= 0);
            mine += __popc(ballot[i]);
        }
        if (lane == 0) sums[warp] = mine;
        __syncthreads();
        uint32_t before = base, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < 32; ++w) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t r = r0 + warp * 128 + i * 32 + lane;
            if (r < rows) {
                const uint32_t slot = before + __popc(ballot[i] & lanemask_lt());
                plan.slot[r] = t[i] >= 0 ? (int32_t)slot : -1;
                if (t[i] >= 0) {
                    plan.row[slot] = (uint32_t)r;
                    plan.target[slot] = t[i];
                    if (grad_loss) {
                        const float g = grad_loss[r * grad_stride];
                        plan.gain[slot] = g;
                        plan.logsum[slot] = logsum[r];
                        if (fabsf(g) < INFINITY) most = fmaxf(most, fabsf(g));
                    }
                }
            }
            before += __popc(ballot[i]);
        }
        base += all;
        __syncthreads();
    }
    most = warp_reduce<OpMax>(most);
    if (lane == 0) tops[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) most = fmaxf(most, tops[w]);
        *plan.count = base;
        *plan.largest = most;
    }
}

// Elements [8 w, 8 w + 8) of a row; zeros from `channels` on.  wide: rows start on 16 bytes.
template <typename T>
__device__ __forceinline__ void ce_load8(T (&v)[8], const T* source, bool wide, uint32_t w, uint32_t channels) {
    if (wide && w * 8 + 8 <= channels) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(v) / 16; ++i) ((uint4*)v)[i] = ((const uint4*)(source + w * 8))[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = w * 8 + i < channels ? source[w * 8 + i] : narrow<T>(0.0f);
    }
}

// Rows of 16-bit elements on 16-byte boundaries; to row s from row[s] (null: s), zeros from row `count` on up to the next
// multiple of 256.  A warp a row.
template <typename T>
__global__ void __launch_bounds__(256)
ce_pack_kernel(const T* from, uint64_t from_stride, const uint32_t* row, const uint32_t* count, uint32_t rows,
               uint32_t channels, void* to, uint64_t to_stride) {
    ce_let_next_start();
    ce_wait_for_last();
    const uint32_t have = count ? *count : rows, last = count ? (have + CE_BM - 1) / CE_BM * CE_BM : rows;
    const uint32_t words = (uint32_t)(to_stride / 8);
    const bool wide = ((uintptr_t)from | from_stride * sizeof(T)) % 16 == 0;
    const uint32_t lane = threadIdx.x & 31;
    for (uint64_t r = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < last; r += (uint64_t)gridDim.x * 8) {
        const T* const source = r < have ? from + (row ? row[r] : r) * from_stride : nullptr;
        uint4* const out = (uint4*)((T*)to + r * to_stride);
        auto copy = [&](uint32_t w) {
            alignas(16) T v[8] = {};
            if (source) ce_load8(v, source, wide, w, channels);
            out[w] = *(const uint4*)v;
        };
        if (wide || !source) {
#pragma unroll 4
            for (uint32_t w = lane; w < words; w += 32) copy(w);
            continue;
        }
        // Pieces with neighbours on both sides: put together from the two on 16 bytes that they lie in, four at a time.
        const uint32_t end = max(channels / 8, 2u) - 1;  // 8 end + 8 <= channels; from 1 on
        const uint32_t phase = (uint32_t)(uintptr_t)source & 15, shift = phase & 2 ? 16 : 0;
        const uint4* const pieces = (const uint4*)((uintptr_t)source & ~(uintptr_t)15);
        for (uint32_t w0 = 1 + lane; w0 < end; w0 += 128) {
            uint4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (w0 + i * 32 < end) a[i] = pieces[w0 + i * 32], b[i] = pieces[w0 + i * 32 + 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t x[8] = {a[i].x, a[i].y, a[i].z, a[i].w, b[i].x, b[i].y, b[i].z, b[i].w};
                uint32_t v[4];
#pragma unroll
                for (uint32_t first = 0; first < 4; ++first) {
                    if (phase >> 2 != first) continue;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = __funnelshift_r(x[first + j], x[first + j + 1], shift);
                }
                if (w0 + i * 32 < end) out[w0 + i * 32] = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
        if (lane == 0) copy(0);
        for (uint32_t w = end + lane; w < words; w += 32) copy(w);
    }
}

// Float32 rows, likewise: as two planes of float16 by a power of two that brings the row's largest finite value to 2^14 ..
// 2^15, whose inverse goes to back[], and (null: not) as three planes of bf16.
struct CeSplit {
    const float* from;
    uint64_t from_stride;
    const uint32_t *row, *count;
    uint32_t rows, channels;
    __half* halves;
    __nv_bfloat16* parts;
    float* back;
    uint64_t to_stride, plane;
};
__global__ void __launch_bounds__(256) ce_split_kernel(const CeSplit p) {
    ce_let_next_start();
    ce_wait_for_last();
    const uint32_t have = p.count ? *p.count : p.rows, last = p.count ? (have + CE_BM - 1) / CE_BM * CE_BM : p.rows;
    const uint32_t words = (uint32_t)(p.to_stride / 8), lane = threadIdx.x & 31;
    const bool wide = ((uintptr_t)p.from | p.from_stride * 4) % 16 == 0;
    for (uint64_t r = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); r < last; r += (uint64_t)gridDim.x * 8) {
        const float* const source = r < have ? p.from + (p.row ? p.row[r] : r) * p.from_stride : nullptr;
        float most = 0.0f;
        if (source) {
#pragma unroll 4
            for (uint32_t w = lane; w < words; w += 32) {
                alignas(16) float v[8];
                ce_load8(v, source, wide, w, p.channels);
#pragma unroll
                for (int i = 0; i < 8; ++i) most = fabsf(v[i]) < INFINITY ? fmaxf(most, fabsf(v[i])) : most;
            }
        }
        const Scale scale = scale_for<120>(warp_max(most));
        if (lane == 0) p.back[r] = scale.back;
#pragma unroll 2
        for (uint32_t w = lane; w < words; w += 32) {
            alignas(16) float v[8] = {};
            if (source) ce_load8(v, source, wide, w, p.channels);
            alignas(16) uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_f16(v[2 * i], v[2 * i + 1], scale.by, hi[i], lo[i]);
            const uint64_t at = r * p.to_stride + w * 8;
            *(uint4*)(p.halves + at) = *(const uint4*)hi, *(uint4*)(p.halves + p.plane + at) = *(const uint4*)lo;
            if (!p.parts) continue;
#pragma unroll
            for (int plane = 0; plane < 3; ++plane) {
                alignas(16) __nv_bfloat16 e[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = narrow<__nv_bfloat16>(v[i]), v[i] -= widen(e[i]);
                *(uint4*)(p.parts + plane * p.plane + at) = *(const uint4*)e;
            }
        }
    }
}

// 32 rows a CTA, its warps over the parts of the vocabulary: logsum and loss.
constexpr int CE_LOSS_WARPS = 32;
__global__ void __launch_bounds__(CE_LOSS_WARPS * 32)
ce_loss_kernel(const float2* part, uint32_t parts, const float* right, CePlan plan, uint32_t rows, uint32_t padded, float* loss,
               float* logsum) {
    __shared__ float2 joined[CE_LOSS_WARPS][32];
    ce_let_next_start();
    ce_wait_for_last();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t r = (uint64_t)blockIdx.x * 32 + lane;
    const int32_t slot = r < rows ? plan.slot[r] : -1;
    float top = -INFINITY, sum = 0.0f;
    auto join = [&](float2 v) {
        const float base = fmaxf(top, v.x), shift = base == -INFINITY ? 0.0f : base;
        sum = sum * ce_exp2((top - shift) * CE_LOG2E) + v.y * ce_exp2((v.x - shift) * CE_LOG2E);
        top = base;
    };
    if (slot >= 0) {
        uint32_t i = warp;
        for (; i + 3 * CE_LOSS_WARPS < parts; i += 4 * CE_LOSS_WARPS) {
            float2 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = part[(uint64_t)(i + j * CE_LOSS_WARPS) * padded + slot];
#pragma unroll
            for (int j = 0; j < 4; ++j) join(v[j]);
        }
        for (; i < parts; i += CE_LOSS_WARPS) join(part[(uint64_t)i * padded + slot]);
    }
    joined[warp][lane] = make_float2(top, sum);
    __syncthreads();
    if (warp == 0 && r < rows) {
        for (int w = 1; w < CE_LOSS_WARPS; ++w) join(joined[w][lane]);
        const float rest = logf(sum);  // sum >= 1, right <= top: the loss is never negative
        if (loss) loss[r] = slot >= 0 ? (top - right[slot]) + rest : 0.0f;
        if (logsum) logsum[r] = slot >= 0 ? top + rest : 0.0f;
    }
}

// Gradient of the hidden states: the parts' sums together, rounded; zeros for rows that took no part.
template <typename T>
__global__ void __launch_bounds__(256)
ce_hidden_kernel(const float* sums, uint64_t stride, uint32_t padded, uint32_t splits, CePlan plan, uint32_t rows,
                 uint32_t channels, T* out, uint64_t out_stride, bool wide) {
    ce_let_next_start();
    ce_wait_for_last();
    const float unit = *plan.largest / CE_GAIN<T>;
    for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const int32_t slot = plan.slot[r];
        T* const to = out + r * out_stride;
        for (uint32_t c = threadIdx.x * 4; c < channels; c += blockDim.x * 4) {
            float4 v = make_float4(0, 0, 0, 0);
            if (slot >= 0)
                for (uint32_t s = 0; s < splits; ++s) {
                    const float4 a = *(const float4*)(sums + ((uint64_t)s * padded + slot) * stride + c);
                    v.x += a.x, v.y += a.y, v.z += a.z, v.w += a.w;
                }
            v.x *= unit, v.y *= unit, v.z *= unit, v.w *= unit;
            if (wide && c + 4 <= channels) {
                if constexpr (sizeof(T) == 4) *(float4*)(to + c) = v;
                else *(uint2*)(to + c) = make_uint2(ce_pack2<T>(v.x, v.y), ce_pack2<T>(v.z, v.w));
            } else {
                const float e[4] = {v.x, v.y, v.z, v.w};
                for (int i = 0; i < 4; ++i)
                    if (c + i < channels) to[c + i] = narrow<T>(e[i]);
            }
        }
    }
}

// ---- host ------------------------------------------------------------------------------------
constexpr uint64_t CE_MAX_ROWS = 1ull << 24, CE_MAX_CHANNELS = 1ull << 20, CE_MAX_VOCAB = 1ull << 30;
constexpr uint64_t CE_PIECE_BYTES = 512ull << 20;  // of G
// The tensor cores' sums are cut off, not rounded, at every step: they come out too small by about 1.2e-9 of themselves a
// term.  Beside the roundings of 16-bit gradients that is nothing, but float32 ones take this many terms a sum at most, and
// add the sums in float32 (weight gradient of 16384 rows in one sum: error 1.9e-5, so 4.8e-6).
constexpr uint64_t CE_EXACT_TERMS = 4096, CE_MAX_SPLITS = 64;
static_assert(CE_EXACT_TERMS % CE_BK == 0, "splits are whole steps");

// The pieces of the temp buffer.
struct CeLayout {
    uint64_t planes, padded, pitch;       // planes of G, and of operands for gradients; packed rows; elements of a packed row
    uint64_t parts, piece, splits, sum_pitch;
    size_t count, slot, row, target, logsum, gain, right, hidden, weight, part, grad, sums, bytes;
    size_t hidden_halves, weight_halves, hidden_back, weight_back;  // float32: what the logits are made of
    CeLayout(int dtype, uint64_t rows, uint64_t channels, uint64_t vocab, bool backward, bool pack_weight) {
        planes = dtype == LCPP_F32 ? 3 : 1;
        padded = align_up(rows, CE_BM);
        pitch = align_up(channels, 8);
        parts = ceil_div(vocab, CE_BN) * 2;
        sum_pitch = align_up(channels, 8);
        uint64_t widest = max(CE_PIECE_BYTES / (planes * padded * 2) / CE_BN * CE_BN, (uint64_t)CE_BN);
        if (planes > 1) widest = min(widest, CE_MAX_SPLITS * CE_EXACT_TERMS);
        const uint64_t pieces = ceil_div(vocab, widest);
        piece = min(align_up(ceil_div(vocab, pieces), CE_BN), align_up(vocab, 16));  // rows of G on 32 bytes
        splits = best_splits(padded, channels, piece, planes);
        size_t at = 0;
        auto take = [&](uint64_t n) {
            const size_t here = at;
            at += align_up(n, 256);
            return here;
        };
        count = take(8), slot = take(rows * 4), row = take(padded * 4), target = take(padded * 4);
        logsum = take(padded * 4), gain = take(padded * 4);
        hidden = weight = hidden_halves = weight_halves = hidden_back = weight_back = 0;
        if (planes == 1 || backward) {
            hidden = take(planes * padded * pitch * 2);
            weight = pack_weight ? take(planes * vocab * pitch * 2) : 0;
        }
        if (planes > 1) {
            hidden_halves = take(2 * padded * pitch * 2), weight_halves = take(2 * vocab * pitch * 2);
            hidden_back = take(padded * 4), weight_back = take(align_up(vocab, CE_BN) * 4);  // read by whole tiles
        }
        right = part = grad = sums = 0;
        if (backward) {
            grad = take(planes * padded * piece * 2);
            sums = take(splits * padded * sum_pitch * 4);
        } else {
            right = take(padded * 4);
            part = take(parts * padded * 8);
        }
        bytes = at;
    }
    // Parts of the hidden gradient's sum over the vocabulary: the number with the least time, of whole waves of tiles (a step
    // of 64 takes 0.33 us) and of the parts' sums (float32, written and read once a piece).
    static uint64_t best_splits(uint64_t padded, uint64_t channels, uint64_t piece, uint64_t planes) {
        const uint64_t pairs = device_info().sms / 2, tiles = padded / CE_BM * ceil_div(channels, CE_BN), steps = ceil_div(piece, CE_BK);
        const uint64_t fewest = planes == 1 ? 1 : ceil_div(piece, CE_EXACT_TERMS);
        uint64_t best = fewest;
        double least = 0;
        for (uint64_t n = fewest; n <= max(fewest, (uint64_t)32) && (n == fewest || n * 16 <= steps); ++n) {
            const double time = (double)ceil_div(tiles * n, pairs) * ceil_div(steps, n) * 0.33 + (double)n * padded * channels * 8 / 6e6;
            if (n == fewest || time < least) best = n, least = time;
        }
        return best;
    }
    CePlan plan(void* temp) const {
        char* const t = (char*)temp;
        return CePlan{(uint32_t*)(t + count), (float*)(t + count) + 1, (int32_t*)(t + slot), (uint32_t*)(t + row),
                      (int32_t*)(t + target), (float*)(t + logsum), (float*)(t + gain)};
    }
};

static bool ce_direct(int dtype, const void* p, uint64_t stride) {  // the tensor memory accelerator can read its rows
    return dtype != LCPP_F32 && (uintptr_t)p % 16 == 0 && stride % 8 == 0;
}

// What a call is given, checked.
struct CeCall {
    int dtype;
    const void *hidden, *weight;
    uint64_t hidden_stride, weight_stride;
    const int32_t* targets;
    uint64_t rows, channels, vocab;
    void* temp;
    cudaStream_t stream;
    uint64_t element() const { return dtype == LCPP_F32 ? 4 : 2; }
    Region r_hidden() const { return Region(hidden, rows, hidden_stride * element(), channels * element()); }
    Region r_weight() const { return Region(weight, vocab, weight_stride * element(), channels * element()); }
    lcpp_status check() const {
        auto stride_ok = [&](uint64_t stride, uint64_t n) { return n <= 1 || (stride >= channels && stride < (1ull << 31)); };
        if (!is_float_dtype(dtype) || rows > CE_MAX_ROWS || channels > CE_MAX_CHANNELS || vocab > CE_MAX_VOCAB || !vocab ||
            !channels)
            return LCPP_ERR_INVALID_ARG;
        if (!rows) return LCPP_OK;
        if (!hidden || !weight || !targets || !stride_ok(hidden_stride, rows) || !stride_ok(weight_stride, vocab))
            return LCPP_ERR_INVALID_ARG;
        if (!elements_aligned(dtype, hidden, weight) || !elements_aligned(LCPP_F32, targets)) return LCPP_ERR_INVALID_ARG;
        return LCPP_OK;
    }
};

// A call's kernels but the first start while the one before ends (programmatic dependent launch): each lets the next
// one in when it starts itself, and waits for the end of the one before ahead of its first access to memory.
template <typename... P, typename... A>
static lcpp_status ce_launch(const char* name, void (*kernel)(P...), uint64_t grid, unsigned threads, size_t smem, bool first, cudaStream_t s,
                             const A&... args) {
    cudaLaunchAttribute how[1];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = how;
    if (!first) {
        how[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        how[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    }
    ProfScope prof(name, s);
    if (cudaLaunchKernelEx(&cfg, kernel, P(args)...) != cudaSuccess) return check_launch();
    count_launch();
    return LCPP_OK;
}

template <typename T, int EPI>
static lcpp_status ce_gemm(const char* name, const CUtensorMap& a, const CUtensorMap& b, const CeGemm& p, uint64_t units,
                           cudaStream_t s) {
    constexpr size_t smem = CE_STAGES * CE_STAGE_BYTES + 1024;
    const DeviceInfo device = device_info();
    static std::atomic<uint64_t> sized{0};  // devices on which the kernel may have this much shared memory
    const uint64_t bit = 1ull << device.device;
    if (!(sized.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(ce_gemm_kernel<T, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return check_launch();
        sized.fetch_or(bit, std::memory_order_relaxed);
    }
    const uint64_t pairs = min(units, (uint64_t)device.sms / 2);
    return ce_launch(name, ce_gemm_kernel<T, EPI>, pairs * 2, CE_THREADS, smem, false, s, a, b, p);
}

struct CeMaps {
    CUtensorMap hidden_k, hidden_n, weight_k, weight_n, grad_k, grad_m;
};

// Plans and packs; then the operands' tensor maps.
template <typename T>
static lcpp_status ce_begin(const CeCall& c, const CeLayout& l, const float* grad_loss, uint64_t grad_stride,
                            const float* logsum, CeMaps* maps) {
    const CePlan plan = l.plan(c.temp);
    char* const t = (char*)c.temp;
    lcpp_status ok = ce_launch("ce_plan", ce_plan_kernel, 1, CE_PLAN_THREADS, 0, true, c.stream, c.targets, grad_loss, grad_stride,
                               logsum, (uint32_t)c.rows, (uint32_t)c.vocab, plan);
    if (ok != LCPP_OK) return ok;
    const uint64_t most = (uint64_t)device_info().sms * 16, hidden_grid = min(ceil_div(l.padded, 8), most), weight_grid = min(ceil_div(c.vocab, 8), most);
    const uint32_t rows = (uint32_t)c.rows, channels = (uint32_t)c.channels, vocab = (uint32_t)c.vocab;
    const void* weight = l.weight ? t + l.weight : c.weight;
    const uint64_t weight_pitch = l.weight || c.vocab == 1 ? l.pitch : c.weight_stride;
    if constexpr (sizeof(T) == 4) {
        const CeSplit hidden{(const float*)c.hidden, c.hidden_stride, plan.row, plan.count, rows, channels, (__half*)(t + l.hidden_halves),
                             (__nv_bfloat16*)(l.hidden ? t + l.hidden : nullptr), (float*)(t + l.hidden_back), l.pitch, l.padded * l.pitch};
        ok = ce_launch("ce_pack", ce_split_kernel, hidden_grid, 256, 0, false, c.stream, hidden);
        if (ok != LCPP_OK) return ok;
        const CeSplit tokens{(const float*)c.weight, c.weight_stride, nullptr, nullptr, vocab, channels, (__half*)(t + l.weight_halves),
                             (__nv_bfloat16*)(l.weight ? t + l.weight : nullptr), (float*)(t + l.weight_back), l.pitch, c.vocab * l.pitch};
        ok = ce_launch("ce_pack", ce_split_kernel, weight_grid, 256, 0, false, c.stream, tokens);
    } else {
        ok = ce_launch("ce_pack", ce_pack_kernel<T>, hidden_grid, 256, 0, false, c.stream, (const T*)c.hidden, c.hidden_stride, plan.row,
                       plan.count, rows, channels, t + l.hidden, l.pitch);
        if (ok == LCPP_OK && l.weight)
            ok = ce_launch("ce_pack", ce_pack_kernel<T>, weight_grid, 256, 0, false, c.stream, (const T*)c.weight, c.weight_stride, nullptr, nullptr,
                           vocab, channels, t + l.weight, l.pitch);
    }
    if (ok != LCPP_OK) return ok;
    auto map = [&](CUtensorMap* m, bool bf16, uint64_t planes, const void* base, uint64_t inner, uint64_t rows, uint64_t pitch, uint32_t box) {
        return make_tensor_map(m, bf16, base, inner, rows, planes, pitch * 2, (planes > 1 ? rows : 1) * pitch * 2, box);
    };
    constexpr bool FINE = sizeof(T) == 4, LOGITS_BF16 = CE_BF16<T, CE_LOGSUM>, GRAD_BF16 = CE_BF16<T, CE_HIDDEN>;
    if (!map(&maps->hidden_k, LOGITS_BF16, FINE ? 2 : 1, t + (FINE ? l.hidden_halves : l.hidden), c.channels, l.padded, l.pitch, 128) ||
        !map(&maps->weight_k, LOGITS_BF16, FINE ? 2 : 1, FINE ? t + l.weight_halves : weight, c.channels, c.vocab, FINE ? l.pitch : weight_pitch, 128))
        return LCPP_ERR_CUDA;
    if (l.grad && (!map(&maps->hidden_n, GRAD_BF16, l.planes, t + l.hidden, c.channels, l.padded, l.pitch, 64) ||
                   !map(&maps->weight_n, GRAD_BF16, l.planes, weight, c.channels, c.vocab, weight_pitch, 64) ||
                   !map(&maps->grad_k, GRAD_BF16, l.planes, t + l.grad, l.piece, l.padded, l.piece, 128) ||
                   !map(&maps->grad_m, GRAD_BF16, l.planes, t + l.grad, l.piece, l.padded, l.piece, 64)))
        return LCPP_ERR_CUDA;
    return LCPP_OK;
}

}  // namespace lcpp

using namespace lcpp;

extern "C" size_t lcpp_cross_entropy_temp_bytes(int dtype, uint64_t rows, uint64_t channels, uint64_t vocab, int backward,
                                                int aligned) {
    if (!is_float_dtype(dtype) || rows > CE_MAX_ROWS || channels > CE_MAX_CHANNELS || vocab > CE_MAX_VOCAB) return 0;
    if (!rows || !channels || !vocab) return 256;
    // with gradients the loss's own buffer may be wanted too
    const bool pack = dtype == LCPP_F32 || !aligned || channels % 8;
    size_t most = CeLayout(dtype, rows, channels, vocab, false, pack).bytes;
    if (!backward) return most;
    // Fewer rows may want more, with larger pieces of G or more splits: the buffer serves any number up to this one.
    most = max(most, CeLayout(dtype, rows, channels, vocab, true, pack).bytes);
    for (uint64_t fewer = CE_BM; fewer < rows; fewer += CE_BM) most = max(most, CeLayout(dtype, fewer, channels, vocab, true, pack).bytes);
    return most;
}

extern "C" lcpp_status lcpp_cross_entropy_forward(int dtype, const void* hidden, uint64_t hidden_stride, const void* weight,
                                                  uint64_t weight_stride, const int32_t* targets, float* loss, float* logsum,
                                                  uint64_t rows, uint64_t channels, uint64_t vocab, void* temp,
                                                  size_t temp_bytes, void* stream) {
    const CeCall c{dtype, hidden, weight, hidden_stride, weight_stride, targets, rows, channels, vocab, temp, (cudaStream_t)stream};
    const lcpp_status ok = c.check();
    if (ok != LCPP_OK || !rows) return ok;
    if ((!loss && !logsum) || !elements_aligned(LCPP_F32, loss, logsum)) return LCPP_ERR_INVALID_ARG;
    const CeLayout l(dtype, rows, channels, vocab, false, !ce_direct(dtype, weight, vocab > 1 ? weight_stride : 0));
    if (!temp || temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % 32) return LCPP_ERR_INVALID_ARG;
    const Region rh = c.r_hidden(), rw = c.r_weight(), rg(targets, rows * 4), rl(loss, rows * 4), rs(logsum, rows * 4),
                 rt(temp, l.bytes);
    if (!rl.apart(rh, rw, rg, rs, rt) || !rs.apart(rh, rw, rg, rt) || !rt.apart(rh, rw, rg)) return LCPP_ERR_INVALID_ARG;
    return dispatch_float(dtype, [&](auto type) -> lcpp_status {
        using T = decltype(type);
        CeMaps maps;
        lcpp_status ok = ce_begin<T>(c, l, nullptr, 0, nullptr, &maps);
        if (ok != LCPP_OK) return ok;
        CeGemm p{};
        p.plan = l.plan(temp);
        p.hidden_back = (const float*)((char*)temp + l.hidden_back), p.weight_back = (const float*)((char*)temp + l.weight_back);
        p.vocab = (uint32_t)vocab, p.channels = (uint32_t)channels;
        p.padded = (uint32_t)l.padded, p.splits = 1;
        p.part = (float2*)((char*)temp + l.part), p.right = (float*)((char*)temp + l.right);
        ok = ce_gemm<T, CE_LOGSUM>("ce_logsum", maps.hidden_k, maps.weight_k, p, l.padded / CE_BM * ceil_div(vocab, CE_BN), c.stream);
        if (ok != LCPP_OK) return ok;
        return ce_launch("ce_loss", ce_loss_kernel, ceil_div(rows, 32), CE_LOSS_WARPS * 32, 0, false, c.stream, (const float2*)p.part, (uint32_t)l.parts,
                         (const float*)p.right, p.plan, (uint32_t)rows, (uint32_t)l.padded, loss, logsum);
    });
}

extern "C" lcpp_status lcpp_cross_entropy_backward(int dtype, const void* hidden, uint64_t hidden_stride, const void* weight,
                                                   uint64_t weight_stride, const int32_t* targets, const float* logsum,
                                                   const float* grad_loss, uint64_t grad_loss_stride, void* grad_hidden,
                                                   uint64_t grad_hidden_stride, void* grad_weight,
                                                   uint64_t grad_weight_stride, uint64_t rows, uint64_t channels,
                                                   uint64_t vocab, void* temp, size_t temp_bytes, void* stream) {
    const CeCall c{dtype, hidden, weight, hidden_stride, weight_stride, targets, rows, channels, vocab, temp, (cudaStream_t)stream};
    const lcpp_status ok = c.check();
    if (ok != LCPP_OK) return ok;
    auto stride_ok = [&](uint64_t stride, uint64_t n) { return n <= 1 || (stride >= channels && stride < (1ull << 31)); };
    if ((grad_hidden && !stride_ok(grad_hidden_stride, rows)) || (grad_weight && !stride_ok(grad_weight_stride, vocab)) ||
        !elements_aligned(dtype, grad_hidden, grad_weight) || !elements_aligned(LCPP_F32, logsum, grad_loss))
        return LCPP_ERR_INVALID_ARG;
    if (!rows) {  // the weight's gradient is a sum over no rows
        if (!grad_weight) return LCPP_OK;
        const uint64_t e = c.element();
        return cudaMemset2DAsync(grad_weight, (vocab > 1 ? grad_weight_stride : channels) * e, 0, channels * e, vocab,
                                 c.stream) == cudaSuccess ? LCPP_OK : check_launch();
    }
    if (!logsum || !grad_loss || (!grad_hidden && !grad_weight) || (grad_loss_stride > 1 && rows > 1 && grad_loss_stride >= 1ull << 31))
        return LCPP_ERR_INVALID_ARG;
    const CeLayout l(dtype, rows, channels, vocab, true, !ce_direct(dtype, weight, vocab > 1 ? weight_stride : 0));
    if (!temp || temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % 32) return LCPP_ERR_INVALID_ARG;
    const uint64_t e = c.element();
    const Region rh = c.r_hidden(), rw = c.r_weight(), rg(targets, rows * 4), rs(logsum, rows * 4),
                 rl(grad_loss, grad_loss_stride ? rows : 1, grad_loss_stride * 4, 4), rt(temp, l.bytes),
                 rgh(grad_hidden, rows, grad_hidden_stride * e, channels * e),
                 rgw(grad_weight, vocab, grad_weight_stride * e, channels * e);
    if (!rgh.apart(rh, rw, rg, rs, rl, rt, rgw) || !rgw.apart(rh, rw, rg, rs, rl, rt) || !rt.apart(rh, rw, rg, rs, rl))
        return LCPP_ERR_INVALID_ARG;
    return dispatch_float(dtype, [&](auto type) -> lcpp_status {
        using T = decltype(type);
        CeMaps maps;
        lcpp_status ok = ce_begin<T>(c, l, grad_loss, grad_loss_stride, logsum, &maps);
        if (ok != LCPP_OK) return ok;
        CeGemm p{};
        p.plan = l.plan(temp);
        p.hidden_back = (const float*)((char*)temp + l.hidden_back), p.weight_back = (const float*)((char*)temp + l.weight_back);
        p.channels = (uint32_t)channels;
        p.padded = (uint32_t)l.padded, p.splits = (uint32_t)l.splits;
        p.grad = (char*)temp + l.grad, p.grad_stride = l.piece, p.grad_wide = 32;
        p.sums = (float*)((char*)temp + l.sums), p.sum_stride = l.sum_pitch;
        p.out = grad_weight, p.out_stride = grad_weight_stride;
        const uintptr_t starts = (uintptr_t)grad_weight | (vocab > 1 ? grad_weight_stride * sizeof(T) : 0);
        p.out_wide = starts % 32 == 0 ? 32 : starts % 16 == 0 ? 16 : 1;
        const uint64_t mt = l.padded / CE_BM, dt = ceil_div(channels, CE_BN);
        for (uint64_t v0 = 0; v0 < vocab; v0 += l.piece) {
            p.vocab0 = (uint32_t)v0, p.vocab = (uint32_t)min(l.piece, vocab - v0), p.add = v0 > 0;
            p.row0 = 0;
            ok = ce_gemm<T, CE_GRAD>("ce_grad", maps.hidden_k, maps.weight_k, p, mt * ceil_div(p.vocab, CE_BN), c.stream);
            if (ok != LCPP_OK) return ok;
            if (grad_hidden) ok = ce_gemm<T, CE_HIDDEN>("ce_hidden", maps.grad_k, maps.weight_n, p, mt * dt * l.splits, c.stream);
            if (ok != LCPP_OK) return ok;
            const uint64_t part = sizeof(T) == 4 ? CE_EXACT_TERMS : l.padded;  // rows
            for (uint64_t row = 0; grad_weight && ok == LCPP_OK && row < rows; row += part) {
                p.row0 = (uint32_t)row, p.row_end = (uint32_t)(row + part), p.add = row > 0;
                ok = ce_gemm<T, CE_WEIGHT>("ce_weight", maps.grad_m, maps.hidden_n, p, ceil_div(p.vocab, CE_BM) * dt, c.stream);
            }
            if (ok != LCPP_OK) return ok;
        }
        if (!grad_hidden) return LCPP_OK;
        const bool wide = ((uintptr_t)grad_hidden | (rows > 1 ? grad_hidden_stride * sizeof(T) : 0)) % 16 == 0;
        return ce_launch("ce_hidden_out", ce_hidden_kernel<T>, min(rows, (uint64_t)device_info().sms * 16), 256, 0, false, c.stream,
                         (const float*)p.sums, l.sum_pitch, (uint32_t)l.padded, (uint32_t)l.splits, p.plan, (uint32_t)rows,
                         (uint32_t)channels, (T*)grad_hidden, grad_hidden_stride, wide);
    });
}
