// Beam search (DeviceBeamSearch): selection over beams and vocabulary, and the
// reordering of per-beam states.
//
// Selection, for each batch entry with K beams over V tokens:
//   logp(k, v) = (z - m) - log(sum_v exp(z - m)),  m = max_v z
//   beam k offers its K best tokens (z descending, equal z: token ascending)
//   with score(k) + logp; a finished beam offers one candidate, (eos, score(k));
//   the K best candidates of all beams (score descending, equal scores: beam,
//   then place in the beam's list ascending) are the new beams.
// A logit of -inf (or NaN) and a score of -inf (or NaN) offer nothing; a new
// beam that nothing fills has score -inf, token max(eos, 0), its own row as
// parent and is finished.  Where m = +inf, its tokens share the probability.
#include <algorithm>
#include "float_types.cuh"

namespace lcpp {

constexpr int BEAM_MAX = 32;       // beams
constexpr int BEAM_THREADS = 256;

// uint32 with the order of float32 values: NaN as -inf, the two zeros alike.
__device__ __forceinline__ uint32_t ordered(float v) {
    v = v != v ? -INFINITY : v + 0.0f;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// ---- Sorted lists across a warp, largest first ---------------------------------
template <typename K>
__device__ __forceinline__ K warp_keep(K a, int xor_lane, bool larger) {
    const K b = __shfl_xor_sync(0xffffffffu, a, xor_lane);
    return (a < b) == larger ? b : a;
}
template <typename K>
__device__ __forceinline__ K warp_sort(K a) {  // bitonic
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) a = warp_keep(a, j, ((lane & j) == 0) == ((lane & k) == 0));
    return a;
}
// The 32 largest of two sorted lists, sorted.
template <typename K>
__device__ __forceinline__ K warp_merge(K a, K b) {
    const int lane = threadIdx.x & 31;
    const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a < r ? r : a;
#pragma unroll
    for (int j = 16; j; j >>= 1) a = warp_keep(a, j, (lane & j) == 0);
    return a;
}
// The 32 largest of n keys, sorted (0 where there are fewer).
__device__ __forceinline__ uint64_t warp_top(const uint64_t* keys, int n) {
    const int lane = threadIdx.x & 31;
    uint64_t top = warp_sort(lane < n ? keys[lane] : 0);
    for (int i = 32; i < n; i += 32) top = warp_merge(top, warp_sort(i + lane < n ? keys[i + lane] : 0));
    return top;
}

// The 32 largest of `lists` sorted lists of n <= 32 keys one behind the other: list by list where they are long, else
// all keys sorted.
__device__ __forceinline__ uint64_t warp_top_lists(const uint64_t* keys, int lists, int n) {
    const int lane = threadIdx.x & 31;
    if (lists > 1 && n < 8) return warp_top(keys, lists * n);
    uint64_t top = lane < n ? keys[lane] : 0;
    for (int i = 1; i < lists; ++i) top = warp_merge(top, lane < n ? keys[i * n + lane] : 0);
    return top;
}

// ---- One part of one row ---------------------------------------------------------
// A CTA reads its part of a row once: each thread takes vectors of 16 bytes,
// BEAM_VECS of them a chunk, and keeps the sum of 2^(z log2(e) - K) with a whole
// number K, so that a larger maximum rescales the sum exactly, and the largest
// value of each chunk.  The beams-th largest of the threads' maxima is at most
// the beams-th best logit of the part: only the few chunks that reach it are read
// again (from L2), and what reaches it there is sorted.  The streaming loop thus
// spends nothing on the selection but a maximum (half an instruction a 2-byte
// element).  512 rows of 100003 f32: 42.6 us on one B200 (4.8 TB/s, 73 % of the
// copy rate), the rest being the end of each CTA, which all reach at about the
// same time; 131072 bf16 41 us (4.5 instructions an element).
constexpr int BEAM_VECS = 4;
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_VECS;  // vectors of a tile of a part
constexpr int BEAM_TILES = 32;                       // tiles of a part at most
constexpr int BEAM_KEYS = 1024;                      // logits that may reach the threads' bound

// Results of one part: its `beams` best keys (ordered logit << 32 | ~token, 0: none), largest logit, and the sum of
// exp(z - largest).
struct BeamTemp {
    uint64_t* key;   // [rows][parts][beams]
    float2* total;   // [rows][parts]
};

// 16 bytes of a row.
template <typename T>
struct BeamVector {
    static constexpr int E = 16 / sizeof(T);
    uint4 w;
    // The vector at address `at`, of which elements [lo, hi) belong to the row; the others read as -inf.
    __device__ __forceinline__ void load(const T* at, int64_t lo, int64_t hi) {
        T t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = e >= lo && e < hi ? at[e] : narrow<T>(-INFINITY);
        memcpy(&w, t, 16);
    }
    // The largest element that is not NaN (-inf if there is none).
    __device__ __forceinline__ float max() const {
        if constexpr (sizeof(T) == 4) {
            return fmaxf(fmaxf(get(0), get(1)), fmaxf(fmaxf(get(2), get(3)), -INFINITY));
        } else {
            using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
            T2 v[4];
            memcpy(v, &w, 16);
            const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
            return fmaxf(fmaxf(widen(m.x), widen(m.y)), -INFINITY);
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
            return __uint_as_float(v[e]);
        } else {
            const uint32_t v[4] = {w.x, w.y, w.z, w.w};
            if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                return __uint_as_float(e % 2 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
            } else {
                __half2 h;
                memcpy(&h, &v[e / 2], 4);
                return e % 2 ? __high2float(h) : __low2float(h);
            }
        }
    }
};

constexpr float BEAM_LOG2E = 1.44269504f;
__device__ __forceinline__ float beam_ex2(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// A row takes part if its beam has a score and is not finished.
__device__ __forceinline__ bool beam_live(const float* scores, const uint8_t* finished, uint64_t row) {
    const float score = scores[row];  // both are asked for before either is looked at
    const uint8_t done = finished ? finished[row] : 0;
    return score > -INFINITY && !done;
}

struct BeamRow {
    int beams;
    uint32_t vocab, part, parts;
};

template <typename T>
struct BeamPartSmem {
    float chunk[BEAM_TILES][BEAM_THREADS];
    uint64_t key[BEAM_KEYS];
    float top[BEAM_THREADS / 32][32], scale[BEAM_THREADS / 32], sum[BEAM_THREADS / 32];
    int count;
};

// Part p.part of the row z: the calling CTA's first warp returns its `beams` best keys, a lane each, and all threads
// (largest, total).  live(): whether the row takes part at all; if not, there are no keys and (-inf, 0).
template <typename T, typename Live>
__device__ __forceinline__ uint64_t beam_part(const T* z, const BeamRow& p, BeamPartSmem<T>& sm, float2* out, Live live) {
    constexpr int E = BeamVector<T>::E, WARPS = BEAM_THREADS / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int shift = (int)(((uintptr_t)z & 15) / sizeof(T));  // elements between the first vector's address and z
    const T* base = z - shift;
    const uint32_t end = shift + p.vocab, vectors = (end + E - 1) / E;  // vocab < 2^31
    const uint32_t tiles = (vectors + BEAM_TILE - 1) / BEAM_TILE;
    const uint32_t tile0 = (uint32_t)((uint64_t)tiles * p.part / p.parts);
    const uint32_t tile1 = (uint32_t)((uint64_t)tiles * (p.part + 1) / p.parts);
    const int n = (int)(tile1 - tile0);
    using Chunk = BeamVector<T>[BEAM_VECS];
    auto load = [&](Chunk& v, uint32_t tile) {
        const uint32_t at0 = tile * BEAM_TILE + tid;
        if ((tile > 0 || shift == 0) && (tile + 1) * BEAM_TILE <= end / E) {  // all inside the row
            const uint4* src = (const uint4*)base + at0;
#pragma unroll
            for (int q = 0; q < BEAM_VECS; ++q) v[q].w = ld_stream(src + q * BEAM_THREADS);
        } else {
#pragma unroll
            for (int q = 0; q < BEAM_VECS; ++q) {
                const uint32_t at = at0 + q * BEAM_THREADS;
                const int64_t first = (int64_t)at * E;  // element of the vectors' count
                if (at < vectors) v[q].load(base + first, shift - first, (int64_t)end - first);
                else v[q].load(base, E, 0);
            }
        }
    };
    if (tid == 0) sm.count = 0;
    float top = -INFINITY, scale = -1e30f, sum = 0.0f;  // sum of 2^(z log2e - scale)
    auto add = [&](const Chunk& v, int j) {
        float m = v[0].max();
#pragma unroll
        for (int q = 1; q < BEAM_VECS; ++q) m = fmaxf(m, v[q].max());
        sm.chunk[j][tid] = m;
        top = fmaxf(top, m);
        const float k = ceilf(m * BEAM_LOG2E);
        if (k > scale) {
            sum *= beam_ex2(scale - k);
            scale = k;
        }
#pragma unroll
        for (int q = 0; q < BEAM_VECS; ++q) {
            float part_sum = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) part_sum += beam_ex2(fmaf(v[q].get(e), BEAM_LOG2E, -scale));
            sum += part_sum;
        }
    };
    Chunk v, ahead;
    if (!live()) {
        *out = make_float2(-INFINITY, 0.0f);
        return 0;
    }
    if (n > 0) load(v, tile0);
    for (int j = 0; j < n; j += 2) {
        if (j + 1 < n) load(ahead, tile0 + j + 1);
        add(v, j);
        if (j + 1 < n) {
            if (j + 2 < n) load(v, tile0 + j + 2);
            add(ahead, j + 1);
        }
    }
    // ---- the part's maximum and sum, and the beams-th largest of the threads' maxima ----
    float sorted = warp_sort(top);
    sm.top[warp][lane] = sorted;
    float warp_scale = scale;
    for (int o = 16; o; o >>= 1) warp_scale = fmaxf(warp_scale, __shfl_xor_sync(0xffffffffu, warp_scale, o));
    float warp_sum = sum * beam_ex2(scale - warp_scale);
    for (int o = 16; o; o >>= 1) warp_sum += __shfl_xor_sync(0xffffffffu, warp_sum, o);
    if (lane == 0) sm.scale[warp] = warp_scale, sm.sum[warp] = warp_sum;
    for (int half = WARPS / 2; half; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            sorted = warp_merge(sorted, sm.top[warp + half][lane]);
            sm.top[warp][lane] = sorted;
        }
    }
    __syncthreads();
    const float largest = sm.top[0][0], bound = sm.top[0][p.beams - 1];
    // ---- what reaches the bound ------------------------------------------------------
    if (top >= bound && top > -INFINITY) {
        for (int j = 0; j < n; ++j) {
            const float m = sm.chunk[j][tid];
            if (!(m >= bound && m > -INFINITY)) continue;
            if (n > 2) {
                load(v, tile0 + j);
            } else if (j == 1) {  // both are still here, the first in v
#pragma unroll
                for (int q = 0; q < BEAM_VECS; ++q) v[q] = ahead[q];
            }
#pragma unroll
            for (int q = 0; q < BEAM_VECS; ++q)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float x = v[q].get(e);
                    if (x >= bound && x > -INFINITY) {
                        const int at = atomicAdd(&sm.count, 1);
                        const uint32_t token = ((tile0 + j) * BEAM_TILE + q * BEAM_THREADS + tid) * E + e - shift;
                        if (at < BEAM_KEYS) sm.key[at] = (uint64_t)ordered(x) << 32 | (uint32_t)~token;
                    }
                }
        }
    }
    __syncthreads();
    const uint32_t first = max((int64_t)tile0 * BEAM_TILE * E - shift, (int64_t)0);
    const uint32_t stop = min((int64_t)tile1 * BEAM_TILE * E - shift, (int64_t)p.vocab);
    uint64_t mine = 0;
    if (sm.count <= BEAM_KEYS) {
        if (warp == 0) mine = warp_top(sm.key, sm.count);
    } else {  // many equal logits: the best below the last one found, `beams` times over
        uint64_t below = ~0ull;
        for (int j = 0; j < p.beams; ++j) {
            uint64_t best = 0;
            for (uint32_t t = first + tid; t < stop; t += BEAM_THREADS) {
                const float x = widen(z[t]);
                const uint64_t key = (uint64_t)ordered(x) << 32 | (uint32_t)~t;
                if (x >= bound && x > -INFINITY && key < below && key > best) best = key;
            }
            for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            __syncthreads();
            if (lane == 0) sm.key[warp] = best;
            __syncthreads();
            for (int w = 0; w < WARPS; ++w) best = max(best, sm.key[w]);
            below = best;
            if (tid == j) mine = best;
        }
    }
    float all_scale = sm.scale[0], total = 0.0f;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) all_scale = fmaxf(all_scale, sm.scale[w]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) total += sm.sum[w] * beam_ex2(sm.scale[w] - all_scale);
    // relative to the largest term, which went through the same product
    total /= beam_ex2(fmaf(largest, BEAM_LOG2E, -all_scale));
    if (!(total >= 0.5f && total < INFINITY) && largest > -INFINITY) {
        // NaN among the logits, a maximum of +inf, or one whose scaled value is out of range: term by term
        total = 0.0f;
        for (uint32_t t = first + tid; t < stop; t += BEAM_THREADS) {
            const float x = fmaxf(widen(z[t]), -INFINITY);
            total += x == largest ? 1.0f : __expf(x - largest);
        }
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        __syncthreads();
        if (lane == 0) sm.sum[warp] = total;
        __syncthreads();
        total = 0.0f;
        for (int w = 0; w < WARPS; ++w) total += sm.sum[w];
    }
    *out = make_float2(largest, total);
    return mine;
}

// ---- One batch entry ----------------------------------------------------------------
// A warp a beam joins the parts of its row; then the first warp takes the best
// of all beams' candidates.  key: [beam][part][beams], total: [beam][part].
struct BeamOut {
    float* scores;
    int32_t *tokens, *parents;
    uint8_t* finished;
};
struct BeamMergeSmem {
    uint64_t top[BEAM_THREADS / 32][32];
    float score[BEAM_MAX * BEAM_MAX];
    int32_t token[BEAM_MAX * BEAM_MAX];
};

__device__ __forceinline__ void beam_merge(const uint64_t* key, const float2* total, uint64_t first, const float* scores,
                                           const uint8_t* finished, int beams, uint32_t parts, int eos,
                                           const BeamOut& out, BeamMergeSmem& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    uint64_t top = 0;  // the best candidates of this warp's beams
    for (int k = warp; k < beams; k += warps) {
        const uint64_t row = first + k;
        const float score = scores[row];
        float best = -INFINITY;
        int32_t token = max(eos, 0);
        if (beam_live(scores, finished, row)) {
            const uint64_t mine = warp_top_lists(key + (uint64_t)k * parts * beams, (int)parts, beams);
            float largest = -INFINITY, sum = 0.0f;
            for (uint32_t i = lane; i < parts; i += 32) largest = fmaxf(largest, total[(uint64_t)k * parts + i].x);
            for (int o = 16; o; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            for (uint32_t i = lane; i < parts; i += 32) {
                const float2 t = total[(uint64_t)k * parts + i];
                if (t.x > -INFINITY) sum += t.x == largest ? t.y : t.y * __expf(t.x - largest);
            }
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (mine) {
                const float z = unordered((uint32_t)(mine >> 32));
                best = score + ((z == largest ? 0.0f : z - largest) - logf(sum));
                token = (int32_t)~(uint32_t)mine;
            }
        } else if (lane == 0 && score > -INFINITY) {
            best = score;  // finished: it stays
        }
        // a beam's candidates are in order: larger scores first, equal ones by place
        const int at = k * beams + lane;
        uint64_t list = 0;
        if (lane < beams) {
            sm.score[at] = best, sm.token[at] = token;
            if (best > -INFINITY) list = (uint64_t)ordered(best) << 32 | (uint32_t)~at;
        }
        top = k == warp ? list : warp_merge(top, list);
    }
    sm.top[warp][lane] = top;
    int half = 1;
    while (2 * half < min(warps, beams)) half *= 2;
    for (; half && beams > 1; half >>= 1) {
        __syncthreads();
        if (warp < half && warp + half < warps) {
            top = warp_merge(top, sm.top[warp + half][lane]);
            sm.top[warp][lane] = top;
        }
    }
    __syncthreads();
    if (warp == 0 && lane < beams) {
        const uint32_t at = ~(uint32_t)top;
        const bool any = top != 0;
        const uint64_t parent = any ? first + at / beams : first + lane;
        const int32_t token = any ? sm.token[at] : max(eos, 0);
        out.scores[first + lane] = any ? sm.score[at] : -INFINITY;
        out.tokens[first + lane] = token;
        out.parents[first + lane] = (int32_t)parent;
        if (out.finished) out.finished[first + lane] = !any || (finished && finished[parent]) || token == eos;
    }
}

// Two kernels: parts of all rows, joined through `tmp`.
template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4)
beam_rows_kernel(const T* logits, uint64_t stride, const float* scores, const uint8_t* finished, int beams,
                 uint32_t vocab, uint32_t parts, BeamTemp tmp) {
    __shared__ BeamPartSmem<T> sm;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint64_t row = blockIdx.x / parts;
    const uint32_t part = blockIdx.x - (uint32_t)row * parts;
    float2 total;
    const uint64_t key = beam_part(logits + row * stride, BeamRow{beams, vocab, part, parts}, sm, &total,
                                   [&] { return beam_live(scores, finished, row); });
    if (threadIdx.x < beams) tmp.key[(row * parts + part) * beams + threadIdx.x] = key;
    if (threadIdx.x == 0) tmp.total[row * parts + part] = total;
}
__global__ void __launch_bounds__(256)
beam_merge_kernel(BeamTemp tmp, const float* scores, const uint8_t* finished, int beams, uint32_t parts, int eos, BeamOut out) {
    __shared__ BeamMergeSmem sm;
    const uint64_t first = (uint64_t)blockIdx.x * beams;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    beam_merge(tmp.key + first * parts * beams, tmp.total + first * parts, first, scores, finished, beams, parts, eos, out, sm);
}

// One kernel: a cluster takes a batch entry, a CTA a part of one of its rows; the first CTA joins them from its
// shared memory.  For short rows, where a second launch and the way through L2 are what counts, and for batches whose
// CTAs fill the SMs by themselves.
constexpr int BEAM_CLUSTER = 8;

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4)
beam_cluster_kernel(const T* logits, uint64_t stride, const float* scores, const uint8_t* finished, int beams,
                    uint32_t vocab, uint32_t parts, int eos, BeamOut out) {
    __shared__ union {
        BeamPartSmem<T> part;
        BeamMergeSmem merge;
    } sm;
    __shared__ uint64_t s_key[BEAM_CLUSTER * BEAM_CLUSTER];
    __shared__ float2 s_total[BEAM_CLUSTER];
    asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    const uint32_t size = beams * parts, rank = blockIdx.x % size, part = rank % parts;
    const uint64_t first = (uint64_t)(blockIdx.x / size) * beams, row = first + rank / parts;
    float2 total;
    const uint64_t key = beam_part(logits + row * stride, BeamRow{beams, vocab, part, parts}, sm.part, &total,
                                   [&] { return beam_live(scores, finished, row); });
    asm volatile("barrier.cluster.wait;" ::: "memory");  // the first CTA has started
    uint32_t key_at, total_at;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(key_at) : "r"((uint32_t)__cvta_generic_to_shared(s_key)));
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(total_at) : "r"((uint32_t)__cvta_generic_to_shared(s_total)));
    if (threadIdx.x < beams)
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(key_at + (rank * beams + threadIdx.x) * 8), "l"(key) : "memory");
    if (threadIdx.x == 0)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(total_at + rank * 8), "f"(total.x), "f"(total.y) : "memory");
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (rank == 0) beam_merge(s_key, s_total, first, scores, finished, beams, parts, eos, out, sm.merge);
}

// ---- Reordering ------------------------------------------------------------------------
// out[l][i] = in[l][parents[i]], rows of bytes; a negative parent: zeros.  A warp
// copies BEAM_COPY vectors a lane of one row, all loads before the first store
// (268 MB of f32 states in 69 us, 7.8 TB/s of bytes asked for: repeated parents
// come from L2).
// V: 16- or 4-byte vectors where everything is a whole number of them, else
// (V = 1) 4-byte words of out put together from the two words of in they lie
// in, with single bytes at the row's ends.
constexpr int BEAM_COPY = 4;
constexpr int BEAM_COPY_WARPS = 4;

template <int V>
__global__ void __launch_bounds__(BEAM_COPY_WARPS * 32)
beam_reorder_kernel(const char* in, uint64_t in_layer, uint64_t in_row, char* out, uint64_t out_layer, uint64_t out_row,
                    const int32_t* parents, uint32_t rows_in, uint32_t rows, uint64_t row_bytes, uint64_t units,
                    uint32_t parts) {
    using Word = std::conditional_t<V == 16, uint4, uint32_t>;
    constexpr int B = sizeof(Word), U = V == 16 ? BEAM_COPY : 2 * BEAM_COPY;
    const uint64_t unit = (uint64_t)blockIdx.x * BEAM_COPY_WARPS + (threadIdx.x >> 5);
    if (unit >= units) return;
    const int lane = threadIdx.x & 31;
    const uint32_t line = (uint32_t)(unit / parts), part = (uint32_t)(unit - (uint64_t)line * parts);
    const uint32_t l = line / rows, i = line - l * rows;
    int64_t from = parents[i];
    if (from >= (int64_t)rows_in) {
        set_error(LCPP_ERR_INVALID_ARG);
        from = -1;
    }
    const char* src = in + l * in_layer + from * in_row;
    char* dst = out + l * out_layer + i * out_row;
    const uint64_t words = row_bytes / B, w0 = (uint64_t)part * (32 * U) + lane;
    Word v[U];
    if constexpr (V > 1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            v[u] = Word{};
            if (from >= 0 && w0 + u * 32 < words) v[u] = ((const Word*)src)[w0 + u * 32];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (w0 + u * 32 < words) ((Word*)dst)[w0 + u * 32] = v[u];
    } else {
        // words of dst from its first word boundary on; both words of in around one hold bytes of the row, except
        // at its ends, where the word is put together from bytes
        const uint64_t head = min((uint64_t)(-(uintptr_t)dst & 3), row_bytes), body = (row_bytes - head) / 4;
        const char* s = src + head;
        const int off = (int)((uintptr_t)s & 3);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t w = w0 + u * 32;
            v[u] = 0;
            if (from >= 0 && w < body) {
                const char* at = s + w * 4;
                if (off == 0) {
                    v[u] = *(const uint32_t*)at;
                } else if (at - off >= src && at - off + 8 <= src + row_bytes) {
                    const uint32_t* q = (const uint32_t*)(at - off);
                    v[u] = __funnelshift_r(q[0], q[1], off * 8);
                } else {
                    for (int b = 0; b < 4; ++b) v[u] |= (uint32_t)(uint8_t)at[b] << 8 * b;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (w0 + u * 32 < body) ((uint32_t*)(dst + head))[w0 + u * 32] = v[u];
        if (part == 0) {  // fewer than 8 bytes at the ends
            const uint64_t rest = row_bytes - head - body * 4;
            if (lane < (int)head) dst[lane] = from >= 0 ? src[lane] : 0;
            const uint64_t e = head + body * 4 + lane;
            if (lane < (int)rest) dst[e] = from >= 0 ? src[e] : 0;
        }
    }
}

// Parts of a row: whole tiles, at least as many as keep a part within BEAM_TILES of them, and as many more as give
// every SM BEAM_PARTS_PER_SM parts.
constexpr int BEAM_PARTS_PER_SM = 3;
constexpr int BEAM_SHORT = 4;
static uint64_t beam_tiles(uint64_t vocab, size_t element) {  // at any alignment
    const uint64_t per_vector = 16 / element;
    return ceil_div(ceil_div(vocab + per_vector - 1, per_vector), BEAM_TILE);
}
static uint32_t beam_parts(uint64_t rows, uint64_t vocab, size_t element, uint64_t sms) {
    const uint64_t tiles = beam_tiles(vocab, element);
    const uint64_t least = ceil_div(tiles, BEAM_TILES);
    const uint64_t wanted = ceil_div(sms * BEAM_PARTS_PER_SM, rows ? rows : 1);
    return (uint32_t)std::max(least, std::min(wanted, tiles));
}
static size_t beam_temp_bytes(uint64_t rows, uint64_t beams, uint64_t parts) {
    return align_up(rows * parts * beams * 8, 256) + align_up(rows * parts * 8, 256);
}

}  // namespace lcpp

using namespace lcpp;

extern "C" size_t lcpp_beam_select_temp_bytes(uint64_t batches, uint32_t beams, uint64_t vocab) {
    if (beams < 1 || beams > BEAM_MAX || vocab < 1) return 0;
    const uint64_t rows = batches * beams;
    const uint64_t sms = device_info().sms;  // float32 has the most parts
    return beam_temp_bytes(rows, beams, beam_parts(rows, vocab, 4, sms));
}

extern "C" lcpp_status lcpp_beam_select(int dtype, const void* logits, uint64_t logits_stride, const float* scores_in,
                                        const uint8_t* finished_in, float* scores_out, int32_t* tokens_out,
                                        int32_t* parents_out, uint8_t* finished_out, uint64_t batches, uint32_t beams,
                                        uint64_t vocab, int32_t eos_token, void* temp, size_t temp_bytes, void* stream) {
    if (!is_float_dtype(dtype) || beams < 1 || beams > BEAM_MAX || vocab < 1 || vocab > 0x7fffffffull ||
        batches > 0x7fffffffull / beams || (eos_token >= 0 && (uint64_t)eos_token >= vocab))
        return LCPP_ERR_INVALID_ARG;
    if (!batches) return LCPP_OK;
    if (!logits || !scores_in || !scores_out || !tokens_out || !parents_out) return LCPP_ERR_INVALID_ARG;
    if (batches * beams > 1 && (logits_stride < vocab || logits_stride > 0x7fffffffull)) return LCPP_ERR_INVALID_ARG;
    if (!temp || temp_bytes < lcpp_beam_select_temp_bytes(batches, beams, vocab)) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % sizeof(uint64_t)) return LCPP_ERR_INVALID_ARG;
    const uint64_t rows = batches * beams;
    if (!elements_aligned(dtype, logits) || !elements_aligned(LCPP_F32, scores_in, scores_out, tokens_out, parents_out))
        return LCPP_ERR_INVALID_ARG;
    // outputs are written while inputs of the same entry may still be read
    const uint64_t e = dtype == LCPP_F32 ? 4 : 2;
    const Region rz(logits, rows, logits_stride * e, vocab * e), rs(scores_in, rows * 4), rf(finished_in, rows),
        so(scores_out, rows * 4), to(tokens_out, rows * 4), po(parents_out, rows * 4), fo(finished_out, rows),
        rt(temp, lcpp_beam_select_temp_bytes(batches, beams, vocab));
    if (!so.apart(rz, rs, rf, to, po, fo, rt) || !to.apart(rz, rs, rf, po, fo, rt) || !po.apart(rz, rs, rf, fo, rt) ||
        !fo.apart(rz, rs, rf, rt) || !rt.apart(rz, rs, rf))
        return LCPP_ERR_INVALID_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    return dispatch_float(dtype, [&](auto t) -> lcpp_status {
        using T = decltype(t);
        const BeamOut out{scores_out, tokens_out, parents_out, finished_out};
        const uint64_t sms = device_info().sms;
        uint32_t parts = beam_parts(rows, vocab, sizeof(T), sms);
        if (rows * parts > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
        // A cluster an entry, where that fills the SMs or leaves a CTA little to read.
        const uint32_t split = BEAM_CLUSTER / beams;
        const uint64_t tiles = beam_tiles(vocab, sizeof(T)), span = split ? ceil_div(tiles, std::min(split, parts)) : ~0ull;
        if (span <= BEAM_SHORT || (span <= BEAM_TILES && rows * std::min(split, parts) >= 2 * sms)) {
            parts = std::min(split, parts);
            cudaLaunchAttribute cluster{};
            cluster.id = cudaLaunchAttributeClusterDimension;
            cluster.val.clusterDim.x = beams * parts;
            cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3((unsigned)(rows * parts));
            cfg.blockDim = dim3(BEAM_THREADS);
            cfg.stream = s;
            cfg.attrs = &cluster;
            cfg.numAttrs = 1;
            ProfScope prof("beam_cluster", s);
            if (cudaLaunchKernelEx(&cfg, beam_cluster_kernel<T>, (const T*)logits, logits_stride, scores_in, finished_in,
                                   (int)beams, (uint32_t)vocab, parts, (int)eos_token, out) != cudaSuccess)
                return check_launch();
            count_launch();
            return check_launch();
        }
        const BeamTemp tmp{(uint64_t*)temp, (float2*)((char*)temp + align_up(rows * parts * beams * 8, 256))};
        {
            ProfScope prof("beam_rows", s);
            beam_rows_kernel<T><<<(unsigned)(rows * parts), BEAM_THREADS, 0, s>>>(
                (const T*)logits, logits_stride, scores_in, finished_in, (int)beams, (uint32_t)vocab, parts, tmp);
        }
        ProfScope prof("beam_merge", s);
        // launched while the rows are under way; it waits for them itself
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned)batches);
        cfg.blockDim = dim3(beams > 1 ? 256 : 32);
        cfg.stream = s;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        if (cudaLaunchKernelEx(&cfg, beam_merge_kernel, tmp, scores_in, finished_in, (int)beams, parts, (int)eos_token,
                               out) != cudaSuccess)
            return check_launch();
        count_launch(2);
        return check_launch();
    });
}

extern "C" lcpp_status lcpp_beam_reorder(const void* in, uint64_t in_layer_bytes, uint64_t in_row_bytes, void* out,
                                         uint64_t out_layer_bytes, uint64_t out_row_bytes, const int32_t* parents,
                                         uint64_t layers, uint64_t rows_in, uint64_t rows, uint64_t row_bytes,
                                         void* stream) {
    if (rows > 0x7fffffffull || rows_in > 0x7fffffffull || layers > 0x7fffffffull || row_bytes > (1ull << 40))
        return LCPP_ERR_INVALID_ARG;
    if (!rows || !layers || !row_bytes) return LCPP_OK;
    if ((!in && rows_in) || !out || !parents || rows * layers > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    if ((rows_in > 1 && in_row_bytes < row_bytes) || (rows > 1 && out_row_bytes < row_bytes) ||
        (layers > 1 && out_layer_bytes < row_bytes) || !elements_aligned(LCPP_I32, parents))
        return LCPP_ERR_INVALID_ARG;
    // no two rows of out in one place: with neither all of a layer nor all of a row's layers together, layers that are
    // dl apart must not come as near as row_bytes to rows that are di apart
    if (layers > 1 && rows > 1 && out_layer_bytes < (rows - 1) * out_row_bytes + row_bytes &&
        out_row_bytes < (layers - 1) * out_layer_bytes + row_bytes)
        for (uint64_t dl = 1; dl < layers && dl * out_layer_bytes < (rows - 1) * out_row_bytes + row_bytes; ++dl) {
            const uint64_t at = dl * out_layer_bytes, di = at / out_row_bytes, past = at % out_row_bytes;
            if ((di >= 1 && di < rows && past < row_bytes) || (di + 1 < rows && out_row_bytes - past < row_bytes))
                return LCPP_ERR_INVALID_ARG;
        }
    // A row may be read after another row's copy took its place.  Apart as they lie, as layers (halves of each layer of
    // one buffer, say) or as rows a stride apart.
    const uint64_t in_block = rows_in ? (rows_in - 1) * in_row_bytes + row_bytes : 0;
    const uint64_t out_block = (rows - 1) * out_row_bytes + row_bytes;
    bool apart = Region(in, layers, in_layer_bytes, in_block).apart(Region(out, layers, out_layer_bytes, out_block));
    if (!apart && rows_in > 1 && rows > 1 && in_row_bytes == out_row_bytes &&
        (layers == 1 || (in_layer_bytes | out_layer_bytes) % in_row_bytes == 0)) {
        const uint64_t l = layers - 1, r = in_row_bytes;
        apart = Region(in, l * (in_layer_bytes / r) + rows_in, r, row_bytes)
                    .apart(Region(out, l * (out_layer_bytes / r) + rows, r, row_bytes));
    }
    if (!apart || !Region(out, layers, out_layer_bytes, out_block).apart(Region(parents, rows * 4))) return LCPP_ERR_INVALID_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    uint64_t bits = (uint64_t)(uintptr_t)in | (uint64_t)(uintptr_t)out | row_bytes;
    if (layers > 1) bits |= in_layer_bytes | out_layer_bytes;
    if (rows_in > 1) bits |= in_row_bytes;
    if (rows > 1) bits |= out_row_bytes;
    auto launch = [&](auto kernel, uint64_t span) -> lcpp_status {
        const uint64_t parts = ceil_div(row_bytes, span), units = rows * layers * parts;
        if (parts > 0xffffffffull || ceil_div(units, BEAM_COPY_WARPS) > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
        ProfScope prof("beam_reorder", s);
        kernel<<<(unsigned)ceil_div(units, BEAM_COPY_WARPS), BEAM_COPY_WARPS * 32, 0, s>>>(
            (const char*)in, in_layer_bytes, in_row_bytes, (char*)out, out_layer_bytes, out_row_bytes, parents,
            (uint32_t)rows_in, (uint32_t)rows, row_bytes, units, (uint32_t)parts);
        count_launch();
        return check_launch();
    };
    if (bits % 16 == 0) return launch(beam_reorder_kernel<16>, 32 * 16 * BEAM_COPY);
    if (bits % 4 == 0) return launch(beam_reorder_kernel<4>, 32 * 4 * 2 * BEAM_COPY);
    return launch(beam_reorder_kernel<1>, 32 * 4 * 2 * BEAM_COPY);
}
