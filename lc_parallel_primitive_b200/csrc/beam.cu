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

// ---- One part of one row ---------------------------------------------------------
// A CTA reads its part of a row once: each thread takes vectors of 16 bytes,
// BEAM_VECS of them a chunk, and keeps the sum of 2^(z log2(e) - K) with a whole
// number K, so that a larger maximum rescales the sum exactly, and the largest
// value of each chunk.  The beams-th largest of the threads' maxima is at most
// the beams-th best logit of the part: only the few chunks that reach it are read
// again (from L2), and what reaches it there is sorted.  The streaming loop thus
// spends nothing on the selection but a maximum (half an instruction a 2-byte
// element).
constexpr int BEAM_VECS = 4;
constexpr int BEAM_TILE = BEAM_THREADS * BEAM_VECS;  // vectors of a tile of a part
constexpr int BEAM_TILES = 16;                       // tiles of a part at most
constexpr int BEAM_KEYS = 1024;                      // logits that may reach the threads' bound

// Results of one part: its `beams` best keys (ordered logit << 32 | ~token, 0: none), largest logit, and the sum of
// exp(z - largest).
struct BeamTemp {
    uint64_t* key;   // [rows][parts][beams]
    float2* total;   // [rows][parts]
};

// The vector at address `at`, of which elements [lo, hi) belong to the row; the others, and NaN, read as -inf.
template <typename T>
struct BeamVector {
    static constexpr int E = 16 / sizeof(T);
    uint4 w;
    __device__ __forceinline__ void load(const T* at, int64_t lo, int64_t hi) {
        if (lo <= 0 && hi >= E) {
            w = ld_stream((const uint4*)at);
            return;
        }
        float v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e >= lo && e < hi ? widen(at[e]) : -INFINITY;
        pack(v);
    }
    __device__ __forceinline__ void pack(const float* v) {
        T t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = narrow<T>(v[e]);
        memcpy(&w, t, 16);
    }
    // No NaN from here on; the largest element.
    __device__ __forceinline__ float clean_max() {
        if constexpr (sizeof(T) == 4) {
            float v[4];
            memcpy(v, &w, 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaxf(v[e], -INFINITY);
            memcpy(&w, v, 16);
            return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        } else {
            using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
            T2 v[4], low;
            memcpy(v, &w, 16);
            low.x = low.y = narrow<T>(-INFINITY);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __hmax2(v[e], low);
            memcpy(&w, v, 16);
            const T2 m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
            return fmaxf(widen(m.x), widen(m.y));
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
    return scores[row] > -INFINITY && !(finished && finished[row]);
}

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS, 4)
beam_rows_kernel(const T* logits, uint64_t stride, const float* scores, const uint8_t* finished, int beams,
                 uint32_t vocab, uint32_t parts, BeamTemp tmp) {
    constexpr int E = BeamVector<T>::E, WARPS = BEAM_THREADS / 32;
    __shared__ float s_chunk[BEAM_TILES][BEAM_THREADS];
    __shared__ uint64_t s_key[BEAM_KEYS];
    __shared__ float s_top[WARPS][32], s_scale[WARPS], s_sum[WARPS];
    __shared__ int s_count;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint64_t row = blockIdx.x / parts;
    const uint32_t part = blockIdx.x - (uint32_t)row * parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (!beam_live(scores, finished, row)) return;
    const T* z = logits + row * stride;
    const int64_t shift = ((uintptr_t)z & 15) / sizeof(T);  // elements between the first vector's address and z
    const T* base = z - shift;
    const uint32_t vectors = (uint32_t)((shift + vocab + E - 1) / E);
    const uint32_t tiles = (vectors + BEAM_TILE - 1) / BEAM_TILE;
    const uint32_t tile0 = (uint32_t)((uint64_t)tiles * part / parts), tile1 = (uint32_t)((uint64_t)tiles * (part + 1) / parts);
    const int n = (int)(tile1 - tile0);
    auto load = [&](BeamVector<T>* v, uint32_t tile) {
#pragma unroll
        for (int q = 0; q < BEAM_VECS; ++q) {
            const uint32_t at = tile * BEAM_TILE + q * BEAM_THREADS + tid;
            // elements of the vector before the row's first and behind its last
            const int64_t first = shift - (int64_t)at * E, end = first + vocab;
            if (at < vectors) v[q].load(base + (int64_t)at * E, first, end);
            else v[q].load(base, E, 0);
        }
    };
    if (tid == 0) s_count = 0;
    float top = -INFINITY, scale = -1e30f, sum = 0.0f;  // sum of 2^(z log2e - scale)
    BeamVector<T> v[BEAM_VECS], ahead[BEAM_VECS];
    if (n > 0) load(v, tile0);
    for (int j = 0; j < n; ++j) {
        if (j + 1 < n) load(ahead, tile0 + j + 1);
        float m = v[0].clean_max();
#pragma unroll
        for (int q = 1; q < BEAM_VECS; ++q) m = fmaxf(m, v[q].clean_max());
        s_chunk[j][tid] = m;
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
#pragma unroll
        for (int q = 0; q < BEAM_VECS; ++q) v[q] = ahead[q];
    }
    // ---- the part's maximum and sum, and the beams-th largest of the threads' maxima ----
    float sorted = warp_sort(top);
    s_top[warp][lane] = sorted;
    float warp_scale = scale;
    for (int o = 16; o; o >>= 1) warp_scale = fmaxf(warp_scale, __shfl_xor_sync(0xffffffffu, warp_scale, o));
    float warp_sum = sum * beam_ex2(scale - warp_scale);
    for (int o = 16; o; o >>= 1) warp_sum += __shfl_xor_sync(0xffffffffu, warp_sum, o);
    if (lane == 0) s_scale[warp] = warp_scale, s_sum[warp] = warp_sum;
    for (int half = WARPS / 2; half; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            sorted = warp_merge(sorted, s_top[warp + half][lane]);
            s_top[warp][lane] = sorted;
        }
    }
    __syncthreads();
    const float largest = s_top[0][0], bound = s_top[0][beams - 1];
    // ---- what reaches the bound ------------------------------------------------------
    for (int j = 0; j < n; ++j) {
        if (!(s_chunk[j][tid] >= bound && s_chunk[j][tid] > -INFINITY)) continue;
        load(v, tile0 + j);
        for (int q = 0; q < BEAM_VECS; ++q) {
            v[q].clean_max();
            for (int e = 0; e < E; ++e) {
                const float x = v[q].get(e);
                if (x >= bound && x > -INFINITY) {
                    const int at = atomicAdd(&s_count, 1);
                    const uint32_t token = (uint32_t)(((int64_t)(tile0 + j) * BEAM_TILE + q * BEAM_THREADS + tid) * E + e - shift);
                    if (at < BEAM_KEYS) s_key[at] = (uint64_t)ordered(x) << 32 | (uint32_t)~token;
                }
            }
        }
    }
    __syncthreads();
    uint64_t* out = tmp.key + (row * parts + part) * beams;
    const uint32_t first = (uint32_t)max((int64_t)tile0 * BEAM_TILE * E - shift, (int64_t)0);
    const uint32_t end = (uint32_t)min((int64_t)tile1 * BEAM_TILE * E - shift, (int64_t)vocab);
    if (s_count <= BEAM_KEYS) {
        if (warp == 0) {
            const uint64_t key = warp_top(s_key, s_count);
            if (lane < beams) out[lane] = key;
        }
    } else {  // many equal logits: the best below the last one found, `beams` times over
        uint64_t below = ~0ull;
        for (int j = 0; j < beams; ++j) {
            uint64_t best = 0;
            for (uint32_t t = first + tid; t < end; t += BEAM_THREADS) {
                const float x = widen(z[t]);
                const uint64_t key = (uint64_t)ordered(x) << 32 | (uint32_t)~t;
                if (x >= bound && x > -INFINITY && key < below && key > best) best = key;
            }
            for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
            __syncthreads();
            if (lane == 0) s_key[warp] = best;
            __syncthreads();
            for (int w = 0; w < WARPS; ++w) best = max(best, s_key[w]);
            below = best;
            if (tid == 0) out[j] = best;
        }
    }
    float all_scale = s_scale[0], total = 0.0f;
    for (int w = 1; w < WARPS; ++w) all_scale = fmaxf(all_scale, s_scale[w]);
    for (int w = 0; w < WARPS; ++w) total += s_sum[w] * beam_ex2(s_scale[w] - all_scale);
    // relative to the largest term, which went through the same product
    total /= beam_ex2(fmaf(largest, BEAM_LOG2E, -all_scale));
    if (!(total >= 0.5f && total < INFINITY) && largest > -INFINITY) {
        // a maximum of +inf or one whose scaled value is out of range: term by term
        total = 0.0f;
        for (uint32_t t = first + tid; t < end; t += BEAM_THREADS) {
            const float x = fmaxf(widen(z[t]), -INFINITY);
            total += x == largest ? 1.0f : __expf(x - largest);
        }
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        __syncthreads();
        if (lane == 0) s_sum[warp] = total;
        __syncthreads();
        total = 0.0f;
        for (int w = 0; w < WARPS; ++w) total += s_sum[w];
    }
    if (tid == 0) tmp.total[row * parts + part] = make_float2(largest, total);
}

// ---- One batch entry ----------------------------------------------------------------
// A warp a beam joins the parts of its row; then the first warp takes the best
// of all beams' candidates.
template <int WARPS>
__global__ void __launch_bounds__(WARPS * 32)
beam_merge_kernel(BeamTemp tmp, const float* scores, const uint8_t* finished, int beams, uint32_t parts, int eos,
                  float* scores_out, int32_t* tokens_out, int32_t* parents_out, uint8_t* finished_out) {
    __shared__ uint64_t s_key[BEAM_MAX * BEAM_MAX];
    __shared__ float s_score[BEAM_MAX * BEAM_MAX];
    __shared__ int32_t s_token[BEAM_MAX * BEAM_MAX];
    const uint64_t first = (uint64_t)blockIdx.x * beams;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int k = warp; k < beams; k += WARPS) {
        const uint64_t row = first + k;
        const float score = scores[row];
        float best = -INFINITY;
        int32_t token = max(eos, 0);
        if (beam_live(scores, finished, row)) {
            const uint64_t key = warp_top(tmp.key + row * parts * beams, (int)(parts * beams));
            float largest = -INFINITY, total = 0.0f;
            for (uint32_t i = lane; i < parts; i += 32) largest = fmaxf(largest, tmp.total[row * parts + i].x);
            for (int o = 16; o; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            for (uint32_t i = lane; i < parts; i += 32) {
                const float2 t = tmp.total[row * parts + i];
                if (t.x > -INFINITY) total += t.x == largest ? t.y : t.y * __expf(t.x - largest);
            }
            for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            if (key) {
                const float z = unordered((uint32_t)(key >> 32));
                best = score + ((z == largest ? 0.0f : z - largest) - logf(total));
                token = (int32_t)~(uint32_t)key;
            }
        } else if (lane == 0 && score > -INFINITY) {
            best = score;  // finished: it stays
        }
        if (lane < beams) {
            const int at = k * beams + lane;
            s_score[at] = best, s_token[at] = token;
            s_key[at] = best > -INFINITY ? (uint64_t)ordered(best) << 32 | (uint32_t)~at : 0;
        }
    }
    __syncthreads();
    if (warp == 0) {
        const uint64_t key = warp_top(s_key, beams * beams);
        if (lane < beams) {
            const uint32_t at = ~(uint32_t)key;
            const bool any = key != 0;
            const uint64_t parent = any ? first + at / beams : first + lane;
            const int32_t token = any ? s_token[at] : max(eos, 0);
            scores_out[first + lane] = any ? s_score[at] : -INFINITY;
            tokens_out[first + lane] = token;
            parents_out[first + lane] = (int32_t)parent;
            if (finished_out) finished_out[first + lane] = !any || (finished && finished[parent]) || token == eos;
        }
    }
}

// ---- Reordering ------------------------------------------------------------------------
// out[l][i] = in[l][parents[i]], rows of bytes; a negative parent: zeros.  A warp
// copies BEAM_COPY vectors a lane of one row, all loads before the first store.
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
constexpr int BEAM_PARTS_PER_SM = 8;
static uint32_t beam_parts(uint64_t rows, uint64_t vocab, size_t element, uint64_t sms) {
    const uint64_t per_vector = 16 / element;
    const uint64_t tiles = ceil_div(ceil_div(vocab + per_vector - 1, per_vector), BEAM_TILE);  // at any alignment
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
    const uint64_t rows = batches * beams;
    cudaStream_t s = (cudaStream_t)stream;
    return dispatch_float(dtype, [&](auto t) -> lcpp_status {
        using T = decltype(t);
        const uint32_t parts = beam_parts(rows, vocab, sizeof(T), device_info().sms);
        if (rows * parts > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
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
        const auto kernel = beams > 1 ? beam_merge_kernel<8> : beam_merge_kernel<1>;
        if (cudaLaunchKernelEx(&cfg, kernel, tmp, scores_in, finished_in, (int)beams, parts, eos_token, scores_out,
                               tokens_out, parents_out, finished_out) != cudaSuccess)
            return LCPP_ERR_CUDA;
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
    if (!in || !out || !parents || rows * layers > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    if ((rows_in > 1 && in_row_bytes < row_bytes) || (rows > 1 && out_row_bytes < row_bytes)) return LCPP_ERR_INVALID_ARG;
    // a row may be read after another row's copy took its place
    const char *i0 = (const char*)in, *o0 = (const char*)out;
    const uint64_t in_span = (layers - 1) * in_layer_bytes + (rows_in ? rows_in - 1 : 0) * in_row_bytes + row_bytes;
    const uint64_t out_span = (layers - 1) * out_layer_bytes + (rows - 1) * out_row_bytes + row_bytes;
    if (o0 < i0 + in_span && i0 < o0 + out_span) return LCPP_ERR_INVALID_ARG;
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
