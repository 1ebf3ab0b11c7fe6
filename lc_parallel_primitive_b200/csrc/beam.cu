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
constexpr uint32_t ORDERED_NONE = 0x007fffffu;  // ordered(-inf)

// Candidate list of one row: key = ordered score << 32 | ~(place), and tokens.
struct BeamTemp {
    float* score;    // [rows][K]
    int32_t* token;  // [rows][K]
};

template <typename T>
__global__ void __launch_bounds__(BEAM_THREADS)
beam_rows_kernel(const T* logits, uint64_t stride, const float* scores, const uint8_t* finished, int beams,
                 uint32_t vocab, int eos, BeamTemp tmp) {
    __shared__ uint64_t s_key[BEAM_THREADS / 32];
    __shared__ float s_sum[BEAM_THREADS / 32];
    const uint64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float score = scores[row];
    const bool done = finished && finished[row];
    float* out_score = tmp.score + row * beams;
    int32_t* out_token = tmp.token + row * beams;
    if (done || !(score > -INFINITY)) {
        if (tid < beams) {
            out_score[tid] = done && tid == 0 && score > -INFINITY ? score : -INFINITY;
            out_token[tid] = max(eos, 0);
        }
        return;
    }
    const T* z = logits + row * stride;
    float top = -INFINITY, total = 0.0f;
    uint64_t below = ~0ull;  // keys of earlier rounds are not below it
    for (int j = 0; j < beams; ++j) {
        uint64_t best = 0;
        for (uint32_t v = tid; v < vocab; v += BEAM_THREADS) {
            const uint64_t key = (uint64_t)ordered(widen(z[v])) << 32 | ~v;
            if (key < below && key > best) best = key;
        }
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        if (lane == 0) s_key[warp] = best;
        __syncthreads();
        best = 0;
        for (int w = 0; w < BEAM_THREADS / 32; ++w) best = max(best, s_key[w]);
        __syncthreads();
        below = best;
        const float zj = best ? unordered((uint32_t)(best >> 32)) : -INFINITY;
        if (j == 0) {
            top = zj;
            float sum = 0.0f;
            for (uint32_t v = tid; v < vocab; v += BEAM_THREADS) {
                const float zv = widen(z[v]);
                if (zv > -INFINITY) sum += zv == top ? 1.0f : __expf(zv - top);
            }
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            if (lane == 0) s_sum[warp] = sum;
            __syncthreads();
            for (int w = 0; w < BEAM_THREADS / 32; ++w) total += s_sum[w];
        }
        if (tid == 0) {
            out_score[j] = zj > -INFINITY ? score + ((zj == top ? 0.0f : zj - top) - logf(total)) : -INFINITY;
            out_token[j] = best ? (int32_t)~(uint32_t)best : max(eos, 0);
        }
    }
}

__global__ void __launch_bounds__(32)
beam_merge_kernel(BeamTemp tmp, const uint8_t* finished, int beams, int eos, float* scores_out, int32_t* tokens_out,
                  int32_t* parents_out, uint8_t* finished_out) {
    const uint64_t first = (uint64_t)blockIdx.x * beams;
    const int lane = threadIdx.x, n = beams * beams;
    uint64_t below = ~0ull;
    for (int j = 0; j < beams; ++j) {
        uint64_t best = 0;
        for (int i = lane; i < n; i += 32) {
            const uint64_t key = (uint64_t)ordered(tmp.score[first * beams + i]) << 32 | ~(uint32_t)i;
            if (key < below && key > best) best = key;
        }
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        below = best;
        if (lane == 0) {
            const bool any = (uint32_t)(best >> 32) > ORDERED_NONE;
            const uint32_t i = ~(uint32_t)best;
            const uint64_t parent = any ? first + i / beams : first + j;
            const int32_t token = any ? tmp.token[first * beams + i] : max(eos, 0);
            scores_out[first + j] = any ? tmp.score[first * beams + i] : -INFINITY;
            tokens_out[first + j] = token;
            parents_out[first + j] = (int32_t)parent;
            if (finished_out) finished_out[first + j] = !any || (finished && finished[parent]) || token == eos;
        }
    }
}

// out[l][i] = in[l][parents[i]], rows of bytes; a negative parent: zeros.
__global__ void __launch_bounds__(256)
beam_reorder_kernel(const char* in, uint64_t in_layer, uint64_t in_row, char* out, uint64_t out_layer, uint64_t out_row,
                    const int32_t* parents, uint64_t rows_in, uint64_t rows, uint64_t row_bytes) {
    const uint64_t i = blockIdx.x % rows, l = blockIdx.x / rows;
    int64_t from = parents[i];
    if (from >= (int64_t)rows_in) {
        set_error(LCPP_ERR_INVALID_ARG);
        from = -1;
    }
    const char* src = in + l * in_layer + from * in_row;
    char* dst = out + l * out_layer + i * out_row;
    for (uint64_t b = threadIdx.x; b < row_bytes; b += 256) dst[b] = from >= 0 ? src[b] : 0;
}

static size_t beam_temp_bytes(uint64_t rows, uint64_t beams) { return 2 * align_up(rows * beams * 4, 256); }

}  // namespace lcpp

using namespace lcpp;

extern "C" size_t lcpp_beam_select_temp_bytes(uint64_t batches, uint32_t beams, uint64_t vocab) {
    (void)vocab;
    if (beams < 1 || beams > BEAM_MAX) return 0;
    return beam_temp_bytes(batches * beams, beams);
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
    BeamTemp tmp{(float*)temp, (int32_t*)((char*)temp + align_up(rows * beams * 4, 256))};
    cudaStream_t s = (cudaStream_t)stream;
    return dispatch_float(dtype, [&](auto t) -> lcpp_status {
        using T = decltype(t);
        ProfScope prof("beam_select", s);
        beam_rows_kernel<T><<<(unsigned)rows, BEAM_THREADS, 0, s>>>((const T*)logits, logits_stride, scores_in,
                                                                    finished_in, (int)beams, (uint32_t)vocab, eos_token, tmp);
        beam_merge_kernel<<<(unsigned)batches, 32, 0, s>>>(tmp, finished_in, (int)beams, eos_token, scores_out,
                                                           tokens_out, parents_out, finished_out);
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
    ProfScope prof("beam_reorder", s);
    beam_reorder_kernel<<<(unsigned)(rows * layers), 256, 0, s>>>((const char*)in, in_layer_bytes, in_row_bytes,
                                                                  (char*)out, out_layer_bytes, out_row_bytes, parents,
                                                                  rows_in, rows, row_bytes);
    count_launch();
    return check_launch();
}
