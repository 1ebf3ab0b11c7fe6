// Gated linear recurrence (DeviceLinearRecurrence): forward over sequences,
// its backward pass, and the single-token step.
//
//   linear:  h_t = a_t h_{t-1} + b_t                   (gate = a, in = b)
//   sigmoid: a_t = 1 / (1 + exp(-g_t)),
//            h_t = a_t h_{t-1} + (1 - a_t) x_t         (gate = g, in = x)
//
// per channel, rows = tokens.  Backward, with lam_t the gradient of h_t and
// mu_t = a_t lam_t that of h_{t-1}:
//   lam_t = dout_t + mu_{t+1}   (mu past the last row = dlast)
//   linear:  da = lam_t h_{t-1},                        db = lam_t
//   sigmoid: dg = lam_t (h_{t-1} - x_t) a_t (1 - a_t),  dx = (1 - a_t) lam_t
// h_{t-1} is recomputed from one saved float32 state per LR_TILE rows, which
// the forward pass writes: 4 / LR_TILE bytes an element instead of reading the
// outputs back, and no rounding of h_{t-1} to the element type.
#include "float_types.cuh"

namespace lcpp {

constexpr int LR_TILE = 128;  // rows between two saved states

struct LrShape {
    uint64_t rows, channels, sequences, length;  // length: rows of a sequence when offsets is null
    const uint32_t* offsets;                     // sequences + 1 row offsets, or null
    // First row and past-the-end row of sequence s, clamped to the rows there are.
    __device__ __forceinline__ uint64_t begin(uint64_t s) const {
        return offsets ? min((uint64_t)offsets[s], rows) : s * length;
    }
};

// Sigmoid: a = 1 / (1 + e) and 1 - a = e a with e = exp(-g), so that
// neither loses its leading digits when the other is near 1.  Past g = -80, e a
// is 1 to float32 (and e overflows soon after); a NaN stays one.
__device__ __forceinline__ float ex2_approx(float v) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float rcp_approx(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
template <int GATE>
struct Gate {
    float a, na;  // a and (sigmoid) 1 - a
    __device__ __forceinline__ explicit Gate(float g) {
        if constexpr (GATE == LCPP_GATE_SIGMOID) {
            const float e = ex2_approx(g * -1.44269504f);
            a = rcp_approx(1.0f + e);
            na = g < -80.0f ? 1.0f : e * a;
        } else {
            a = g;
            na = 1.0f;
        }
    }
    __device__ __forceinline__ float next(float h, float x) const {
        return GATE == LCPP_GATE_SIGMOID ? fmaf(a, h, na * x) : fmaf(a, h, x);
    }
    __device__ __forceinline__ float grad_gate(float lam, float before, float x) const {
        return GATE == LCPP_GATE_SIGMOID ? lam * (before - x) * (a * na) : lam * before;
    }
    __device__ __forceinline__ float grad_in(float lam) const { return GATE == LCPP_GATE_SIGMOID ? na * lam : lam; }
};

struct LrForward {
    LrShape sh;
    const void *gate, *in;
    void* out;
    uint64_t gate_stride, in_stride, out_stride, init_stride;
    const float* init;
    float *last, *saved;
};

struct LrBackward {
    LrShape sh;
    const void *gate, *in, *grad_out;
    void *grad_gate, *grad_in;
    uint64_t gate_stride, in_stride, grad_out_stride, grad_gate_stride, grad_in_stride, init_stride;
    const float *init, *grad_last, *saved;
    float* grad_init;
};

constexpr int LR_THREADS = 128;

// One thread per (sequence, channel), row after row.
template <typename T, int GATE>
__global__ void __launch_bounds__(LR_THREADS) lr_forward_kernel(LrForward p) {
    const uint64_t c = (uint64_t)blockIdx.y * LR_THREADS + threadIdx.x;
    if (c >= p.sh.channels) return;
    const T *gate = (const T*)p.gate + c, *in = (const T*)p.in + c;
    T* out = (T*)p.out + c;
    for (uint64_t s = blockIdx.x; s < p.sh.sequences; s += gridDim.x) {
        const uint64_t lo = p.sh.begin(s), hi = p.sh.begin(s + 1);
        float h = p.init ? p.init[s * p.init_stride + c] : 0.0f;
        for (uint64_t r = lo; r < hi; ++r) {
            if (p.saved && r % LR_TILE == 0) p.saved[r / LR_TILE * p.sh.channels + c] = h;
            h = Gate<GATE>(widen(gate[r * p.gate_stride])).next(h, widen(in[r * p.in_stride]));
            out[r * p.out_stride] = narrow<T>(h);
        }
        if (p.last) p.last[s * p.sh.channels + c] = h;
    }
    // rows that belong to no sequence
    if (blockIdx.x == 0) {
        for (uint64_t r = 0; r < p.sh.begin(0); ++r) out[r * p.out_stride] = narrow<T>(0.0f);
        for (uint64_t r = p.sh.begin(p.sh.sequences); r < p.sh.rows; ++r) out[r * p.out_stride] = narrow<T>(0.0f);
    }
}

template <typename T, int GATE>
__global__ void __launch_bounds__(LR_THREADS) lr_backward_kernel(LrBackward p) {
    const uint64_t c = (uint64_t)blockIdx.y * LR_THREADS + threadIdx.x;
    if (c >= p.sh.channels) return;
    const T *gate = (const T*)p.gate + c, *in = (const T*)p.in + c, *grad_out = (const T*)p.grad_out + c;
    T *grad_gate = (T*)p.grad_gate + c, *grad_in = (T*)p.grad_in + c;
    float before[LR_TILE];
    for (uint64_t s = blockIdx.x; s < p.sh.sequences; s += gridDim.x) {
        const uint64_t lo = p.sh.begin(s), hi = p.sh.begin(s + 1);
        float mu = p.grad_last ? p.grad_last[s * p.sh.channels + c] : 0.0f;
        for (uint64_t end = hi; end > lo;) {  // tiles from the last to the first
            const uint64_t tile = (end - 1) / LR_TILE, first = max(tile * LR_TILE, lo);
            float h = first > lo ? p.saved[tile * p.sh.channels + c]
                      : p.init   ? p.init[s * p.init_stride + c]
                                 : 0.0f;
            for (uint64_t r = first; r < end; ++r) {
                before[r - first] = h;
                h = Gate<GATE>(widen(gate[r * p.gate_stride])).next(h, widen(in[r * p.in_stride]));
            }
            for (uint64_t r = end; r-- > first;) {
                const Gate<GATE> g(widen(gate[r * p.gate_stride]));
                const float x = widen(in[r * p.in_stride]);
                const float lam = mu + (p.grad_out ? widen(grad_out[r * p.grad_out_stride]) : 0.0f);
                grad_gate[r * p.grad_gate_stride] = narrow<T>(g.grad_gate(lam, before[r - first], x));
                grad_in[r * p.grad_in_stride] = narrow<T>(g.grad_in(lam));
                mu = g.a * lam;
            }
            end = first;
        }
        if (p.grad_init) p.grad_init[s * p.sh.channels + c] = mu;
    }
    if (blockIdx.x == 0) {
        auto clear = [&](uint64_t r) {
            grad_gate[r * p.grad_gate_stride] = narrow<T>(0.0f);
            grad_in[r * p.grad_in_stride] = narrow<T>(0.0f);
        };
        for (uint64_t r = 0; r < p.sh.begin(0); ++r) clear(r);
        for (uint64_t r = p.sh.begin(p.sh.sequences); r < p.sh.rows; ++r) clear(r);
    }
}

// One token: row i continues the state of row parents[i] (itself without
// parents; zero for a negative parent).
template <typename T, int GATE>
__global__ void __launch_bounds__(256)
lr_step_kernel(const T* gate, uint64_t gate_stride, const T* in, uint64_t in_stride, const float* states_in,
               uint64_t rows_in, const int32_t* parents, float* states_out, T* out, uint64_t out_stride,
               uint64_t rows, uint64_t channels) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * channels) return;
    const uint64_t r = i / channels, c = i - r * channels;
    int64_t from = parents ? (int64_t)parents[r] : (int64_t)r;
    if (from >= (int64_t)rows_in) {
        set_error(LCPP_ERR_INVALID_ARG);
        from = -1;
    }
    const float before = states_in && from >= 0 ? states_in[from * channels + c] : 0.0f;
    const float h = Gate<GATE>(widen(gate[r * gate_stride + c])).next(before, widen(in[r * in_stride + c]));
    states_out[i] = h;
    if (out) out[r * out_stride + c] = narrow<T>(h);
}

constexpr uint64_t LR_MAX_ROWS = 0xffffffffull;  // offsets are 32-bit
constexpr uint64_t LR_MAX_CHANNELS = 1ull << 20;

static lcpp_status lr_check(int gate, int dtype, const LrShape& sh, const void* gate_in, const void* in) {
    if ((gate != LCPP_GATE_LINEAR && gate != LCPP_GATE_SIGMOID) || !is_float_dtype(dtype)) return LCPP_ERR_INVALID_ARG;
    if (sh.rows > LR_MAX_ROWS || sh.channels > LR_MAX_CHANNELS || sh.sequences > LR_MAX_ROWS) return LCPP_ERR_INVALID_ARG;
    if (!sh.offsets && (sh.length > LR_MAX_ROWS || sh.sequences * sh.length != sh.rows)) return LCPP_ERR_INVALID_ARG;
    if (sh.rows && sh.channels && (!gate_in || !in || !sh.sequences)) return LCPP_ERR_INVALID_ARG;
    return LCPP_OK;
}
// A row stride must reach past the channels (one row may have any).
static bool lr_stride_ok(uint64_t stride, uint64_t rows, uint64_t channels) {
    return rows <= 1 || (stride >= channels && stride < (1ull << 31));
}

template <typename F>
static lcpp_status lr_dispatch(int gate, int dtype, F&& f) {
    return dispatch_float(dtype, [&](auto t) -> lcpp_status {
        if (gate == LCPP_GATE_SIGMOID) return f(t, std::integral_constant<int, LCPP_GATE_SIGMOID>{});
        return f(t, std::integral_constant<int, LCPP_GATE_LINEAR>{});
    });
}

}  // namespace lcpp

using namespace lcpp;

extern "C" size_t lcpp_linear_recurrence_temp_bytes(uint64_t rows, uint64_t channels) {
    (void)rows;
    (void)channels;
    return 256;
}

extern "C" size_t lcpp_linear_recurrence_saved_bytes(uint64_t rows, uint64_t channels) {
    return align_up(ceil_div(rows, LR_TILE) * channels * sizeof(float), 256);
}

extern "C" lcpp_status lcpp_linear_recurrence_forward(
    int gate, int dtype, const void* gate_in, uint64_t gate_stride, const void* in, uint64_t in_stride, void* out,
    uint64_t out_stride, uint64_t rows, uint64_t channels, uint64_t num_sequences, uint64_t length,
    const uint32_t* offsets, const float* init, uint64_t init_stride, float* last, void* saved, void* temp,
    size_t temp_bytes, void* stream) {
    const LrShape sh{rows, channels, num_sequences, length, offsets};
    const lcpp_status ok = lr_check(gate, dtype, sh, gate_in, in);
    if (ok != LCPP_OK) return ok;
    if (!channels || !num_sequences) return LCPP_OK;
    if (rows && (!out || !lr_stride_ok(gate_stride, rows, channels) || !lr_stride_ok(in_stride, rows, channels) ||
                 !lr_stride_ok(out_stride, rows, channels)))
        return LCPP_ERR_INVALID_ARG;
    if (!temp || temp_bytes < lcpp_linear_recurrence_temp_bytes(rows, channels)) return LCPP_ERR_TEMP_TOO_SMALL;
    const LrForward p{sh, gate_in, in, out, gate_stride, in_stride, out_stride, init_stride, init, last, (float*)saved};
    cudaStream_t s = (cudaStream_t)stream;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        const dim3 grid((unsigned)min(num_sequences, (uint64_t)65536), (unsigned)ceil_div(channels, LR_THREADS));
        ProfScope prof("lr_forward", s);
        lr_forward_kernel<decltype(t), decltype(g)::value><<<grid, LR_THREADS, 0, s>>>(p);
        count_launch();
        return check_launch();
    });
}

extern "C" lcpp_status lcpp_linear_recurrence_backward(
    int gate, int dtype, const void* gate_in, uint64_t gate_stride, const void* in, uint64_t in_stride,
    const void* saved, const float* init, uint64_t init_stride, const void* grad_out, uint64_t grad_out_stride,
    const float* grad_last, void* grad_gate, uint64_t grad_gate_stride, void* grad_in, uint64_t grad_in_stride,
    float* grad_init, uint64_t rows, uint64_t channels, uint64_t num_sequences, uint64_t length,
    const uint32_t* offsets, void* temp, size_t temp_bytes, void* stream) {
    const LrShape sh{rows, channels, num_sequences, length, offsets};
    const lcpp_status ok = lr_check(gate, dtype, sh, gate_in, in);
    if (ok != LCPP_OK) return ok;
    if (!channels || !num_sequences) return LCPP_OK;
    if (rows && (!saved || !grad_gate || !grad_in || !lr_stride_ok(gate_stride, rows, channels) ||
                 !lr_stride_ok(in_stride, rows, channels) || !lr_stride_ok(grad_gate_stride, rows, channels) ||
                 !lr_stride_ok(grad_in_stride, rows, channels) ||
                 (grad_out && !lr_stride_ok(grad_out_stride, rows, channels))))
        return LCPP_ERR_INVALID_ARG;
    if (!temp || temp_bytes < lcpp_linear_recurrence_temp_bytes(rows, channels)) return LCPP_ERR_TEMP_TOO_SMALL;
    const LrBackward p{sh, gate_in, in, grad_out, grad_gate, grad_in, gate_stride, in_stride, grad_out_stride,
                       grad_gate_stride, grad_in_stride, init_stride, init, grad_last, (const float*)saved, grad_init};
    cudaStream_t s = (cudaStream_t)stream;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        const dim3 grid((unsigned)min(num_sequences, (uint64_t)65536), (unsigned)ceil_div(channels, LR_THREADS));
        ProfScope prof("lr_backward", s);
        lr_backward_kernel<decltype(t), decltype(g)::value><<<grid, LR_THREADS, 0, s>>>(p);
        count_launch();
        return check_launch();
    });
}

extern "C" lcpp_status lcpp_linear_recurrence_step(int gate, int dtype, const void* gate_in, uint64_t gate_stride,
                                                   const void* in, uint64_t in_stride, const float* states_in,
                                                   uint64_t rows_in, const int32_t* parents, float* states_out,
                                                   void* out, uint64_t out_stride, uint64_t rows, uint64_t channels,
                                                   void* stream) {
    if ((gate != LCPP_GATE_LINEAR && gate != LCPP_GATE_SIGMOID) || !is_float_dtype(dtype)) return LCPP_ERR_INVALID_ARG;
    if (rows > 0x7fffffffull || rows_in > 0x7fffffffull || channels > LR_MAX_CHANNELS) return LCPP_ERR_INVALID_ARG;
    if (!rows || !channels) return LCPP_OK;
    if (!gate_in || !in || !states_out || !lr_stride_ok(gate_stride, rows, channels) ||
        !lr_stride_ok(in_stride, rows, channels) || (out && !lr_stride_ok(out_stride, rows, channels)))
        return LCPP_ERR_INVALID_ARG;
    if (states_in && !parents && rows_in < rows) return LCPP_ERR_INVALID_ARG;
    if (parents && states_in) {  // a row may be read after another row's new state took its place
        const char *i0 = (const char*)states_in, *o0 = (const char*)states_out;
        if (o0 < i0 + rows_in * channels * sizeof(float) && i0 < o0 + rows * channels * sizeof(float))
            return LCPP_ERR_INVALID_ARG;
    }
    cudaStream_t s = (cudaStream_t)stream;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        ProfScope prof("lr_step", s);
        lr_step_kernel<T, decltype(g)::value><<<(unsigned)ceil_div(rows * channels, 256), 256, 0, s>>>(
            (const T*)gate_in, gate_stride, (const T*)in, in_stride, states_in, rows_in, parents, states_out, (T*)out,
            out_stride, rows, channels);
        count_launch();
        return check_launch();
    });
}
