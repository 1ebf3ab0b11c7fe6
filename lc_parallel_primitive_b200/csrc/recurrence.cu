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

constexpr int LR_TILE = 128;                  // rows of a tile, and rows between two saved states
constexpr int LR_WARPS = 8;
constexpr int LR_THREADS = LR_WARPS * 32;
constexpr int LR_ROWS = LR_TILE / LR_WARPS;   // consecutive rows of one warp
constexpr uint32_t LR_ALL = (1u << LR_ROWS) - 1;
constexpr int LR_LANE_BYTES = 4;              // of one row, per lane: 1 float or 2 halves
constexpr int LR_ROW_BYTES = 32 * LR_LANE_BYTES;
constexpr int LR_BUF = LR_TILE * LR_ROW_BYTES;  // 16 KiB: one matrix of a tile

struct LrShape {
    uint64_t rows, channels, sequences, length;  // length: rows of a sequence when offsets is null
    const uint32_t* offsets;                     // sequences + 1 row offsets, or null
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
    __device__ __forceinline__ float add(float x) const { return GATE == LCPP_GATE_SIGMOID ? na * x : x; }  // b
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

// ---- Which rows begin and end sequences ------------------------------------
// Found by each warp for its LR_ROWS rows; bit i stands for row first + i.
struct LrMarks {
    uint32_t head, tail, valid;  // first / last row of a sequence; row of any sequence
    int64_t base;                // offsets: sequence of lane 0's offset
    uint32_t off;                // offsets: offsets[base + lane]
};

// Number of offsets[0 .. count) that are <= row, minus 1 (-1: none); the warp narrows the range 32-fold a step.
__device__ __forceinline__ int64_t lr_search(const uint32_t* offsets, uint64_t count, uint64_t row) {
    const int lane = threadIdx.x & 31;
    uint64_t lo = 0, n = count;  // the answer + 1 lies in [lo, lo + n]
    while (n > 0) {
        const uint64_t step = (n + 31) / 32, at = lo + (lane + 1) * step - 1;
        const bool le = at < lo + n && offsets[at] <= row;
        const int full = __popc(__ballot_sync(0xffffffffu, le));  // leading lanes, the offsets ascend
        lo += full * step;
        n = min(step - 1, full * step < n ? n - full * step : 0);
    }
    return (int64_t)lo - 1;
}

__device__ __forceinline__ LrMarks lr_marks(const LrShape& sh, uint64_t first) {
    const int lane = threadIdx.x & 31;
    LrMarks m;
    m.base = 0;
    m.off = 0;
    if (!sh.offsets) {
        const uint32_t row = (uint32_t)first + lane, length = (uint32_t)sh.length;
        const uint32_t at = __ballot_sync(0xffffffffu, row % length == 0);
        m.valid = __ballot_sync(0xffffffffu, lane < LR_ROWS && first + lane < sh.rows);
        m.head = at & m.valid;
        m.tail = (at >> 1) & m.valid;
        return m;
    }
    const uint64_t S = sh.sequences;
    const uint64_t lo = sh.offsets[0], hi = min((uint64_t)sh.offsets[S], sh.rows);
    m.valid = __ballot_sync(0xffffffffu, lane < LR_ROWS && first + lane >= lo && first + lane < hi);
    uint32_t head = 0, tail = 0;
    const int64_t at = max(lr_search(sh.offsets, S + 1, first), (int64_t)0);
    m.base = at;
    for (uint64_t i = at; ; i += 32) {
        const uint32_t off = i + lane <= S ? sh.offsets[i + lane] : 0xffffffffu;
        if (i == (uint64_t)at) m.off = off;
        if (off >= first && off < first + LR_ROWS) head |= 1u << (off - first);
        if (off > first && off <= first + LR_ROWS && off > lo) tail |= 1u << (off - first - 1);
        if (i + 32 > S || __any_sync(0xffffffffu, off > first + LR_ROWS)) break;
    }
    m.head = __reduce_or_sync(0xffffffffu, head) & m.valid;
    m.tail = __reduce_or_sync(0xffffffffu, tail) & m.valid;
    return m;
}

// Sequence of a valid row of the warp (warp-uniform call).
__device__ __forceinline__ uint64_t lr_sequence(const LrShape& sh, const LrMarks& m, uint64_t row) {
    if (!sh.offsets) return (uint32_t)row / (uint32_t)sh.length;
    const uint32_t le = __ballot_sync(0xffffffffu, m.off <= row);
    int64_t s = m.base + __popc(le) - 1;
    if (le == 0xffffffffu) s = lr_search(sh.offsets, sh.sequences + 1, row);
    return (uint64_t)min(max(s, (int64_t)0), (int64_t)sh.sequences - 1);
}

// ---- Look-back between the tiles of a column -----------------------------------
// A tile maps the state before it to the state after it, h -> A h + H.  Words
// are float32 and their own flag: LR_NONE (a NaN that arithmetic does not make)
// until published, so no status word and no ordering is needed.  pair[tile]
// [channel] = (A, H) of the tile alone, state[tile][channel] = the state after it.
constexpr uint32_t LR_NONE = 0xffffffffu;

struct LrChain {
    uint32_t* ticket;  // starts at LR_NONE
    float2* pair;
    float* state;
    uint64_t width;  // channels, rounded up to whole column tiles
};
__device__ __forceinline__ float lr_word(float v) { return __float_as_uint(v) == LR_NONE ? __uint_as_float(0x7fffffffu) : v; }
__device__ __forceinline__ bool lr_there(float v) { return __float_as_uint(v) != LR_NONE; }
__device__ __forceinline__ void lr_put(float* p, float v) {
    asm volatile("st.relaxed.gpu.global.f32 [%0], %1;" ::"l"(p), "f"(lr_word(v)) : "memory");
}
__device__ __forceinline__ void lr_put(float2* p, float2 v) {
    asm volatile("st.relaxed.gpu.global.v2.f32 [%0], {%1, %2};" ::"l"(p), "f"(lr_word(v.x)), "f"(lr_word(v.y)) : "memory");
}
__device__ __forceinline__ float lr_get(const float* p) {
    float v;
    asm volatile("ld.relaxed.gpu.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float2 lr_get(const float2* p) {
    float2 v;
    asm volatile("ld.relaxed.gpu.global.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
    return v;
}

// The next tile's number, for all threads of the CTA.
__device__ __forceinline__ uint32_t lr_ticket(const LrChain& ch, uint32_t* shared) {
    __syncthreads();
    if (threadIdx.x == 0) *shared = atomicAdd(ch.ticket, 1u) + 1u;
    __syncthreads();
    return *shared;
}

// ---- Tiles in shared memory ----------------------------------------------------
// How rows can be copied: by 16-byte or 4-byte asynchronous copies, or element
// by element (2-byte elements on odd addresses or strides).
enum { LR_COPY16 = 0, LR_COPY4 = 1, LR_COPY_ELEMENT = 2 };

// Copies rows [row0, row0 + LR_TILE) x one column tile of a matrix to buf
// (LR_ROW_BYTES a row); rows from `rows` on and channels from `channels` on are
// left as they are.  Asynchronous copies are part of the caller's next commit.
template <typename T, int COPY>
__device__ __forceinline__ void lr_fetch(char* buf, const T* m, uint64_t stride, uint64_t row0, uint64_t rows,
                                         uint32_t channel0, uint32_t channels) {
    const int tid = threadIdx.x;
    const uint32_t left = (uint32_t)min((uint64_t)LR_TILE, rows - row0);
    if constexpr (COPY == LR_COPY16) {
        constexpr int PER_ROW = LR_ROW_BYTES / 16, STEP = LR_THREADS / PER_ROW, V = 16 / sizeof(T);
        const uint32_t r0 = tid / PER_ROW, c = (tid % PER_ROW) * V;
        if (channel0 + c >= channels) return;
        const T* src = m + (row0 + r0) * stride + channel0 + c;
        char* dst = buf + tid * 16;
#pragma unroll
        for (int j = 0; j < LR_TILE / STEP; ++j, src += STEP * stride)
            if (r0 + j * STEP < left) cp_async16(dst + j * LR_THREADS * 16, src);
    } else if constexpr (COPY == LR_COPY4) {
        constexpr int V = 4 / sizeof(T);
        const uint32_t r0 = tid / 32, c = (tid % 32) * V;
        if (channel0 + c >= channels) return;
        const T* src = m + (row0 + r0) * stride + channel0 + c;
        char* dst = buf + tid * 4;
#pragma unroll 8
        for (int j = 0; j < LR_TILE / LR_WARPS; ++j, src += LR_WARPS * stride)
            if (r0 + j * LR_WARPS < left) cp_async4(dst + j * LR_THREADS * 4, src);
    } else {
        constexpr int PER_ROW = LR_ROW_BYTES / sizeof(T), STEP = LR_THREADS / PER_ROW;
        const uint32_t r0 = tid / PER_ROW, c = tid % PER_ROW;
        if (channel0 + c >= channels) return;
        const T* src = m + (row0 + r0) * stride + channel0 + c;
        T* dst = (T*)buf + tid;
#pragma unroll 16
        for (int j = 0; j < LR_TILE / STEP; ++j, src += STEP * stride)
            if (r0 + j * STEP < left) dst[j * LR_THREADS] = *src;
    }
}

// One lane's channels of one row, in shared memory.
template <typename T> struct LrLane;
template <> struct LrLane<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ void load(const char* row, float* v) { v[0] = ((const float*)row)[threadIdx.x & 31]; }
};
template <> struct LrLane<__half> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void load(const char* row, float* v) {
        const float2 f = __half22float2(((const __half2*)row)[threadIdx.x & 31]);
        v[0] = f.x, v[1] = f.y;
    }
};
template <> struct LrLane<__nv_bfloat16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void load(const char* row, float* v) {
        const uint32_t b = ((const uint32_t*)row)[threadIdx.x & 31];
        v[0] = __uint_as_float(b << 16), v[1] = __uint_as_float(b & 0xffff0000u);
    }
};
// Stores one lane's channels (`left` of them in range; wide: 4-byte stores are aligned).
template <typename T, bool WIDE>
__device__ __forceinline__ void lr_store(T* p, const float* v, int left) {
    if constexpr (sizeof(T) == 4) {
        if (left > 0) *p = v[0];
    } else if constexpr (WIDE) {
        if (left > 0) {
            uint32_t b;
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 h = __floats2half2_rn(v[0], v[1]);
                memcpy(&b, &h, 4);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
                memcpy(&b, &h, 4);
            }
            *(uint32_t*)p = b;
        }
    } else {
        if (left > 0) p[0] = narrow<T>(v[0]);
        if (left > 1) p[1] = narrow<T>(v[1]);
    }
}

// The state before tile k of a column (REVERSE: behind it), from the LR_WINDOW
// tiles before it, two of which each warp reads.  The CTA reads the window
// again until every channel finds a state in it, and goes from the nearest one
// down the tiles, state = A state + H, just as those tiles do themselves: the
// result does not depend on how far back the state was found.
constexpr int LR_WINDOW = 2 * LR_WARPS;

template <int N, bool REVERSE>
__device__ __forceinline__ void lr_lookback(const LrChain& ch, int64_t k, int64_t tiles, uint32_t channel0,
                                            uint32_t channels, float2* s_win, float* carry) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t limit = g_spin_limit;
    uint32_t spins = 0;
    while (true) {
        float st[2][N];
        float2 pr[2][N];
        bool there;
        do {  // until each of this warp's tiles shows its map or its state
            there = true;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t d = 1 + warp + j * LR_WARPS, p = REVERSE ? k + d : k - d;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const uint32_t c = channel0 + lane * N + i;
                    st[j][i] = 0.0f;  // before the first tile the state is 0
                    pr[j][i] = make_float2(0.0f, 0.0f);
                    if (p >= 0 && p < tiles && c < channels) {
                        st[j][i] = lr_get(ch.state + (uint64_t)p * ch.width + c);
                        pr[j][i] = lr_get(ch.pair + (uint64_t)p * ch.width + c);
                        there &= lr_there(st[j][i]) || (lr_there(pr[j][i].x) && lr_there(pr[j][i].y));
                    }
                }
            }
            if (!there) {
                if (++spins > limit) {
                    set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
                    break;
                }
                if (spins > 16) __nanosleep(32);
            }
        } while (!there);
        // a state is handed over as (LR_NONE, state)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i)
                s_win[(warp + j * LR_WARPS) * 32 * N + lane * N + i] =
                    lr_there(st[j][i]) ? make_float2(__uint_as_float(LR_NONE), st[j][i]) : pr[j][i];
        __syncthreads();
        bool open = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int j = 0;
            while (j < LR_WINDOW && lr_there(s_win[j * 32 * N + lane * N + i].x)) ++j;
            open |= j == LR_WINDOW;
            carry[i] = j < LR_WINDOW ? s_win[j * 32 * N + lane * N + i].y : 0.0f;
            while (j-- > 0) {
                const float2 w = s_win[j * 32 * N + lane * N + i];
                carry[i] = fmaf(w.x, carry[i], w.y);
            }
        }
        if (!__syncthreads_or(open && spins <= limit)) return;
        if (++spins > limit) set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
    }
}

// ---- Forward ---------------------------------------------------------------------
template <typename T, int GATE, int COPY>
__global__ void __launch_bounds__(LR_THREADS, 3) lr_forward_kernel(LrForward p, LrChain ch, uint32_t row_tiles, uint32_t col_tiles) {
    constexpr int N = LrLane<T>::N, C = 32 * N;
    extern __shared__ __align__(128) char smem[];  // [2 stages][gate, in][LR_BUF]
    __shared__ float2 s_agg[LR_WARPS * C], s_win[LR_WINDOW * C];
    __shared__ uint32_t s_reset[LR_WARPS], s_ticket;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t channels = (uint32_t)p.sh.channels;
    const uint64_t total = (uint64_t)row_tiles * col_tiles;
    const bool chained = row_tiles > 1;

    auto fetch = [&](uint64_t t, int stage) {
        if (t < total) {
            const uint64_t row0 = t / col_tiles * LR_TILE;
            const uint32_t c0 = (uint32_t)(t % col_tiles) * C;
            char* buf = smem + stage * 2 * LR_BUF;
            lr_fetch<T, COPY>(buf, (const T*)p.gate, p.gate_stride, row0, p.sh.rows, c0, channels);
            lr_fetch<T, COPY>(buf + LR_BUF, (const T*)p.in, p.in_stride, row0, p.sh.rows, c0, channels);
        }
        cp_async_commit();
    };
    // Tiles in the order of their tickets, down the rows: a tile waits only for tiles of smaller tickets, which
    // CTAs take in ascending order, so the smallest unfinished one never waits.
    uint64_t cur = blockIdx.x, next = (uint64_t)blockIdx.x + gridDim.x;
    if (chained) {
        cur = lr_ticket(ch, &s_ticket);
        fetch(cur, 0);
        next = lr_ticket(ch, &s_ticket);
    } else {
        fetch(cur, 0);
    }
    fetch(next, 1);
    for (int stage = 0; cur < total; stage ^= 1) {
        const uint32_t k = (uint32_t)(cur / col_tiles), c0 = (uint32_t)(cur % col_tiles) * C;
        const uint64_t first = (uint64_t)k * LR_TILE + warp * LR_ROWS;
        const uint32_t c = c0 + lane * N;
        const int left = (int)min((uint32_t)N, channels - min(channels, c));
        const LrMarks m = lr_marks(p.sh, first);
        cp_async_wait_prior1();
        __syncthreads();
        uint32_t taken = 0;
        if (chained && tid == 0) taken = atomicAdd(ch.ticket, 1u) + 1u;
        // ---- this warp's rows alone: h_after = A h_before + H ---------------------
        const char* buf = smem + stage * 2 * LR_BUF + warp * LR_ROWS * LR_ROW_BYTES;
        const bool plain = m.valid == LR_ALL && m.head == 0;
        float pre[LR_ROWS][N], loc[LR_ROWS][N], A[N], H[N];  // row r: h = pre h_before + loc
        auto init = [&](int r, float* h) {  // state before the first row of a sequence
            const uint64_t s = lr_sequence(p.sh, m, first + r);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = p.init && i < left ? p.init[s * p.init_stride + c + i] : 0.0f;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) A[i] = 1.0f, H[i] = 0.0f;
#pragma unroll
        for (int r = 0; r < LR_ROWS; ++r) {
            float g[N], x[N];
            LrLane<T>::load(buf + r * LR_ROW_BYTES, g);
            LrLane<T>::load(buf + LR_BUF + r * LR_ROW_BYTES, x);
            if (!plain) {
                if (m.head >> r & 1) {
                    init(r, H);
#pragma unroll
                    for (int i = 0; i < N; ++i) A[i] = 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const Gate<GATE> gt(g[i]);
                H[i] = fmaf(gt.a, H[i], gt.add(x[i]));
                A[i] *= gt.a;
                if (!plain && !(m.valid >> r & 1)) A[i] = 0.0f, H[i] = 0.0f;
                pre[r][i] = A[i], loc[r][i] = H[i];
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s_agg[warp * C + lane * N + i] = make_float2(A[i], H[i]);
        if (lane == 0) s_reset[warp] = !plain;  // nothing from before the warp's rows passes them
        if (chained && tid == 0) s_ticket = taken;
        __syncthreads();
        const uint64_t after = chained ? s_ticket : next + gridDim.x;
        // ---- the tile as a whole is published --------------------------------------
        bool reset = false;
        float before[N], tA[N], tH[N];  // (A, H) of the warps before this one; of the tile
        float bA[N];
        bool breset = false;
#pragma unroll
        for (int i = 0; i < N; ++i) tA[i] = 1.0f, tH[i] = 0.0f, bA[i] = 1.0f, before[i] = 0.0f;
#pragma unroll
        for (int w = 0; w < LR_WARPS; ++w) {
            if (w == warp) {
                breset = reset;
#pragma unroll
                for (int i = 0; i < N; ++i) bA[i] = tA[i], before[i] = tH[i];
            }
            const bool cuts = s_reset[w];
            reset |= cuts;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 a = s_agg[w * C + lane * N + i];
                tH[i] = cuts ? a.y : fmaf(a.x, tH[i], a.y);
                tA[i] = cuts ? 0.0f : tA[i] * a.x;
            }
        }
        const uint64_t at = (uint64_t)k * ch.width + c;
        const bool more = k + 1 < row_tiles;
        if (more && warp == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) {
                    if (reset) lr_put(ch.state + at + i, tH[i]);
                    else if (k > 0) lr_put(ch.pair + at + i, make_float2(tA[i], tH[i]));
                    else lr_put(ch.state + at + i, tH[i]);
                }
        }
        fetch(after, stage);  // every warp has read this stage
        // ---- the state before the tile ----------------------------------------------
        float carry[N];
#pragma unroll
        for (int i = 0; i < N; ++i) carry[i] = 0.0f;
        if (k > 0) {
            lr_lookback<N, false>(ch, k, row_tiles, c0, channels, s_win, carry);
            if (more && warp == 0 && !reset)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < left) lr_put(ch.state + at + i, fmaf(tA[i], carry[i], tH[i]));
        }
        if (p.saved && warp == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) p.saved[(uint64_t)k * channels + c + i] = carry[i];
        // ---- outputs -------------------------------------------------------------------
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!breset) before[i] = fmaf(bA[i], carry[i], before[i]);
        T* out = (T*)p.out + first * p.out_stride + c;
        if (plain && m.tail == 0) {
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r) {
                float h[N];
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] = fmaf(pre[r][i], before[i], loc[r][i]);
                lr_store<T, COPY != LR_COPY_ELEMENT>(out + r * p.out_stride, h, left);
            }
        } else {
            // From the first head or padding row on nothing depends on the state before the warp's rows (not even as
            // 0 times it, which an infinity or NaN of another sequence would survive).
            const int reach = __ffs(m.head | ~m.valid) - 1;
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r) {
                float h[N];
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] = r < reach ? fmaf(pre[r][i], before[i], loc[r][i]) : loc[r][i];
                if (first + r < p.sh.rows) lr_store<T, COPY != LR_COPY_ELEMENT>(out + r * p.out_stride, h, left);
                if ((m.tail >> r & 1) && p.last) {
                    const uint64_t s = lr_sequence(p.sh, m, first + r);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i < left) p.last[s * channels + c + i] = h[i];
                }
            }
        }
        cur = next, next = after;
    }
    cp_async_wait_all();
}

// Before a chained or packed call: the chain's words are LR_NONE, and sequences without rows pass their state
// on, to[s] = from[s] (0 without from).
__global__ void __launch_bounds__(256)
lr_prepare_kernel(uint4* words, uint64_t count, LrShape sh, const float* from, uint64_t from_stride, float* to) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (uint64_t)gridDim.x * 256)
        words[i] = make_uint4(LR_NONE, LR_NONE, LR_NONE, LR_NONE);
    if (!to) return;
    for (uint64_t s = blockIdx.x; s < sh.sequences; s += gridDim.x) {
        if (sh.offsets ? min((uint64_t)sh.offsets[s], sh.rows) < min((uint64_t)sh.offsets[s + 1], sh.rows) : sh.length > 0)
            continue;
        for (uint64_t c = threadIdx.x; c < sh.channels; c += 256)
            to[s * sh.channels + c] = from ? from[s * from_stride + c] : 0.0f;
    }
}

// ---- Backward --------------------------------------------------------------------
// Tiles from the last to the first: the chain carries mu, mu_before = A mu_after + M.
template <typename T, int GATE, int COPY>
__global__ void __launch_bounds__(LR_THREADS, 2) lr_backward_kernel(LrBackward p, LrChain ch, uint32_t row_tiles, uint32_t col_tiles) {
    constexpr int N = LrLane<T>::N, C = 32 * N;
    extern __shared__ __align__(128) char smem[];  // [2 stages][gate, in, grad_out][LR_BUF]
    __shared__ float2 s_agg[LR_WARPS * C], s_win[LR_WINDOW * C];
    __shared__ float s_mu[LR_WARPS * C];
    __shared__ uint32_t s_cut[LR_WARPS], s_ticket;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t channels = (uint32_t)p.sh.channels;
    const uint64_t total = (uint64_t)row_tiles * col_tiles;
    const bool chained = row_tiles > 1;

    auto fetch = [&](uint64_t t, int stage) {
        if (t < total) {
            const uint64_t row0 = (row_tiles - 1 - t / col_tiles) * LR_TILE;
            const uint32_t c0 = (uint32_t)(t % col_tiles) * C;
            char* buf = smem + stage * 3 * LR_BUF;
            lr_fetch<T, COPY>(buf, (const T*)p.gate, p.gate_stride, row0, p.sh.rows, c0, channels);
            lr_fetch<T, COPY>(buf + LR_BUF, (const T*)p.in, p.in_stride, row0, p.sh.rows, c0, channels);
            if (p.grad_out)
                lr_fetch<T, COPY>(buf + 2 * LR_BUF, (const T*)p.grad_out, p.grad_out_stride, row0, p.sh.rows, c0, channels);
        }
        cp_async_commit();
    };
    uint64_t cur = blockIdx.x, next = (uint64_t)blockIdx.x + gridDim.x;  // as in the forward kernel
    if (chained) {
        cur = lr_ticket(ch, &s_ticket);
        fetch(cur, 0);
        next = lr_ticket(ch, &s_ticket);
    } else {
        fetch(cur, 0);
    }
    fetch(next, 1);
    for (int stage = 0; cur < total; stage ^= 1) {
        const uint32_t k = row_tiles - 1 - (uint32_t)(cur / col_tiles), c0 = (uint32_t)(cur % col_tiles) * C;
        const uint64_t first = (uint64_t)k * LR_TILE + warp * LR_ROWS;
        const uint32_t c = c0 + lane * N;
        const int left = (int)min((uint32_t)N, channels - min(channels, c));
        float start[N];  // state before the tile
#pragma unroll
        for (int i = 0; i < N; ++i) start[i] = i < left ? p.saved[(uint64_t)k * channels + c + i] : 0.0f;
        const LrMarks m = lr_marks(p.sh, first);
        cp_async_wait_prior1();
        __syncthreads();
        uint32_t taken = 0;
        if (chained && tid == 0) taken = atomicAdd(ch.ticket, 1u) + 1u;
        const char* buf = smem + stage * 3 * LR_BUF + warp * LR_ROWS * LR_ROW_BYTES;
        const bool plain = m.valid == LR_ALL && m.head == 0 && m.tail == 0;
        auto init = [&](int r, float* h) {
            const uint64_t s = lr_sequence(p.sh, m, first + r);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = p.init && i < left ? p.init[s * p.init_stride + c + i] : 0.0f;
        };
        auto last = [&](int r, float* mu) {
            const uint64_t s = lr_sequence(p.sh, m, first + r);
#pragma unroll
            for (int i = 0; i < N; ++i) mu[i] = p.grad_last && i < left ? p.grad_last[s * channels + c + i] : 0.0f;
        };
        // ---- this warp's rows alone, in both directions ------------------------------
        float a[LR_ROWS][N], h[LR_ROWS][N], A[N], H[N], M[N];  // h: b first, the state before the row later
#pragma unroll
        for (int i = 0; i < N; ++i) A[i] = 1.0f, H[i] = 0.0f, M[i] = 0.0f;
#pragma unroll
        for (int r = 0; r < LR_ROWS; ++r) {
            float g[N], x[N];
            LrLane<T>::load(buf + r * LR_ROW_BYTES, g);
            LrLane<T>::load(buf + LR_BUF + r * LR_ROW_BYTES, x);
            if (!plain && (m.head >> r & 1)) init(r, H);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const Gate<GATE> gt(g[i]);
                a[r][i] = gt.a, h[r][i] = gt.add(x[i]);
                H[i] = fmaf(a[r][i], H[i], h[r][i]);
                A[i] *= a[r][i];
            }
        }
        auto grad = [&](int r, float* v) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = 0.0f;
            if (p.grad_out) LrLane<T>::load(buf + 2 * LR_BUF + r * LR_ROW_BYTES, v);
        };
#pragma unroll
        for (int r = LR_ROWS - 1; r >= 0; --r) {
            float v[N];
            grad(r, v);
            if (!plain && (m.tail >> r & 1)) last(r, M);
#pragma unroll
            for (int i = 0; i < N; ++i) M[i] = a[r][i] * (v[i] + M[i]);
            if (!plain && !(m.valid >> r & 1))
#pragma unroll
                for (int i = 0; i < N; ++i) M[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s_agg[warp * C + lane * N + i] = make_float2(A[i], H[i]);
            s_mu[warp * C + lane * N + i] = M[i];
        }
        // bit 0: no state from before the warp's rows passes them; bit 1: no gradient from behind them does
        if (lane == 0) s_cut[warp] = (m.valid != LR_ALL || m.head ? 1u : 0u) | (m.valid != LR_ALL || m.tail ? 2u : 0u);
        if (chained && tid == 0) s_ticket = taken;
        __syncthreads();
        const uint64_t after = chained ? s_ticket : next + gridDim.x;
        // ---- the state before this warp's rows ------------------------------------------
#pragma unroll
        for (int w = 0; w < LR_WARPS - 1; ++w)
            if (w < warp) {
                const bool cuts = s_cut[w] & 1u;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float2 v = s_agg[w * C + lane * N + i];
                    start[i] = cuts ? v.y : fmaf(v.x, start[i], v.y);
                }
            }
        // ---- the tile's gradient map is published ---------------------------------------
        bool cut = false, behind_cut = false;
        float tA[N], tM[N], bA[N], mu[N];  // of the tile; of the warps behind this one
#pragma unroll
        for (int i = 0; i < N; ++i) tA[i] = 1.0f, tM[i] = 0.0f, bA[i] = 1.0f, mu[i] = 0.0f;
#pragma unroll
        for (int w = LR_WARPS - 1; w >= 0; --w) {
            if (w == warp) {
                behind_cut = cut;
#pragma unroll
                for (int i = 0; i < N; ++i) bA[i] = tA[i], mu[i] = tM[i];
            }
            const bool cuts = s_cut[w] & 2u;
            cut |= cuts;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float Aw = s_agg[w * C + lane * N + i].x, Mw = s_mu[w * C + lane * N + i];
                tM[i] = cuts ? Mw : fmaf(Aw, tM[i], Mw);
                tA[i] = cuts ? 0.0f : tA[i] * Aw;
            }
        }
        const uint64_t at = (uint64_t)k * ch.width + c;
        const bool more = k > 0;
        if (more && warp == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) {
                    if (cut || k + 1 == row_tiles) lr_put(ch.state + at + i, tM[i]);
                    else lr_put(ch.pair + at + i, make_float2(tA[i], tM[i]));
                }
        }
        // ---- states before each row: while the chain is on its way ----------------------
#pragma unroll
        for (int r = 0; r < LR_ROWS; ++r) {
            if (!plain && (m.head >> r & 1)) init(r, start);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float b = h[r][i];
                h[r][i] = start[i];
                start[i] = fmaf(a[r][i], start[i], b);
            }
        }
        if (k + 1 < row_tiles) {
            float carry[N];
            lr_lookback<N, true>(ch, k, row_tiles, c0, channels, s_win, carry);
            if (more && warp == 0 && !cut)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < left) lr_put(ch.state + at + i, fmaf(tA[i], carry[i], tM[i]));
            if (!behind_cut)
#pragma unroll
                for (int i = 0; i < N; ++i) mu[i] = fmaf(bA[i], carry[i], mu[i]);
        }
        // ---- gradients ---------------------------------------------------------------------
        T* out_gate = (T*)p.grad_gate + first * p.grad_gate_stride + c;
        T* out_in = (T*)p.grad_in + first * p.grad_in_stride + c;
        constexpr bool WIDE = COPY != LR_COPY_ELEMENT;
#pragma unroll
        for (int r = LR_ROWS - 1; r >= 0; --r) {
            float g[N], x[N], v[N], dg[N], dx[N];
            LrLane<T>::load(buf + r * LR_ROW_BYTES, g);
            LrLane<T>::load(buf + LR_BUF + r * LR_ROW_BYTES, x);
            grad(r, v);
            if (!plain && (m.tail >> r & 1)) last(r, mu);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const Gate<GATE> gt(g[i]);
                const float lam = v[i] + mu[i];
                dg[i] = gt.grad_gate(lam, h[r][i], x[i]);
                dx[i] = gt.grad_in(lam);
                mu[i] = a[r][i] * lam;
            }
            if (plain) {
                lr_store<T, WIDE>(out_gate + r * p.grad_gate_stride, dg, left);
                lr_store<T, WIDE>(out_in + r * p.grad_in_stride, dx, left);
            } else {
                if (!(m.valid >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) dg[i] = dx[i] = mu[i] = 0.0f;
                if (first + r < p.sh.rows) {
                    lr_store<T, WIDE>(out_gate + r * p.grad_gate_stride, dg, left);
                    lr_store<T, WIDE>(out_in + r * p.grad_in_stride, dx, left);
                }
                if ((m.head >> r & 1) && p.grad_init) {
                    const uint64_t s = lr_sequence(p.sh, m, first + r);
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (i < left) p.grad_init[s * channels + c + i] = mu[i];
                }
            }
        }
        __syncthreads();  // the stage is free
        fetch(after, stage);
        cur = next, next = after;
    }
    cp_async_wait_all();
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
    const Gate<GATE> g(widen(gate[r * gate_stride + c]));
    const float h = fmaf(g.a, before, g.add(widen(in[r * in_stride + c])));
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

// Temp: [ticket | pad to 256][pair: row tiles x width float2][state: row tiles x width float], all LR_NONE at the start.
static uint64_t lr_width(uint64_t channels) { return align_up(channels, 64); }
static size_t lr_chain_bytes(uint64_t rows, uint64_t channels) {
    const uint64_t tiles = ceil_div(rows, LR_TILE);
    return tiles > 1 ? 256 + tiles * lr_width(channels) * 12 : 0;
}
static LrChain lr_chain(void* temp, uint64_t rows, uint64_t channels) {
    const uint64_t n = ceil_div(rows, LR_TILE) * lr_width(channels);
    char* t = (char*)temp;
    return LrChain{(uint32_t*)t, (float2*)(t + 256), (float*)(t + 256 + n * 8), lr_width(channels)};
}

// How the rows of these matrices can be copied.
struct LrCopy {
    uint64_t bits;  // all addresses and byte strides or-ed together
    LrCopy(uint64_t channels, size_t e) : bits(channels * e) {}
    LrCopy& add(const void* p, uint64_t stride, size_t e) {
        bits |= (uint64_t)(uintptr_t)p | stride * e;
        return *this;
    }
    int kind() const { return bits % 16 == 0 ? LR_COPY16 : bits % 4 == 0 ? LR_COPY4 : LR_COPY_ELEMENT; }
};

static lcpp_status lr_prepare(const LrShape& sh, void* temp, const float* from, uint64_t from_stride, float* to,
                              cudaStream_t s) {
    const uint64_t words = lr_chain_bytes(sh.rows, sh.channels) / 16;
    if (!sh.offsets && sh.length) to = nullptr;  // no sequence is empty
    if (!words && !to) return LCPP_OK;
    const uint64_t grid = max(ceil_div(words, 256 * 4), to ? min(sh.sequences, (uint64_t)1024) : 0);
    ProfScope prof("lr_prepare", s);
    lr_prepare_kernel<<<(unsigned)min(grid, (uint64_t)device_info().sms * 8), 256, 0, s>>>((uint4*)temp, words, sh, from,
                                                                                       from_stride, to);
    count_launch();
    return check_launch();
}

template <typename K, typename P>
static lcpp_status lr_launch(K kernel, const char* name, const P& p, const LrShape& sh, int channels_per_tile,
                             size_t smem, int ctas_per_sm, void* temp, cudaStream_t s) {
    const uint64_t row_tiles = ceil_div(sh.rows, LR_TILE), col_tiles = ceil_div(sh.channels, channels_per_tile);
    if (row_tiles * col_tiles > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return LCPP_ERR_CUDA;
    const uint64_t grid = min(row_tiles * col_tiles, (uint64_t)device_info().sms * ctas_per_sm);
    ProfScope prof(name, s);
    kernel<<<(unsigned)grid, LR_THREADS, smem, s>>>(p, lr_chain(temp, sh.rows, sh.channels), (uint32_t)row_tiles,
                                                    (uint32_t)col_tiles);
    count_launch();
    return check_launch();
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
    return max(lr_chain_bytes(rows, channels), (size_t)256);
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
    const lcpp_status ready = lr_prepare(sh, temp, init, init_stride, last, s);
    if (ready != LCPP_OK || !rows) return ready;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        constexpr int G = decltype(g)::value, C = 32 * LR_LANE_BYTES / sizeof(T);
        const int copy = LrCopy(channels, sizeof(T)).add(gate_in, gate_stride, sizeof(T)).add(in, in_stride, sizeof(T))
                             .add(out, out_stride, sizeof(T)).kind();
        auto launch = [&](auto kernel) { return lr_launch(kernel, "lr_forward", p, sh, C, 4 * LR_BUF, 3, temp, s); };
        if (copy == LR_COPY16) return launch(lr_forward_kernel<T, G, LR_COPY16>);
        if (copy == LR_COPY4) return launch(lr_forward_kernel<T, G, LR_COPY4>);
        return launch(lr_forward_kernel<T, G, LR_COPY_ELEMENT>);
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
    const lcpp_status ready = lr_prepare(sh, temp, grad_last, channels, grad_init, s);
    if (ready != LCPP_OK || !rows) return ready;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        constexpr int G = decltype(g)::value, C = 32 * LR_LANE_BYTES / sizeof(T);
        LrCopy align(channels, sizeof(T));
        align.add(gate_in, gate_stride, sizeof(T)).add(in, in_stride, sizeof(T))
            .add(grad_gate, grad_gate_stride, sizeof(T)).add(grad_in, grad_in_stride, sizeof(T));
        if (grad_out) align.add(grad_out, grad_out_stride, sizeof(T));
        const int copy = align.kind();
        auto launch = [&](auto kernel) { return lr_launch(kernel, "lr_backward", p, sh, C, 6 * LR_BUF, 2, temp, s); };
        if (copy == LR_COPY16) return launch(lr_backward_kernel<T, G, LR_COPY16>);
        if (copy == LR_COPY4) return launch(lr_backward_kernel<T, G, LR_COPY4>);
        return launch(lr_backward_kernel<T, G, LR_COPY_ELEMENT>);
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
