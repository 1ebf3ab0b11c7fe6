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
//
// Both passes read each operand once and write each result once.  A tile is
// LR_TILE rows x one lane word (4 bytes) per lane of a warp; the compute warps
// of a CTA take LR_ROWS rows each and turn them into the affine map
// h_after = A h_before + H that the rows are.  Look-back warps join the maps of
// the CTA's warps and of the tiles before (a decoupled look-back, Merrill &
// Garland 2016, over affine maps) while the compute warps already turn the next
// tile into its maps, so that the chain from tile to tile has a whole tile's
// time to arrive.
//
// Measured on one B200: forward 65536 x 2048 bf16 196 us (4.1 TB/s, 63 % of the
// copy rate; 160 us with the chain's result dropped), f32 16384 x 2048 87 us;
// backward 65536 x 2048 bf16 316 us (65 %).  Bound by instructions (34 and 67 an
// element, 64 and 77 % of the issue slots), of which address and tile bookkeeping is
// half: 8 rows a lane do not amortise it, but 16 rows (with half the warps, or
// two CTAs of 8 warps an SM) take 229-235 / 379-398 us, since either the warps
// or the registers for two tiles at once run out.
#include "float_types.cuh"

namespace lcpp {

constexpr int LR_WARPS = 16;                    // compute warps
constexpr int LR_ROWS = 8;                      // consecutive rows of one warp
constexpr int LR_TILE = LR_WARPS * LR_ROWS;     // rows of a tile, and rows between two saved states
constexpr uint32_t LR_ALL = (1u << LR_ROWS) - 1;

// Division of 32-bit numbers by a fixed one: the high half of n * ceil(2^64 / d) is n / d for all n, d < 2^32
// (the error n / 2^64 cannot reach the next quotient, 1 / d away).
struct LrDivisor {
    uint32_t d;
    uint64_t m;
    explicit LrDivisor(uint64_t v) : d((uint32_t)v), m(v > 1 ? ~0ull / v + 1 : 0) {}
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return m ? (uint32_t)__umul64hi(m, n) : n; }
};

struct LrShape {
    uint64_t rows, channels, sequences;
    LrDivisor length;         // rows of a sequence when offsets is null
    const uint32_t* offsets;  // sequences + 1 row offsets, or null
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
    __device__ __forceinline__ float grad_gate(float before, float x) const {  // of h, by the gate
        return GATE == LCPP_GATE_SIGMOID ? (before - x) * (a * na) : before;
    }
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
// Every row has a code: LR_OUTSIDE (of all sequences), or LR_HEAD and LR_TAIL
// bits with the row's sequence (0 where neither bit is set).  Computed where
// all sequences have one length, else written by lr_prepare_kernel.
constexpr uint32_t LR_OUTSIDE = 1u << 31, LR_HEAD = 1u << 30, LR_TAIL = 1u << 29, LR_SEQUENCE = LR_TAIL - 1;

__device__ __forceinline__ uint32_t lr_code(const LrShape& sh, uint64_t row, const uint32_t* fetched) {
    if (row >= sh.rows) return LR_OUTSIDE;
    if (sh.offsets) return *fetched;
    const uint32_t r = (uint32_t)row, s = sh.length.div(r), at = r - s * sh.length.d;
    return (at == 0 ? LR_HEAD : 0) | (at + 1 == sh.length.d ? LR_TAIL : 0) | s;
}
// A warp's rows: no mark; one head and one tail at most (their states are read before the loop over the rows, which
// only selects); anything else.
enum { LR_PLAIN = 0, LR_SINGLE = 1, LR_MANY = 2 };

// The codes of a warp's rows, lane r holding row r's, and masks of them.
struct LrMarks {
    uint32_t code, head, tail, valid;
    __device__ __forceinline__ LrMarks() : code(0), head(0), tail(0), valid(LR_ALL) {}  // all inside a sequence
    __device__ __forceinline__ explicit LrMarks(uint32_t c) : code(c) {
        const bool mine = (threadIdx.x & 31) < LR_ROWS;
        head = __ballot_sync(0xffffffffu, mine && (c & LR_HEAD));
        tail = __ballot_sync(0xffffffffu, mine && (c & LR_TAIL));
        valid = __ballot_sync(0xffffffffu, mine && !(c & LR_OUTSIDE));
    }
    // Sequence of row r, which is a head or tail.
    __device__ __forceinline__ uint64_t sequence(const LrShape& sh, int r) const {
        return min((uint64_t)(__shfl_sync(0xffffffffu, code, r) & LR_SEQUENCE), sh.sequences - 1);
    }
    __device__ __forceinline__ int kind() const {
        if (valid != LR_ALL || (head & (head - 1)) || (tail & (tail - 1))) return LR_MANY;
        return head | tail ? LR_SINGLE : LR_PLAIN;
    }
    // Nothing from before the rows passes them; nothing from behind them does.
    __device__ __forceinline__ bool cuts() const { return head || valid != LR_ALL; }
    __device__ __forceinline__ bool cuts_back() const { return tail || valid != LR_ALL; }
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

// ---- Look-back between the tiles of a column -----------------------------------
// A tile maps the state before it to the state after it, h -> A h + H.  A tile's
// record for a channel is (A, H, state after it, -).  Words are float32 and their
// own flag: LR_NONE (a NaN that arithmetic does not make) until published, so no
// status word and no ordering is needed.
constexpr uint32_t LR_NONE = 0xffffffffu;

struct LrChain {
    float4* record;  // [row tile][width]
    uint64_t width;  // channels, rounded up to whole column tiles
};
__device__ __forceinline__ float lr_word(float v) { return __float_as_uint(v) == LR_NONE ? __uint_as_float(0x7fffffffu) : v; }
__device__ __forceinline__ bool lr_there(float v) { return __float_as_uint(v) != LR_NONE; }
__device__ __forceinline__ void lr_put_state(float4* r, float v) {
    asm volatile("st.relaxed.gpu.global.f32 [%0], %1;" ::"l"(&r->z), "f"(lr_word(v)) : "memory");
}
__device__ __forceinline__ void lr_put_map(float4* r, float a, float h) {
    asm volatile("st.relaxed.gpu.global.v2.f32 [%0], {%1, %2};" ::"l"(r), "f"(lr_word(a)), "f"(lr_word(h)) : "memory");
}
__device__ __forceinline__ float4 lr_get(const float4* r) {
    float4 v;
    asm volatile("ld.relaxed.gpu.global.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(r) : "memory");
    return v;
}

// The state of one channel behind the nearest of `left` tiles, whose records
// are at r, r + step, ... (with none left, the state is 0).  The lane reads W
// of them until one shows its state and all nearer ones their maps, and goes
// from there down the tiles, state = A state + H, as those tiles do themselves:
// the result does not depend on how far back the state was found.  Bounded by
// the spin limit, after which the error word is set.
// More records a read reach further where many tiles of a column are under way,
// but take time and registers: with 16 (8) instead of LR_FAR (LR_NEAR) the
// backward pass over 65536 x 1000 f32 spills and takes 345 us instead of 238,
// though the forward pass over 65536 x 128 bf16, with 74 tiles under way, 42
// instead of 49; 8 everywhere 60 there.  At 12 and 6 the forward kernels of 2-byte
// elements at odd addresses still spill 156 bytes, four backward ones 4 or 8.
constexpr int LR_NEAR = 6, LR_FAR = 12;

template <int W>
__device__ __forceinline__ float lr_lookback(const float4* r, int64_t step, uint32_t left, bool active) {
    const uint32_t limit = g_spin_limit;
    for (uint32_t spins = 0;; ++spins) {
        float4 v[W];
#pragma unroll
        for (int j = 0; j < W; ++j) {
            v[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (j < left) v[j] = lr_get(r + j * step);
        }
        uint32_t states = 0, maps = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            states |= lr_there(v[j].z) ? 1u << j : 0;
            maps |= lr_there(v[j].x) && lr_there(v[j].y) ? 1u << j : 0;
        }
        const int from = __ffs(states) - 1;  // the nearest with a state, if all nearer ones have maps
        const bool found = from >= 0 && (~maps & ((1u << from) - 1)) == 0;
        if (__all_sync(0xffffffffu, found || !active)) {
            float carry = 0.0f;
#pragma unroll
            for (int j = W - 1; j >= 0; --j) carry = j > from ? carry : j == from ? v[j].z : fmaf(v[j].x, carry, v[j].y);
            return carry;
        }
        if (spins >= limit) {
            if (!found && active) set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
            return 0.0f;
        }
        if (spins > 64) __nanosleep(32);
    }
}

// ---- Warps and their barriers ---------------------------------------------------
// A CTA has LR_WARPS compute warps, and for each 32 channels one publishing and
// one look-back warp, a channel a lane.  Tile i of a CTA (its i-th) uses buffer
// i & 1.  The compute warps write their maps and arrive at barriers 1 + (i & 1),
// on which the publishing warps wait, and 5 + (i & 1), for the look-back warps.
// The publishing warps join the maps and publish the tile's, a tile ahead of its
// outputs and whatever the look-back warps still wait for; these find the state
// before the tile meanwhile, and write every warp's start.  Both then arrive at
// 3 + (i & 1), on which the compute warps wait.  A compute warp writes the maps
// of tile i + 2 after it has waited for the starts of tile i, so two buffers do.
__device__ __forceinline__ void lr_sync(int barrier, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}
__device__ __forceinline__ void lr_arrive(int barrier, int threads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

// ---- Rows in shared memory -------------------------------------------------------
// A row of a tile is 32 words of 4 bytes, one a lane: 1 float or 2 halves.  How
// rows are copied, all asynchronously: 16 or 4 bytes at a time where rows are
// aligned so, else (2-byte elements on odd addresses or strides) the 33 aligned
// words around a row's elements, which the reader shifts.
enum { LR_COPY16 = 0, LR_COPY4 = 1, LR_COPY_ODD = 2 };

// One lane's part of copying a warp's rows of a column tile.
template <typename T, int COPY>
struct LrFetch {
    static constexpr int PER_ROW = COPY == LR_COPY16 ? 8 : 32;          // lanes a row
    static constexpr int STEP = 32 / PER_ROW;                           // rows a step
    static constexpr int BYTES = COPY == LR_COPY16 ? 16 : 4;            // a copy
    static constexpr int PITCH = COPY == LR_COPY_ODD ? 132 : 128;       // of rows in shared memory, in bytes
    static constexpr int BUF = LR_ROWS * PITCH;                         // a warp's rows
    const char* m;  // this lane's part of the warp's first rows
    uint64_t row_bytes;
    const char *begin, *end;  // of the matrix (LR_COPY_ODD)
    __device__ __forceinline__ LrFetch(const void* matrix, uint64_t stride, int warp, const LrShape& sh) {
        const int lane = threadIdx.x & 31;
        row_bytes = stride * sizeof(T);
        m = (const char*)matrix + (warp * LR_ROWS + lane / PER_ROW) * row_bytes + lane % PER_ROW * BYTES;
        begin = (const char*)matrix;
        end = begin + ((sh.rows - 1) * stride + sh.channels) * sizeof(T);
    }
    // Copies the warp's rows (n of them in range) of the tile `offset` bytes into the matrix, `channels` of whose
    // channels are in range, to buf; what is out of range is left as it is.  Part of the warp's next commit.
    __device__ __forceinline__ void copy(char* buf, uint64_t offset, int n, uint32_t channels) const {
        const int lane = threadIdx.x & 31, r0 = lane / PER_ROW, at = lane % PER_ROW * BYTES;
        const uint64_t step_bytes = row_bytes * STEP;
        const char* src = m + offset;
        char* dst = buf + r0 * PITCH + at;
        if constexpr (COPY != LR_COPY_ODD) {
            if (at >= channels * (int)sizeof(T)) return;
#pragma unroll
            for (int j = 0; j < LR_ROWS / STEP; ++j, src += step_bytes)
                if (r0 + j * STEP < n) {
                    if constexpr (COPY == LR_COPY16) cp_async16(dst + j * STEP * PITCH, src);
                    else cp_async4(dst + j * STEP * PITCH, src);
                }
        } else {
            // words 0 .. 31 of the rows, a row a step, of those that hold one of its channels; then the 33rd words, a
            // row a lane
            const int bytes = channels * (int)sizeof(T);
            const char* row0 = src - at;
            const char* tail = row0 + lane * row_bytes + 128;
            const bool tails = lane < min(n, LR_ROWS) && bytes == 128 && ((uintptr_t)tail & 2);
            if (n >= LR_ROWS && row0 >= begin + 4 && row0 + (LR_ROWS - 1) * row_bytes + 136 <= end) {
#pragma unroll
                for (int j = 0; j < LR_ROWS; ++j, src += step_bytes) {
                    const int odd = (int)((uintptr_t)src & 2);
                    if (at < bytes + odd) cp_async4(dst + j * PITCH, src - odd);
                }
                if (tails) cp_async4(buf + lane * PITCH + 128, tail - 2);
            } else {
                for (int j = 0; j < min(n, LR_ROWS); ++j, src += step_bytes) {
                    const int odd = (int)((uintptr_t)src & 2);
                    if (at < bytes + odd) word(dst + j * PITCH, src - odd);
                }
                if (tails) word(buf + lane * PITCH + 128, tail - 2);
            }
        }
    }
    // One aligned word, which at the matrix's ends is half outside it.
    __device__ __forceinline__ void word(char* dst, const char* src) const {
        if (src >= begin && src + 4 <= end) cp_async4(dst, src);
        else if (src >= begin) *(uint16_t*)dst = *(const uint16_t*)src;
        else *(uint16_t*)(dst + 2) = *(const uint16_t*)(src + 2);
    }
};

// Which of a warp's rows of a matrix start in the middle of a word (2-byte elements), as bits.
__device__ __forceinline__ uint32_t lr_odd_rows(const void* matrix, uint64_t offset, uint64_t stride) {
    return ((uintptr_t)matrix + offset & 2 ? 0xffu : 0u) ^ (stride & 1 ? 0xaau : 0u);  // a warp's first row is even
}

// A warp's rows of a matrix, as copied: one lane's word of row r.
template <typename T, int COPY>
struct LrRows {
    const uint32_t* words;
    uint32_t odd;  // LR_COPY_ODD: bit r: row r starts in the middle of a word
    __device__ __forceinline__ LrRows(const char* buf, const void* matrix, uint64_t offset, uint64_t stride)
        : words((const uint32_t*)buf + (threadIdx.x & 31)), odd(0) {
        if constexpr (COPY == LR_COPY_ODD) {
            odd = lr_odd_rows(matrix, offset, stride);
        }
    }
    __device__ __forceinline__ uint32_t operator[](int r) const {
        const uint32_t* w = words + r * (LrFetch<T, COPY>::PITCH / 4);
        if constexpr (COPY == LR_COPY_ODD) return __funnelshift_r(w[0], w[1], odd >> r & 1 ? 16 : 0);
        else return w[0];
    }
};

// One lane's word of a row: its channels widened, and narrowed again.
template <typename T> struct LrWord;
template <> struct LrWord<float> {
    static constexpr int N = 1;
    static __device__ __forceinline__ void widen(uint32_t w, float* v) { v[0] = __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t narrow(const float* v) { return __float_as_uint(v[0]); }
};
template <> struct LrWord<__half> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float* v) {
        __half2 h;
        memcpy(&h, &w, 4);
        const float2 f = __half22float2(h);
        v[0] = f.x, v[1] = f.y;
    }
    static __device__ __forceinline__ uint32_t narrow(const float* v) {
        const __half2 h = __floats2half2_rn(v[0], v[1]);
        uint32_t w;
        memcpy(&w, &h, 4);
        return w;
    }
};
template <> struct LrWord<__nv_bfloat16> {
    static constexpr int N = 2;
    static __device__ __forceinline__ void widen(uint32_t w, float* v) {
        v[0] = __uint_as_float(w << 16), v[1] = __uint_as_float(w & 0xffff0000u);
    }
    static __device__ __forceinline__ uint32_t narrow(const float* v) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
        uint32_t w;
        memcpy(&w, &h, 4);
        return w;
    }
};
// Stores one row, a lane its channels, `left` of them (if positive) in range.  A call of the whole warp; odd
// (LR_COPY_ODD): the row starts in the middle of a word, so that a lane's second and the next lane's first channel
// share one.
template <typename T, int COPY>
__device__ __forceinline__ void lr_store(T* p, const float* v, int left, bool odd) {
    const uint32_t w = LrWord<T>::narrow(v);
    if constexpr (COPY != LR_COPY_ODD) {
        if (left > 0) *(uint32_t*)p = w;
    } else {
        const uint32_t next = __shfl_down_sync(0xffffffffu, w, 1);
        const int lane = threadIdx.x & 31;
        uint16_t* h = (uint16_t*)p;
        if (odd) {
            if (lane == 0 && left > 0) h[0] = (uint16_t)w;
            if (left > 2 && lane < 31) *(uint32_t*)(h + 1) = __funnelshift_r(w, next, 16);
            else if (left > 1) h[1] = (uint16_t)(w >> 16);
        } else {
            if (left > 1) *(uint32_t*)h = w;
            else if (left > 0) h[0] = (uint16_t)w;
        }
    }
}
// What a kernel of this file knows about its tiles: CTA b takes tiles b, b + grid, ..., numbered along the
// channels first.  All CTAs of a chained launch are resident (a cooperative launch), so a tile may wait for the
// tiles before it wherever they are.
struct LrTiles {
    uint32_t row_tiles;
    LrDivisor col_tiles;
    const uint32_t* codes;  // of the rows (with offsets)
    bool narrow;            // many tiles of a column are under way at a time
    __device__ __forceinline__ uint32_t count() const {
        const uint32_t total = row_tiles * col_tiles.d;
        return blockIdx.x < total ? (total - blockIdx.x - 1) / gridDim.x + 1 : 0;
    }
    // Tile i of this CTA: its row tile, counted from the first (or last) one, and its column tile.
    __device__ __forceinline__ uint2 tile(uint32_t i) const {
        const uint32_t t = blockIdx.x + i * gridDim.x, k = col_tiles.div(t);
        return make_uint2(k, t - k * col_tiles.d);
    }
};
// Which warps of a CTA cut the chain, as bits, from one word each.
__device__ __forceinline__ uint32_t lr_cuts(const uint32_t* cut, uint32_t bit) {
    const int lane = threadIdx.x & 31;
    return __ballot_sync(0xffffffffu, lane < LR_WARPS && (cut[lane % LR_WARPS] & bit));
}

// What the compute warps have to know about a tile, worked out by a publishing warp a few tiles ahead: eight slots,
// of which tile i's is written before the arrival for the starts of tile i - 6 and read until tile i is finished.
struct alignas(16) LrSlot {
    uint64_t offset[5];      // of the tile in each matrix, in bytes
    uint32_t row, channel;   // its first
    uint32_t rows, channels; // that are in range
    uint32_t plain;          // a bit a warp: its rows are all inside a sequence (where all have one length)
    uint32_t pad;
};
constexpr int LR_SLOTS = 8, LR_AHEAD = 6;
static_assert(LR_SLOTS >= LR_AHEAD + 2, "a slot is rewritten after its tile is finished");

template <int M>
__device__ __forceinline__ void lr_slot(LrSlot& slot, const LrShape& sh, uint64_t row, uint64_t channel, uint32_t columns,
                                        int element, const uint64_t (&stride)[M]) {
    const int lane = threadIdx.x & 31;
    bool plain = false;
    if (!sh.offsets && lane < LR_WARPS) {
        const uint64_t first = row + lane * LR_ROWS;
        const uint32_t r = (uint32_t)first, at = r - sh.length.div(r) * sh.length.d;
        plain = at > 0 && at + LR_ROWS < sh.length.d && first + LR_ROWS <= sh.rows;
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, plain);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < M; ++i) slot.offset[i] = (row * stride[i] + channel) * element;
        slot.row = (uint32_t)row, slot.channel = (uint32_t)channel;
        slot.rows = (uint32_t)min(sh.rows - row, (uint64_t)LR_TILE);
        slot.channels = (uint32_t)min(sh.channels - channel, (uint64_t)columns);
        slot.plain = bits;
    }
}

// Asks for the states (C floats from `channel` on) of the sequences that begin (LR_HEAD) or end (LR_TAIL) in a warp's
// rows of the next tile, so that they will be found in L1: a warp that waits for them there holds up its whole CTA
// (backward, 32768 x 1536 f16 in 300 sequences: 176 us against 188 without).
template <int C>
__device__ __forceinline__ void lr_touch(const LrShape& sh, uint32_t code, uint32_t mark, const float* from, uint64_t stride,
                                         uint32_t channel) {
    if (!from) return;
    const int lane = threadIdx.x & 31;
    for (uint32_t rows = __ballot_sync(0xffffffffu, code & mark); rows; rows &= rows - 1) {
        const uint32_t s = __shfl_sync(0xffffffffu, code, __ffs(rows) - 1) & LR_SEQUENCE;
        const float* at = from + min((uint64_t)s, sh.sequences - 1) * stride + channel;
#pragma unroll
        for (int i = 0; i < C; i += 32)
            if (channel + i + lane < sh.channels) {
                float v;
                asm volatile("ld.global.ca.f32 %0, [%1];" : "=f"(v) : "l"(at + i + lane));
            }
    }
}

// The kernels are launched while lr_prepare_kernel runs: what reads the rows' codes or touches records waits for it.
__device__ __forceinline__ void lr_prepared() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- Forward ---------------------------------------------------------------------
// The maps keep both prefixes of every row in registers (pre, loc): outputs are
// one multiply-add each, and the gate is evaluated once.  Two tiles are held at
// a time.
template <typename T>
struct LrConfig {
    static constexpr int N = LrWord<T>::N;                 // channels a lane; publishing warps, and look-back warps
    static constexpr int C = 32 * N;                       // channels of a tile
    static constexpr int THREADS = (LR_WARPS + 2 * N) * 32;
    static constexpr int MAPPED = THREADS - 32 * N;        // of a barrier of the compute warps and one kind of helpers
};

template <typename T, int COPY>
struct LrForwardSmem {
    static constexpr int STAGES = 4, C = LrConfig<T>::C;
    char rows[STAGES][LR_WARPS][2][LrFetch<T, COPY>::BUF];  // gate, in
    uint32_t code[STAGES][LR_WARPS][LR_ROWS];
    float2 map[2][LR_WARPS][C];  // (A, H) of a warp's rows
    float start[2][LR_WARPS][C];
    uint32_t cut[2][LR_WARPS];   // nothing from before a warp's rows passes them
    LrSlot slot[LR_SLOTS];
};

template <typename T, int GATE, int COPY>
__global__ void __launch_bounds__(LrConfig<T>::THREADS, 1) lr_forward_kernel(LrForward p, LrChain ch, LrTiles tl) {
    using Config = LrConfig<T>;
    using Smem = LrForwardSmem<T, COPY>;
    constexpr int N = Config::N, C = Config::C;
    static_assert(Smem::STAGES + 2 <= LR_AHEAD, "tile i + STAGES is fetched after the starts of tile i - 2");
    extern __shared__ __align__(128) char smem_raw[];
    Smem& sm = *(Smem*)smem_raw;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    if (p.sh.offsets || warp >= LR_WARPS) lr_prepared();
    const uint32_t channels = (uint32_t)p.sh.channels, count = tl.count();

    const uint64_t strides[3] = {p.gate_stride, p.in_stride, p.out_stride};
    auto slot = [&](uint32_t i) {
        if (i >= count) return;
        const uint2 t = tl.tile(i);
        lr_slot(sm.slot[i % LR_SLOTS], p.sh, (uint64_t)t.x * LR_TILE, (uint64_t)t.y * C, C, sizeof(T), strides);
    };
    if (warp < LR_AHEAD) slot(warp);
    __syncthreads();

    if (warp >= LR_WARPS) {
        const bool publishes = warp >= LR_WARPS + N;
        const int cc = (warp - LR_WARPS) % N * 32 + lane;
        // the code of a tile's first row, read a tile ahead: nothing passes a head or enters outside a sequence
        auto first_code = [&](uint32_t i) -> uint32_t {
            const uint64_t row = (uint64_t)tl.tile(min(i, count - 1)).x * LR_TILE;
            return lr_code(p.sh, row, tl.codes + row);
        };
        uint32_t code = first_code(0);
        for (uint32_t i = 0; i < count; ++i) {
            const int b = i & 1;
            const uint2 t = tl.tile(i);
            const uint32_t k = t.x, c = t.y * C + cc;
            float4* record = ch.record + (uint64_t)k * ch.width + c;
            const bool active = c < channels, more = active && k + 1 < tl.row_tiles;
            const bool enters = !publishes && k > 0 && !(code & (LR_HEAD | LR_OUTSIDE));
            code = first_code(i + 1);
            float carry = 0.0f;
            if (enters) {
                const int64_t step = -(int64_t)ch.width;
                carry = tl.narrow ? lr_lookback<LR_FAR>(record + step, step, k, active)
                                  : lr_lookback<LR_NEAR>(record + step, step, k, active);
            }
            lr_sync((publishes ? 1 : 5) + b, Config::MAPPED);
            const uint32_t cuts = lr_cuts(sm.cut[b], 1);
            float A = 1.0f, H = 0.0f, a[LR_WARPS], h[LR_WARPS];
#pragma unroll
            for (int w = 0; w < LR_WARPS; ++w) {
                const float2 v = sm.map[b][w][cc];
                a[w] = v.x, h[w] = v.y;
                H = cuts >> w & 1 ? h[w] : fmaf(a[w], H, h[w]);
                A *= a[w];
            }
            if (publishes) {
                if (more) {
                    if (cuts || k == 0) lr_put_state(record, H);
                    else lr_put_map(record, A, H);
                }
                if (warp == LR_WARPS + N) slot(i + LR_AHEAD);
            } else {
                if (more && !cuts && k > 0) lr_put_state(record, fmaf(A, carry, H));
                if (p.saved && active) p.saved[(uint64_t)k * channels + c] = carry;
#pragma unroll
                for (int w = 0; w < LR_WARPS; ++w) {
                    sm.start[b][w][cc] = carry;
                    carry = cuts >> w & 1 ? h[w] : fmaf(a[w], carry, h[w]);
                }
            }
            lr_arrive(3 + b, Config::THREADS);
        }
        return;
    }

    const int column = lane * N;
    const LrFetch<T, COPY> fetch_gate(p.gate, p.gate_stride, warp, p.sh), fetch_in(p.in, p.in_stride, warp, p.sh);
    T* const out0 = (T*)p.out + (uint64_t)(warp * LR_ROWS) * p.out_stride + column;
    auto fetch = [&](uint32_t i) {
        if (i < count) {
            const uint32_t st = i % Smem::STAGES;
            const LrSlot& sl = sm.slot[i % LR_SLOTS];
            const int n = (int)sl.rows - warp * LR_ROWS;
            fetch_gate.copy(sm.rows[st][warp][0], sl.offset[0], n, sl.channels);
            fetch_in.copy(sm.rows[st][warp][1], sl.offset[1], n, sl.channels);
            if (p.sh.offsets && lane < min(n, LR_ROWS))
                cp_async4(&sm.code[st][warp][lane], tl.codes + sl.row + warp * LR_ROWS + lane);
        }
        cp_async_commit();
    };
    // The codes of this warp's rows of tile i (0 if it is known that none has a mark), a tile ahead of their use.
    auto codes_ahead = [&](uint32_t i) -> uint32_t {
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        if (i >= count || (sl.plain >> warp & 1) || lane >= LR_ROWS) return 0;
        const uint64_t row = (uint64_t)sl.row + warp * LR_ROWS + lane;
        return lr_code(p.sh, row, tl.codes + row);
    };
    uint32_t ahead = codes_ahead(1);
    // The marks of a warp's rows in a tile, and what the loops over the rows have to do about them.
    auto marks = [&](const LrSlot& sl, uint32_t st, int* kind) -> LrMarks {
        *kind = LR_PLAIN;
        if (sl.plain >> warp & 1) return LrMarks();
        const uint64_t row = (uint64_t)sl.row + warp * LR_ROWS + lane;
        const uint32_t code = lane < LR_ROWS ? lr_code(p.sh, row, &sm.code[st][warp][lane]) : 0;
        if (!__any_sync(0xffffffffu, code & (LR_OUTSIDE | LR_HEAD | LR_TAIL))) return LrMarks();
        const LrMarks m(code);
        *kind = m.kind();
        return m;
    };
    // The state of the sequence that begins (ends) in row r of a warp's rows: `from` [sequence][stride].
    auto edge = [&](const LrMarks& m, const LrSlot& sl, int r, const float* from, uint64_t stride, float* v) {
        const uint64_t s = m.sequence(p.sh, r);
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = from && column + i < sl.channels ? from[s * stride + sl.channel + column + i] : 0.0f;
    };
    struct Rows {  // a tile between its two halves: row r is h = pre h_before + loc
        float pre[LR_ROWS][N], loc[LR_ROWS][N];
        LrMarks m;
        int kind;
    };
    auto maps = [&](uint32_t i, Rows& w) {
        const uint32_t st = i % Smem::STAGES;
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        cp_async_wait_prior<Smem::STAGES - 1>();
        __syncwarp();
        w.m = marks(sl, st, &w.kind);
        const LrRows<T, COPY> gate(sm.rows[st][warp][0], p.gate, sl.offset[0], p.gate_stride),
            in(sm.rows[st][warp][1], p.in, sl.offset[1], p.in_stride);
        float A[N], H[N];
#pragma unroll
        for (int i = 0; i < N; ++i) A[i] = 1.0f, H[i] = 0.0f;
        auto rows = [&](auto tag) {
            constexpr int kind = decltype(tag)::value;
            const LrMarks& m = w.m;
            const int head = __ffs(m.head) - 1;
            float init[N];
            if (kind == LR_SINGLE && head >= 0) edge(m, sl, head, p.init, p.init_stride, init);
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r) {
                float g[N], x[N];
                LrWord<T>::widen(gate[r], g);
                LrWord<T>::widen(in[r], x);
                if (kind == LR_MANY) edge(m, sl, r, p.init, p.init_stride, init);
                if (kind == LR_SINGLE ? r == head : kind == LR_MANY && (m.head >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) A[i] = 0.0f, H[i] = init[i];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const Gate<GATE> gt(g[i]);
                    H[i] = fmaf(gt.a, H[i], gt.add(x[i]));
                    A[i] *= gt.a;
                }
                if (kind == LR_MANY && !(m.valid >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) A[i] = H[i] = 0.0f;
#pragma unroll
                for (int i = 0; i < N; ++i) w.pre[r][i] = A[i], w.loc[r][i] = H[i];
            }
        };
        if (w.kind == LR_PLAIN) rows(std::integral_constant<int, LR_PLAIN>{});
        else if (w.kind == LR_SINGLE) rows(std::integral_constant<int, LR_SINGLE>{});
        else rows(std::integral_constant<int, LR_MANY>{});
        const int b = i & 1;
#pragma unroll
        for (int i = 0; i < N; ++i) sm.map[b][warp][column + i] = make_float2(A[i], H[i]);
        if (lane == 0) sm.cut[b][warp] = w.m.cuts();
        lr_arrive(1 + b, Config::MAPPED);
        lr_arrive(5 + b, Config::MAPPED);
        __syncwarp();  // the stage is read
        fetch(i + Smem::STAGES);
        if (__any_sync(0xffffffffu, ahead & (LR_HEAD | LR_TAIL)))
            lr_touch<C>(p.sh, ahead, LR_HEAD, p.init, p.init_stride, sm.slot[(i + 1) % LR_SLOTS].channel);
        ahead = codes_ahead(i + 2);
    };
    auto finish = [&](uint32_t i, const Rows& w) {
        const int b = i & 1;
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        const int left = (int)sl.channels - column;
        T* out = (T*)((char*)out0 + sl.offset[2]);
        const uint32_t odd = COPY == LR_COPY_ODD ? lr_odd_rows(p.out, sl.offset[2], p.out_stride) : 0;
        float start[N];
        lr_sync(3 + b, Config::THREADS);
#pragma unroll
        for (int i = 0; i < N; ++i) start[i] = sm.start[b][warp][column + i];
        if (w.kind == LR_PLAIN) {
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r, out += p.out_stride) {
                float h[N];
#pragma unroll
                for (int i = 0; i < N; ++i) h[i] = fmaf(w.pre[r][i], start[i], w.loc[r][i]);
                lr_store<T, COPY>(out, h, left, odd >> r & 1);
            }
            return;
        }
        // From the first head or outside row on nothing depends on the state before the warp's rows (not even as 0
        // times it, which an infinity or NaN of another sequence would survive).
        const LrMarks& m = w.m;
        const int rows = (int)sl.rows - warp * LR_ROWS;
        const int reach = __ffs(m.head | ~m.valid) - 1;
#pragma unroll
        for (int r = 0; r < LR_ROWS; ++r, out += p.out_stride) {
            float h[N];
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = r < reach ? fmaf(w.pre[r][i], start[i], w.loc[r][i]) : w.loc[r][i];
            if (r < rows) lr_store<T, COPY>(out, h, left, odd >> r & 1);
            if ((m.tail >> r & 1) && p.last) {
                float* last = p.last + m.sequence(p.sh, r) * channels + sl.channel + column;
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < left) last[i] = h[i];
            }
        }
    };
#pragma unroll
    for (int i = 0; i < Smem::STAGES; ++i) fetch(i);
    Rows even, odd;  // the maps of tile i + 1, then the outputs of tile i
    if (count > 0) maps(0, even);
    for (uint32_t i = 0; i < count; i += 2) {
        if (i + 1 < count) maps(i + 1, odd);
        finish(i, even);
        if (i + 2 < count) maps(i + 2, even);
        if (i + 1 < count) finish(i + 1, odd);
    }
    cp_async_wait_all();
}

// ---- Backward --------------------------------------------------------------------
// Tiles from the last to the first: the chain carries mu, mu_before = A mu_behind + M.
// The maps need the gates of a tile once for both directions; its rows stay in
// shared memory and the gates are evaluated again for the gradients (4 of the
// special function unit's operations an element, 58 % of its rate at the copy
// rate), since keeping them would take three registers an element.
template <typename T, int COPY>
struct LrBackwardSmem {
    static constexpr int STAGES = 3, C = LrConfig<T>::C;
    char rows[STAGES][LR_WARPS][3][LrFetch<T, COPY>::BUF];  // gate, in, grad_out
    uint32_t code[STAGES][LR_WARPS][LR_ROWS];
    float2 map[2][LR_WARPS][C];                   // (A, H) of a warp's rows, and M
    float grad_map[2][LR_WARPS][C];
    float start[2][LR_WARPS][C], grad_start[2][LR_WARPS][C];
    // bit 0: no state from before a warp's rows passes them; bit 1: no gradient from behind them does
    uint32_t cut[2][LR_WARPS];
    LrSlot slot[LR_SLOTS];
};

template <typename T, int GATE, int COPY>
__global__ void __launch_bounds__(LrConfig<T>::THREADS, 1) lr_backward_kernel(LrBackward p, LrChain ch, LrTiles tl) {
    using Config = LrConfig<T>;
    using Smem = LrBackwardSmem<T, COPY>;
    constexpr int N = Config::N, C = Config::C;
    static_assert(Smem::STAGES <= LR_AHEAD, "tile i + STAGES is fetched after the starts of tile i");
    extern __shared__ __align__(128) char smem_raw[];
    Smem& sm = *(Smem*)smem_raw;
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    if (p.sh.offsets || warp >= LR_WARPS) lr_prepared();
    const uint32_t channels = (uint32_t)p.sh.channels, count = tl.count();
    auto row_tile = [&](uint2 t) { return tl.row_tiles - 1 - t.x; };

    const uint64_t strides[5] = {p.gate_stride, p.in_stride, p.grad_out_stride, p.grad_gate_stride, p.grad_in_stride};
    auto slot = [&](uint32_t i) {
        if (i >= count) return;
        const uint2 t = tl.tile(i);
        lr_slot(sm.slot[i % LR_SLOTS], p.sh, (uint64_t)row_tile(t) * LR_TILE, (uint64_t)t.y * C, C, sizeof(T), strides);
    };
    if (warp < LR_AHEAD) slot(warp);
    __syncthreads();

    if (warp >= LR_WARPS) {
        const bool publishes = warp >= LR_WARPS + N;
        const int cc = (warp - LR_WARPS) % N * 32 + lane;
        // the code of a tile's last row, read a tile ahead: nothing passes a tail or enters outside a sequence
        auto last_code = [&](uint32_t i) -> uint32_t {
            const uint64_t row = (uint64_t)(tl.row_tiles - tl.tile(min(i, count - 1)).x) * LR_TILE - 1;
            return lr_code(p.sh, row, tl.codes + row);
        };
        uint32_t code = last_code(0);
        for (uint32_t i = 0; i < count; ++i) {
            const int b = i & 1;
            const uint2 t = tl.tile(i);
            const uint32_t k = row_tile(t), c = t.y * C + cc;
            float4* record = ch.record + (uint64_t)k * ch.width + c;
            const bool active = c < channels, more = active && k > 0, chained = k + 1 < tl.row_tiles;
            // the publishing warps also carry the states on, from the saved one
            float carry = 0.0f, state = publishes && active ? p.saved[(uint64_t)k * channels + c] : 0.0f;
            const bool enters = !publishes && chained && !(code & (LR_TAIL | LR_OUTSIDE));
            code = last_code(i + 1);
            if (enters) {
                const int64_t step = ch.width;
                carry = tl.narrow ? lr_lookback<LR_FAR>(record + step, step, t.x, active)
                                  : lr_lookback<LR_NEAR>(record + step, step, t.x, active);
            }
            lr_sync((publishes ? 1 : 5) + b, Config::MAPPED);
            const uint32_t cuts = lr_cuts(sm.cut[b], 2);
            float A = 1.0f, M = 0.0f, a[LR_WARPS], v[LR_WARPS];
#pragma unroll
            for (int w = LR_WARPS - 1; w >= 0; --w) {
                a[w] = sm.map[b][w][cc].x, v[w] = sm.grad_map[b][w][cc];
                M = cuts >> w & 1 ? v[w] : fmaf(a[w], M, v[w]);
                A *= a[w];
            }
            if (publishes) {
                if (more) {
                    if (cuts || !chained) lr_put_state(record, M);
                    else lr_put_map(record, A, M);
                }
                if (warp == LR_WARPS + N) slot(i + LR_AHEAD);
                const uint32_t heads = lr_cuts(sm.cut[b], 1);
#pragma unroll
                for (int w = 0; w < LR_WARPS; ++w) {
                    sm.start[b][w][cc] = state;
                    const float h = sm.map[b][w][cc].y;
                    state = heads >> w & 1 ? h : fmaf(a[w], state, h);
                }
            } else {
                if (more && !cuts && chained) lr_put_state(record, fmaf(A, carry, M));
#pragma unroll
                for (int w = LR_WARPS - 1; w >= 0; --w) {
                    sm.grad_start[b][w][cc] = carry;
                    carry = cuts >> w & 1 ? v[w] : fmaf(a[w], carry, v[w]);
                }
            }
            lr_arrive(3 + b, Config::THREADS);
        }
        return;
    }

    const int column = lane * N;
    const LrFetch<T, COPY> fetch_gate(p.gate, p.gate_stride, warp, p.sh), fetch_in(p.in, p.in_stride, warp, p.sh),
        fetch_grad(p.grad_out, p.grad_out_stride, warp, p.sh);
    const uint64_t bottom = warp * LR_ROWS + LR_ROWS - 1;  // the warp's last row
    T* const out_gate0 = (T*)p.grad_gate + bottom * p.grad_gate_stride + column;
    T* const out_in0 = (T*)p.grad_in + bottom * p.grad_in_stride + column;
    auto fetch = [&](uint32_t i) {
        if (i < count) {
            const uint32_t st = i % Smem::STAGES;
            const LrSlot& sl = sm.slot[i % LR_SLOTS];
            const int n = (int)sl.rows - warp * LR_ROWS;
            fetch_gate.copy(sm.rows[st][warp][0], sl.offset[0], n, sl.channels);
            fetch_in.copy(sm.rows[st][warp][1], sl.offset[1], n, sl.channels);
            if (p.grad_out) fetch_grad.copy(sm.rows[st][warp][2], sl.offset[2], n, sl.channels);
            if (p.sh.offsets && lane < min(n, LR_ROWS))
                cp_async4(&sm.code[st][warp][lane], tl.codes + sl.row + warp * LR_ROWS + lane);
        }
        cp_async_commit();
    };
    // The codes of this warp's rows of tile i (0 if it is known that none has a mark), a tile ahead of their use.
    auto codes_ahead = [&](uint32_t i) -> uint32_t {
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        if (i >= count || (sl.plain >> warp & 1) || lane >= LR_ROWS) return 0;
        const uint64_t row = (uint64_t)sl.row + warp * LR_ROWS + lane;
        return lr_code(p.sh, row, tl.codes + row);
    };
    uint32_t ahead = codes_ahead(1);
    // The marks of a warp's rows in a tile, and what the loops over the rows have to do about them.
    auto marks = [&](const LrSlot& sl, uint32_t st, int* kind) -> LrMarks {
        *kind = LR_PLAIN;
        if (sl.plain >> warp & 1) return LrMarks();
        const uint64_t row = (uint64_t)sl.row + warp * LR_ROWS + lane;
        const uint32_t code = lane < LR_ROWS ? lr_code(p.sh, row, &sm.code[st][warp][lane]) : 0;
        if (!__any_sync(0xffffffffu, code & (LR_OUTSIDE | LR_HEAD | LR_TAIL))) return LrMarks();
        const LrMarks m(code);
        *kind = m.kind();
        return m;
    };
    // The state of the sequence that begins (ends) in row r of a warp's rows: `from` [sequence][stride].
    auto edge = [&](const LrMarks& m, const LrSlot& sl, int r, const float* from, uint64_t stride, float* v) {
        const uint64_t s = m.sequence(p.sh, r);
#pragma unroll
        for (int i = 0; i < N; ++i)
            v[i] = from && column + i < sl.channels ? from[s * stride + sl.channel + column + i] : 0.0f;
    };
    if (!p.grad_out) {  // zeros that stay
        for (int st = 0; st < Smem::STAGES; ++st)
            for (int j = lane; j < LrFetch<T, COPY>::BUF / 4; j += 32) ((uint32_t*)sm.rows[st][warp][2])[j] = 0;
        __syncwarp();
    }
    auto maps = [&](uint32_t i) -> int {
        const uint32_t st = i % Smem::STAGES;
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        cp_async_wait_prior<Smem::STAGES - 2>();
        __syncwarp();
        int what;
        const LrMarks m = marks(sl, st, &what);
        const LrRows<T, COPY> gate(sm.rows[st][warp][0], p.gate, sl.offset[0], p.gate_stride),
            in(sm.rows[st][warp][1], p.in, sl.offset[1], p.in_stride),
            grad(sm.rows[st][warp][2], p.grad_out, sl.offset[2], p.grad_out_stride);
        float A[N], H[N], M[N];
#pragma unroll
        for (int i = 0; i < N; ++i) A[i] = 1.0f, H[i] = 0.0f, M[i] = 0.0f;
        auto rows = [&](auto tag) {
            constexpr int kind = decltype(tag)::value;
            float a[LR_ROWS][N], init[N], last[N];
            const int head = __ffs(m.head) - 1, tail = __ffs(m.tail) - 1;
            if (kind == LR_SINGLE && head >= 0) edge(m, sl, head, p.init, p.init_stride, init);
            if (kind == LR_SINGLE && tail >= 0) edge(m, sl, tail, p.grad_last, channels, last);
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r) {
                float g[N], x[N];
                LrWord<T>::widen(gate[r], g);
                LrWord<T>::widen(in[r], x);
                if (kind == LR_MANY) edge(m, sl, r, p.init, p.init_stride, init);
                if (kind == LR_SINGLE ? r == head : kind == LR_MANY && (m.head >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) H[i] = init[i];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const Gate<GATE> gt(g[i]);
                    a[r][i] = gt.a;
                    H[i] = fmaf(gt.a, H[i], gt.add(x[i]));
                    A[i] *= gt.a;
                }
            }
#pragma unroll
            for (int r = LR_ROWS - 1; r >= 0; --r) {
                float v[N];
                LrWord<T>::widen(grad[r], v);
                if (kind == LR_MANY) edge(m, sl, r, p.grad_last, channels, last);
                if (kind == LR_SINGLE ? r == tail : kind == LR_MANY && (m.tail >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) M[i] = last[i];
#pragma unroll
                for (int i = 0; i < N; ++i) M[i] = a[r][i] * (v[i] + M[i]);
                if (kind == LR_MANY && !(m.valid >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) M[i] = 0.0f;
            }
        };
        if (what == LR_PLAIN) rows(std::integral_constant<int, LR_PLAIN>{});
        else if (what == LR_SINGLE) rows(std::integral_constant<int, LR_SINGLE>{});
        else rows(std::integral_constant<int, LR_MANY>{});
        const int b = i & 1;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            sm.map[b][warp][column + i] = make_float2(A[i], H[i]);
            sm.grad_map[b][warp][column + i] = M[i];
        }
        if (lane == 0) sm.cut[b][warp] = (m.cuts() ? 1u : 0u) | (m.cuts_back() ? 2u : 0u);
        lr_arrive(1 + b, Config::MAPPED);
        lr_arrive(5 + b, Config::MAPPED);
        if (__any_sync(0xffffffffu, ahead & (LR_HEAD | LR_TAIL))) {
            const uint32_t channel = sm.slot[(i + 1) % LR_SLOTS].channel;
            lr_touch<C>(p.sh, ahead, LR_HEAD, p.init, p.init_stride, channel);
            lr_touch<C>(p.sh, ahead, LR_TAIL, p.grad_last, channels, channel);
        }
        ahead = codes_ahead(i + 2);
        return what;
    };
    auto finish = [&](uint32_t i, int what) {
        const int b = i & 1;
        const uint32_t st = i % Smem::STAGES;
        const LrSlot& sl = sm.slot[i % LR_SLOTS];
        const int left = (int)sl.channels - column;
        const LrMarks m = what == LR_PLAIN ? LrMarks() : marks(sl, st, &what);
        const LrRows<T, COPY> gate(sm.rows[st][warp][0], p.gate, sl.offset[0], p.gate_stride),
            in(sm.rows[st][warp][1], p.in, sl.offset[1], p.in_stride),
            grad(sm.rows[st][warp][2], p.grad_out, sl.offset[2], p.grad_out_stride);
        T* out_gate = (T*)((char*)out_gate0 + sl.offset[3]);
        T* out_in = (T*)((char*)out_in0 + sl.offset[4]);
        const uint32_t odd_gate = COPY == LR_COPY_ODD ? lr_odd_rows(p.grad_gate, sl.offset[3], p.grad_gate_stride) : 0;
        auto keep = [&](int r, const float* v) {  // the gradient of the initial state
            if (!p.grad_init) return;
            float* to = p.grad_init + m.sequence(p.sh, r) * channels + sl.channel + column;
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) to[i] = v[i];
        };
        const uint32_t odd_in = COPY == LR_COPY_ODD ? lr_odd_rows(p.grad_in, sl.offset[4], p.grad_in_stride) : 0;
        auto rows = [&](auto tag) {
            constexpr int kind = decltype(tag)::value;
            float h[N], mu[N], a[LR_ROWS][N], na[LR_ROWS][N], dgate[LR_ROWS][N];  // dgate: of the gate, per unit of lam
            float init[N], last[N], first[N] = {};
            const int head = __ffs(m.head) - 1, tail = __ffs(m.tail) - 1;
            if (kind == LR_SINGLE && head >= 0) edge(m, sl, head, p.init, p.init_stride, init);
            if (kind == LR_SINGLE && tail >= 0) edge(m, sl, tail, p.grad_last, channels, last);
            const int n = kind == LR_MANY ? (int)sl.rows - warp * LR_ROWS : LR_ROWS;
            lr_sync(3 + b, Config::THREADS);
#pragma unroll
            for (int i = 0; i < N; ++i) h[i] = sm.start[b][warp][column + i], mu[i] = sm.grad_start[b][warp][column + i];
#pragma unroll
            for (int r = 0; r < LR_ROWS; ++r) {
                float g[N], x[N];
                LrWord<T>::widen(gate[r], g);
                LrWord<T>::widen(in[r], x);
                if (kind == LR_MANY) edge(m, sl, r, p.init, p.init_stride, init);
                if (kind == LR_SINGLE ? r == head : kind == LR_MANY && (m.head >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) h[i] = init[i];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const Gate<GATE> gt(g[i]);
                    a[r][i] = gt.a, na[r][i] = gt.na;
                    dgate[r][i] = gt.grad_gate(h[i], x[i]);
                    h[i] = fmaf(gt.a, h[i], gt.add(x[i]));
                }
            }
#pragma unroll
            for (int r = LR_ROWS - 1; r >= 0; --r, out_gate -= p.grad_gate_stride, out_in -= p.grad_in_stride) {
                float v[N], dg[N], dx[N];
                LrWord<T>::widen(grad[r], v);
                if (kind == LR_MANY) edge(m, sl, r, p.grad_last, channels, last);
                if (kind == LR_SINGLE ? r == tail : kind == LR_MANY && (m.tail >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) mu[i] = last[i];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float lam = v[i] + mu[i];
                    dg[i] = lam * dgate[r][i];
                    dx[i] = GATE == LCPP_GATE_SIGMOID ? na[r][i] * lam : lam;
                    mu[i] = a[r][i] * lam;
                }
                if (kind == LR_MANY && !(m.valid >> r & 1))
#pragma unroll
                    for (int i = 0; i < N; ++i) dg[i] = dx[i] = mu[i] = 0.0f;
                if (r < n) {
                    lr_store<T, COPY>(out_gate, dg, left, odd_gate >> r & 1);
                    lr_store<T, COPY>(out_in, dx, left, odd_in >> r & 1);
                }
                if (kind == LR_SINGLE)
#pragma unroll
                    for (int i = 0; i < N; ++i) first[i] = r == head ? mu[i] : first[i];
                if (kind == LR_MANY && (m.head >> r & 1)) keep(r, mu);
            }
            if (kind == LR_SINGLE && head >= 0) keep(head, first);
        };
        if (what == LR_PLAIN) rows(std::integral_constant<int, LR_PLAIN>{});
        else if (what == LR_SINGLE) rows(std::integral_constant<int, LR_SINGLE>{});
        else rows(std::integral_constant<int, LR_MANY>{});
        __syncwarp();  // the stage is read
        fetch(i + Smem::STAGES);
    };
#pragma unroll
    for (int i = 0; i < Smem::STAGES; ++i) fetch(i);
    int kind = LR_PLAIN, before = LR_PLAIN;
    for (uint32_t i = 0; i <= count; ++i, before = kind) {  // each compiled once: the instruction cache counts here
        if (i < count) kind = maps(i);
        if (i > 0) finish(i - 1, before);
    }
    cp_async_wait_all();
}

// ---- Before a chained or packed call ------------------------------------------------
// The chain's words become LR_NONE, the rows get their codes (with offsets, a
// warp a tile), and sequences without rows pass their state on, to[s] = from[s]
// (0 without from).
__global__ void __launch_bounds__(128)
lr_prepare_kernel(uint4* words, uint64_t count, uint32_t* codes, LrShape sh, const float* from, uint64_t from_stride, float* to) {
    __shared__ uint32_t s_code[4][LR_TILE];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint64_t i = (uint64_t)blockIdx.x * 128 + threadIdx.x; i < count; i += (uint64_t)gridDim.x * 128)
        words[i] = make_uint4(LR_NONE, LR_NONE, LR_NONE, LR_NONE);
    if (sh.offsets) {
        const uint64_t S = sh.sequences, tiles = (sh.rows + LR_TILE - 1) / LR_TILE;
        for (uint64_t k = (uint64_t)blockIdx.x * 4 + warp; k < tiles; k += (uint64_t)gridDim.x * 4) {
            const uint64_t first = k * LR_TILE, end = min(first + LR_TILE, sh.rows);
            const uint64_t lo = sh.offsets[0], hi = sh.offsets[S];
            const int64_t base = max(lr_search(sh.offsets, S + 1, first), (int64_t)0);
            for (int r = lane; r < LR_TILE; r += 32) s_code[warp][r] = first + r >= lo && first + r < hi ? 0 : LR_OUTSIDE;
            __syncwarp();
            for (uint64_t i = base;; i += 32) {
                const uint64_t s = i + lane;
                uint64_t begin = ~0ull, stop = 0;
                if (s < S) begin = sh.offsets[s], stop = min((uint64_t)sh.offsets[s + 1], sh.rows);
                if (begin < stop) {
                    if (begin >= first && begin < end) atomicOr(&s_code[warp][begin - first], LR_HEAD | (uint32_t)s);
                    if (stop > first && stop <= end) atomicOr(&s_code[warp][stop - 1 - first], LR_TAIL | (uint32_t)s);
                }
                if (__any_sync(0xffffffffu, begin >= end)) break;
            }
            __syncwarp();
            for (int r = lane; r < (int)(end - first); r += 32) codes[first + r] = s_code[warp][r];
            __syncwarp();
        }
    }
    if (!to) return;
    for (uint64_t s = blockIdx.x; s < sh.sequences; s += gridDim.x) {
        if (sh.offsets ? min((uint64_t)sh.offsets[s], sh.rows) < min((uint64_t)sh.offsets[s + 1], sh.rows) : sh.length.d > 0)
            continue;
        for (uint64_t c = threadIdx.x; c < sh.channels; c += 128)
            to[s * sh.channels + c] = from ? from[s * from_stride + c] : 0.0f;
    }
}

// ---- One token ---------------------------------------------------------------------
// Row i continues the state of row parents[i] (itself without parents; zero for
// a negative parent).  Bound by the bytes (2048 x 4096 bf16: 18.5 us, 97 % of the
// copy rate); a warp takes U x 32 vectors of V channels of a row, so that enough
// loads are under way at any alignment.
constexpr int LR_STEP_WARPS = 4;

template <typename T, int V>
struct alignas(V * sizeof(T)) LrVector {
    T v[V];
};

template <typename T, int GATE, int V, int U>
__global__ void __launch_bounds__(LR_STEP_WARPS * 32)
lr_step_kernel(const T* gate, uint64_t gate_stride, const T* in, uint64_t in_stride, const float* states_in,
               uint32_t rows_in, const int32_t* parents, float* states_out, T* out, uint64_t out_stride,
               uint32_t rows, uint32_t channels, uint32_t parts) {
    constexpr int VS = V > 4 ? 4 : V;  // states a load
    using Vector = LrVector<T, V>;
    using States = LrVector<float, VS>;
    const uint32_t unit = blockIdx.x * LR_STEP_WARPS + (threadIdx.x >> 5), r = unit / parts;
    if (r >= rows) return;
    const uint32_t c0 = (unit - r * parts) * (32 * V * U) + (threadIdx.x & 31) * V;
    int64_t from = parents ? (int64_t)parents[r] : (int64_t)r;
    Vector g[U], x[U];
    States h[U][V / VS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t c = c0 + u * 32 * V;
        if (c < channels) {
            g[u] = *(const Vector*)(gate + r * gate_stride + c);
            x[u] = *(const Vector*)(in + r * in_stride + c);
        }
    }
    if (!states_in) {
        from = -1;
    } else if (from >= (int64_t)rows_in) {
        set_error(LCPP_ERR_INVALID_ARG);
        from = -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V / VS; ++j) {
            const uint32_t c = c0 + u * 32 * V;
#pragma unroll
            for (int i = 0; i < VS; ++i) h[u][j].v[i] = 0.0f;
            if (from >= 0 && c < channels) h[u][j] = *(const States*)(states_in + from * channels + c + j * VS);
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t c = c0 + u * 32 * V;
        if (c >= channels) break;
        Vector y;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float& s = h[u][i / VS].v[i % VS];
            const Gate<GATE> gt(widen(g[u].v[i]));
            s = fmaf(gt.a, s, gt.add(widen(x[u].v[i])));
            y.v[i] = narrow<T>(s);
        }
#pragma unroll
        for (int j = 0; j < V / VS; ++j) *(States*)(states_out + (uint64_t)r * channels + c + j * VS) = h[u][j];
        if (out) *(Vector*)(out + r * out_stride + c) = y;
    }
}

constexpr uint64_t LR_MAX_ROWS = 0xffffffffull;  // offsets are 32-bit
constexpr uint64_t LR_MAX_CHANNELS = 1ull << 20;

static lcpp_status lr_check(int gate, int dtype, const LrShape& sh, const void* gate_in, const void* in) {
    if ((gate != LCPP_GATE_LINEAR && gate != LCPP_GATE_SIGMOID) || !is_float_dtype(dtype)) return LCPP_ERR_INVALID_ARG;
    if (sh.rows > LR_MAX_ROWS || sh.channels > LR_MAX_CHANNELS || sh.sequences > LR_SEQUENCE) return LCPP_ERR_INVALID_ARG;
    if (!sh.offsets && sh.sequences * sh.length.d != sh.rows) return LCPP_ERR_INVALID_ARG;
    if (sh.rows && sh.channels && (!gate_in || !in || (!sh.sequences && !sh.offsets))) return LCPP_ERR_INVALID_ARG;
    return LCPP_OK;
}
// A row stride must reach past the channels (one row may have any).
static bool lr_stride_ok(uint64_t stride, uint64_t rows, uint64_t channels) {
    return rows <= 1 || (stride >= channels && stride < (1ull << 31));
}

// Temp: [row codes u32][records: row tiles x width float4].
static uint64_t lr_width(uint64_t channels) { return align_up(channels, 64); }
static size_t lr_chain_bytes(uint64_t rows, uint64_t channels) {
    const uint64_t tiles = ceil_div(rows, LR_TILE);
    return tiles > 1 ? tiles * lr_width(channels) * 16 : 0;
}
static size_t lr_code_bytes(uint64_t rows) { return align_up(rows * 4, 256); }
static LrChain lr_chain(void* temp, uint64_t rows, uint64_t channels) {
    return LrChain{(float4*)((char*)temp + lr_code_bytes(rows)), lr_width(channels)};
}

// The operands' memory.  Tiles read and write at different times, so an output may be an input only where each element
// is written by the lane that has read it: in the same place of the matrix.
static Region lr_scratch(const LrShape& sh, const void* temp) {
    return Region(temp, lr_code_bytes(sh.rows) + lr_chain_bytes(sh.rows, sh.channels));
}
static Region lr_matrix(const void* p, const LrShape& sh, uint64_t stride, uint64_t element) {
    return Region(p, sh.rows, stride * element, sh.channels * element);
}
static Region lr_states(const float* p, const LrShape& sh, uint64_t stride) {
    return Region(p, stride ? sh.sequences : 1, stride * 4, sh.channels * 4);
}
static Region lr_offsets(const LrShape& sh) { return Region(sh.offsets, (sh.sequences + 1) * 4); }
static Region lr_saved(const void* p, const LrShape& sh) { return Region(p, ceil_div(sh.rows, LR_TILE) * sh.channels * 4); }

// How the rows of these matrices can be copied.
struct LrCopy {
    uint64_t bits;  // all addresses and byte strides or-ed together
    LrCopy(uint64_t channels, size_t e) : bits(channels * e) {}
    LrCopy& add(const void* p, uint64_t stride, size_t e) {
        bits |= (uint64_t)(uintptr_t)p | stride * e;
        return *this;
    }
    int kind() const { return bits % 16 == 0 ? LR_COPY16 : bits % 4 == 0 ? LR_COPY4 : LR_COPY_ODD; }
};

static lcpp_status lr_prepare(const LrShape& sh, void* temp, const float* from, uint64_t from_stride, float* to,
                              bool* prepared, cudaStream_t s) {
    const uint64_t words = lr_chain_bytes(sh.rows, sh.channels) / 16;
    if (!sh.offsets && sh.length.d) to = nullptr;  // no sequence is empty
    *prepared = words || to || sh.offsets;
    if (!*prepared) return LCPP_OK;
    uint64_t grid = max(ceil_div(words, 128 * 4), to ? min(sh.sequences, (uint64_t)1024) : 1);
    if (sh.offsets) grid = max(grid, ceil_div(ceil_div(sh.rows, LR_TILE), 4));
    ProfScope prof("lr_prepare", s);
    lr_prepare_kernel<<<(unsigned)min(grid, (uint64_t)device_info().sms * 16), 128, 0, s>>>(
        (uint4*)lr_chain(temp, sh.rows, sh.channels).record, words, (uint32_t*)temp, sh, from, from_stride, to);
    count_launch();
    return check_launch();
}

// Launches KERNEL over all tiles.
template <typename T, auto KERNEL, typename P>
static lcpp_status lr_launch(size_t smem, const char* name, const P& p, const LrShape& sh, void* temp, bool prepared,
                             cudaStream_t s) {
    const uint64_t row_tiles = ceil_div(sh.rows, LR_TILE), col_tiles = ceil_div(sh.channels, LrConfig<T>::C);
    if (row_tiles * col_tiles > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    const DeviceInfo device = device_info();
    const uint64_t grid = min(row_tiles * col_tiles, (uint64_t)device.sms);
    const LrTiles tl{(uint32_t)row_tiles, LrDivisor(col_tiles), (const uint32_t*)temp, grid > LR_NEAR * col_tiles};
    static std::atomic<uint64_t> sized{0};  // devices on which the kernel may have this much shared memory
    const uint64_t bit = 1ull << device.device;
    if (!(sized.load(std::memory_order_relaxed) & bit)) {
        if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return check_launch();
        sized.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchAttribute how[2];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(LrConfig<T>::THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = how;
    if (row_tiles > 1) {  // tiles wait for one another
        how[cfg.numAttrs].id = cudaLaunchAttributeCooperative;
        how[cfg.numAttrs++].val.cooperative = 1;
    }
    if (prepared) {  // launched while lr_prepare_kernel runs
        how[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        how[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    ProfScope prof(name, s);
    if (cudaLaunchKernelEx(&cfg, KERNEL, p, lr_chain(temp, sh.rows, sh.channels), tl) != cudaSuccess) return check_launch();
    count_launch();
    return LCPP_OK;
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
    return max(lr_code_bytes(rows) + lr_chain_bytes(rows, channels), (size_t)256);
}

extern "C" size_t lcpp_linear_recurrence_saved_bytes(uint64_t rows, uint64_t channels) {
    return align_up(ceil_div(rows, LR_TILE) * channels * sizeof(float), 256);  // a state per tile
}

extern "C" lcpp_status lcpp_linear_recurrence_forward(
    int gate, int dtype, const void* gate_in, uint64_t gate_stride, const void* in, uint64_t in_stride, void* out,
    uint64_t out_stride, uint64_t rows, uint64_t channels, uint64_t num_sequences, uint64_t length,
    const uint32_t* offsets, const float* init, uint64_t init_stride, float* last, void* saved, void* temp,
    size_t temp_bytes, void* stream) {
    if (!offsets && length > LR_MAX_ROWS) return LCPP_ERR_INVALID_ARG;
    const LrShape sh{rows, channels, num_sequences, LrDivisor(offsets ? 0 : length), offsets};
    const lcpp_status ok = lr_check(gate, dtype, sh, gate_in, in);
    if (ok != LCPP_OK) return ok;
    if (!channels || (!num_sequences && !rows)) return LCPP_OK;
    if (!num_sequences) init = nullptr, last = nullptr;  // all rows are padding, and no state exists
    if (!elements_aligned(dtype, gate_in, in, out) || !elements_aligned(LCPP_F32, offsets, init, last, saved))
        return LCPP_ERR_INVALID_ARG;
    if (rows && (!out || !lr_stride_ok(gate_stride, rows, channels) || !lr_stride_ok(in_stride, rows, channels) ||
                 !lr_stride_ok(out_stride, rows, channels)))
        return LCPP_ERR_INVALID_ARG;
    if (!temp || temp_bytes < lcpp_linear_recurrence_temp_bytes(rows, channels)) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % sizeof(float4)) return LCPP_ERR_INVALID_ARG;
    const uint64_t e = dtype == LCPP_F32 ? 4 : 2;
    const Region rg = lr_matrix(gate_in, sh, gate_stride, e), ri = lr_matrix(in, sh, in_stride, e),
                 ro = lr_matrix(out, sh, out_stride, e), r0 = lr_states(init, sh, init_stride),
                 rl = lr_states(last, sh, channels), rs = lr_saved(saved, sh), rt = lr_scratch(sh, temp),
                 rf = lr_offsets(sh);
    if (!ro.apart_or_same(rg, ri) || !ro.apart(r0, rl, rs, rt, rf) || !rl.apart_or_same(r0) ||
        !rl.apart(rg, ri, rs, rt, rf) || !rs.apart(rg, ri, r0, rt, rf) || !rt.apart(rg, ri, r0, rf))
        return LCPP_ERR_INVALID_ARG;
    const LrForward p{sh, gate_in, in, out, gate_stride, in_stride, out_stride, init_stride, init, last, (float*)saved};
    cudaStream_t s = (cudaStream_t)stream;
    bool prepared = false;
    const lcpp_status ready = lr_prepare(sh, temp, init, init_stride, last, &prepared, s);
    if (ready != LCPP_OK || !rows) return ready;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        constexpr int G = decltype(g)::value;
        const int copy = LrCopy(channels, sizeof(T)).add(gate_in, gate_stride, sizeof(T)).add(in, in_stride, sizeof(T))
                             .add(out, out_stride, sizeof(T)).kind();
        auto launch = [&](auto c) {
            constexpr int COPY = decltype(c)::value;
            return lr_launch<T, lr_forward_kernel<T, G, COPY>>(sizeof(LrForwardSmem<T, COPY>), "lr_forward", p, sh, temp, prepared, s);
        };
        if (copy == LR_COPY16) return launch(std::integral_constant<int, LR_COPY16>{});
        if constexpr (sizeof(T) == 2) {
            if (copy == LR_COPY_ODD) return launch(std::integral_constant<int, LR_COPY_ODD>{});
        }
        return launch(std::integral_constant<int, LR_COPY4>{});
    });
}

extern "C" lcpp_status lcpp_linear_recurrence_backward(
    int gate, int dtype, const void* gate_in, uint64_t gate_stride, const void* in, uint64_t in_stride,
    const void* saved, const float* init, uint64_t init_stride, const void* grad_out, uint64_t grad_out_stride,
    const float* grad_last, void* grad_gate, uint64_t grad_gate_stride, void* grad_in, uint64_t grad_in_stride,
    float* grad_init, uint64_t rows, uint64_t channels, uint64_t num_sequences, uint64_t length,
    const uint32_t* offsets, void* temp, size_t temp_bytes, void* stream) {
    if (!offsets && length > LR_MAX_ROWS) return LCPP_ERR_INVALID_ARG;
    const LrShape sh{rows, channels, num_sequences, LrDivisor(offsets ? 0 : length), offsets};
    const lcpp_status ok = lr_check(gate, dtype, sh, gate_in, in);
    if (ok != LCPP_OK) return ok;
    if (!channels || (!num_sequences && !rows)) return LCPP_OK;
    if (!num_sequences) init = grad_last = nullptr, grad_init = nullptr;
    if (!elements_aligned(dtype, gate_in, in, grad_out, grad_gate, grad_in) ||
        !elements_aligned(LCPP_F32, saved, offsets, init, grad_last, grad_init))
        return LCPP_ERR_INVALID_ARG;
    if (rows && (!saved || !grad_gate || !grad_in || !lr_stride_ok(gate_stride, rows, channels) ||
                 !lr_stride_ok(in_stride, rows, channels) || !lr_stride_ok(grad_gate_stride, rows, channels) ||
                 !lr_stride_ok(grad_in_stride, rows, channels) ||
                 (grad_out && !lr_stride_ok(grad_out_stride, rows, channels))))
        return LCPP_ERR_INVALID_ARG;
    if (!temp || temp_bytes < lcpp_linear_recurrence_temp_bytes(rows, channels)) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % sizeof(float4)) return LCPP_ERR_INVALID_ARG;
    const uint64_t e = dtype == LCPP_F32 ? 4 : 2;
    const Region rg = lr_matrix(gate_in, sh, gate_stride, e), ri = lr_matrix(in, sh, in_stride, e),
                 ro = lr_matrix(grad_out, sh, grad_out_stride, e), rgg = lr_matrix(grad_gate, sh, grad_gate_stride, e),
                 rgi = lr_matrix(grad_in, sh, grad_in_stride, e), r0 = lr_states(init, sh, init_stride),
                 rl = lr_states(grad_last, sh, channels), rg0 = lr_states(grad_init, sh, channels),
                 rs = lr_saved(saved, sh), rt = lr_scratch(sh, temp), rf = lr_offsets(sh);
    if (!rgg.apart_or_same(rg, ri, ro) || !rgg.apart(rgi, r0, rl, rg0, rs, rt, rf) || !rgi.apart_or_same(rg, ri, ro) ||
        !rgi.apart(r0, rl, rg0, rs, rt, rf) || !rg0.apart_or_same(r0) || !rg0.apart(rg, ri, ro, rl, rs, rt, rf) ||
        !rt.apart(rg, ri, ro, r0, rl, rs, rf))
        return LCPP_ERR_INVALID_ARG;
    const LrBackward p{sh, gate_in, in, grad_out, grad_gate, grad_in, gate_stride, in_stride, grad_out_stride,
                       grad_gate_stride, grad_in_stride, init_stride, init, grad_last, (const float*)saved, grad_init};
    cudaStream_t s = (cudaStream_t)stream;
    bool prepared = false;
    const lcpp_status ready = lr_prepare(sh, temp, grad_last, channels, grad_init, &prepared, s);
    if (ready != LCPP_OK || !rows) return ready;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        constexpr int G = decltype(g)::value;
        LrCopy align(channels, sizeof(T));
        align.add(gate_in, gate_stride, sizeof(T)).add(in, in_stride, sizeof(T))
            .add(grad_gate, grad_gate_stride, sizeof(T)).add(grad_in, grad_in_stride, sizeof(T));
        if (grad_out) align.add(grad_out, grad_out_stride, sizeof(T));
        const int copy = align.kind();
        auto launch = [&](auto c) {
            constexpr int COPY = decltype(c)::value;
            return lr_launch<T, lr_backward_kernel<T, G, COPY>>(sizeof(LrBackwardSmem<T, COPY>), "lr_backward", p, sh, temp, prepared, s);
        };
        if (copy == LR_COPY16) return launch(std::integral_constant<int, LR_COPY16>{});
        if constexpr (sizeof(T) == 2) {
            if (copy == LR_COPY_ODD) return launch(std::integral_constant<int, LR_COPY_ODD>{});
        }
        return launch(std::integral_constant<int, LR_COPY4>{});
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
    if (!elements_aligned(dtype, gate_in, in, out) || !elements_aligned(LCPP_F32, states_in, parents, states_out))
        return LCPP_ERR_INVALID_ARG;
    if (states_in && !parents && rows_in < rows) return LCPP_ERR_INVALID_ARG;
    const uint64_t e = dtype == LCPP_F32 ? 4 : 2;
    const Region rg(gate_in, rows, gate_stride * e, channels * e), ri(in, rows, in_stride * e, channels * e),
        ro(out, rows, out_stride * e, channels * e), rn(states_out, rows, channels * 4, channels * 4),
        rs(states_in, parents ? rows_in : rows, channels * 4, channels * 4), rp(parents, rows * 4);
    if (!rn.apart_or_same(rg, ri, ro) || !rn.apart(rp) || !ro.apart_or_same(rg, ri) || !ro.apart(rp))
        return LCPP_ERR_INVALID_ARG;
    // with parents a row may be read after another row's new state took its place
    if (parents ? !rs.apart(rn, ro) : !rs.apart_or_same(rn, ro)) return LCPP_ERR_INVALID_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    return lr_dispatch(gate, dtype, [&](auto t, auto g) -> lcpp_status {
        using T = decltype(t);
        constexpr int G = decltype(g)::value, WIDE = 16 / sizeof(T);
        // the widest vectors that every row of every operand is a whole number of
        uint64_t bits = (uint64_t)(uintptr_t)gate_in | (uint64_t)(uintptr_t)in | (uint64_t)(uintptr_t)out;
        if (rows > 1) bits |= (gate_stride | in_stride | (out ? out_stride : 0)) * sizeof(T);
        const uint64_t states = (uint64_t)(uintptr_t)states_in | (uint64_t)(uintptr_t)states_out;
        auto fits = [&](int v) { return channels % v == 0 && bits % (v * sizeof(T)) == 0 && states % (v > 4 ? 16 : v * 4) == 0; };
        auto launch = [&](auto kernel, int span) -> lcpp_status {
            const uint64_t parts = ceil_div(channels, span), units = parts * rows;
            if (ceil_div(units, LR_STEP_WARPS) > 0x3fffffffull) return LCPP_ERR_INVALID_ARG;
            ProfScope prof("lr_step", s);
            kernel<<<(unsigned)ceil_div(units, LR_STEP_WARPS), LR_STEP_WARPS * 32, 0, s>>>(
                (const T*)gate_in, gate_stride, (const T*)in, in_stride, states_in, (uint32_t)rows_in, parents, states_out,
                (T*)out, out_stride, (uint32_t)rows, (uint32_t)channels, (uint32_t)parts);
            count_launch();
            return check_launch();
        };
        if (fits(WIDE)) return launch(lr_step_kernel<T, G, WIDE, 1>, 32 * WIDE);
        if (fits(2)) return launch(lr_step_kernel<T, G, 2, 2>, 32 * 2 * 2);
        return launch(lr_step_kernel<T, G, 1, 4>, 32 * 4);
    });
}
