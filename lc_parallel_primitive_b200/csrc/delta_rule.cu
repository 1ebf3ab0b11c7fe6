// Gated delta rule (DeviceDeltaRule): forward over sequences by chunks of 64 rows, its backward pass, and the
// single-token step.  Per sequence and head, with the state S of value_dim x key_dim and a_t = exp(decay_t):
//
//   S' = a_t S_{t-1},  u_t = beta_t (v_t - S' k_t),  S_t = S' + u_t k_t^T,  o_t = scale S_t q_t
//
// Within a chunk that starts from S0, with g_i = a_1 ... a_i, D_ij = g_i / g_j (j <= i), e_j = g_64 / g_j and
//   N_ij = D_ij k_i.k_j (j < i),  A_ij = scale D_ij q_i.k_j (j <= i):
//   w = (I + N B)^-1 (V - g K S0^T),  u = B w                (B = diag(beta); w and u have a row per token)
//   O = scale g Q S0^T + A u,  S_64 = g_64 S0 + sum_j e_j u_j k_j^T
// Backward, X the gradient of S_64:
//   du = A^T dO + e K X^T,  z = (I + B N)^-T du,  y = B z = dV,  dbeta_j = w_j.z_j
//   dS0 = g_64 X + sum_i (scale g_i dO_i q_i^T - g_i y_i k_i^T)
//   dA = dO u^T, dN = -y u^T (masked);  dq = scale g dO S0 + scale (D dA) K
//   dk = erase + write,  erase = (D dN) K - g y S0,  write = e u X + scale (D dA)^T Q + (D dN)^T K
//   the gradient of log g_i is q_i.dq_i + k_i.erase_i - k_i.write_i, and that of log g_64 has sum_j e_j k_j.(u_j X) +
//   g_64 <S0, X> besides; ddecay_t sums them from t to the chunk's end.
//
// dr_prepare_kernel computes, for all chunks at once, what does not depend on the state: A, the inverse, and the decays.
// dr_forward_kernel and dr_backward_kernel go through a sequence's chunks in order with the state (its gradient) in
// registers: a warp owns 16 of the value dimensions, for which the recurrence needs nothing of any other warp, and the
// accumulators of one product are the operands of the next.  dr_gradient_kernel is parallel over chunks again.
//
// Products are of bf16 with float32 sums.  A float32 value enters as the sum of two bf16 (16 bits, 2^-18) in as many
// products as that takes, so that states, which live for a whole sequence, keep float32's order of error; bf16 inputs
// are exact as they are, float16 and float32 ones are split the same way (dr_pack_kernel).
#include "float_types.cuh"
#include "warp_mma.cuh"

namespace lcpp {

constexpr int DR_CHUNK = 64;
constexpr int DR_MAX_DIM = 128;
constexpr int DR_TILE = DR_CHUNK * DR_CHUNK;  // elements of a chunk's square matrices
constexpr float DR_LEAST_DECAY = -150.0f;     // exp of less is 0 in float32 anyway, and -inf has no differences

struct DrShape {
    uint64_t rows, length;
    const uint32_t* offsets;
    uint32_t sequences, heads, key_heads, key_dim, value_dim;
    float scale;
    __device__ __forceinline__ uint64_t start(uint32_t s) const { return offsets ? offsets[s] : s * length; }
    // Chunks have slots, base(s) of a sequence's first: as many as there are rows / 64 before it, and one more for each
    // sequence before it, are always enough.
    __device__ __forceinline__ uint64_t base(uint32_t s) const { return start(s) / DR_CHUNK + s; }
};
// The chunk in a slot: its first row and how many of its rows exist (0: none).
struct DrChunk {
    uint64_t row;
    uint32_t rows, sequence;
    __device__ __forceinline__ DrChunk(const DrShape& sh, uint64_t slot) : row(0), rows(0), sequence(0) {
        uint32_t lo = 0, hi = sh.sequences;  // the last sequence whose base is not past the slot
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (sh.base(mid) <= slot) lo = mid;
            else hi = mid;
        }
        sequence = lo;
        const uint64_t from = sh.start(lo), to = min(sh.start(lo + 1), sh.rows), base = sh.base(lo);
        if (slot < base) return;
        row = from + (slot - base) * DR_CHUNK;
        if (row < to) rows = (uint32_t)min((uint64_t)DR_CHUNK, to - row);
    }
};

// A matrix [rows][heads][dim] as bf16: the caller's own, or two planes by slot (64 rows each, zeros where there are none).
struct DrOperand {
    const __nv_bfloat16* at;
    uint64_t row;    // elements from a row to the next
    uint64_t plane;
    uint32_t head;   // and from a head to the next
    uint32_t dim;    // columns to read, a multiple of 8
    bool packed;
    __device__ __forceinline__ const __nv_bfloat16* rows(uint64_t slot, const DrChunk& c, uint32_t h) const {
        return at + (packed ? slot * DR_CHUNK : c.row) * row + (uint64_t)h * head;
    }
    __device__ __forceinline__ int have(const DrChunk& c) const { return packed ? DR_CHUNK : (int)c.rows; }
};

// What dr_prepare_kernel writes by slot and head.
struct DrPrepared {
    __nv_bfloat16 *inverse, *read;  // two planes of 64 x 64: (I + N B)^-1 or (I + B N)^-1, and A
    float* gates;                   // g, e, beta (64 each)
    __device__ __forceinline__ uint64_t at(const DrShape& sh, uint64_t slot, uint32_t h) const { return slot * sh.heads + h; }
};
// Matrices of two planes by slot and head: states [value_dim][key columns], values [value_dim][64].
struct DrPlanes {
    __nv_bfloat16* at;
    uint64_t size;  // elements of one plane
    __device__ __forceinline__ __nv_bfloat16* of(const DrShape& sh, uint64_t slot, uint32_t h) const {
        return at + (slot * sh.heads + h) * 2 * size;
    }
};

// ---- operands in two planes ---------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
dr_pack_kernel(DrShape sh, const T* from, uint64_t from_stride, uint32_t heads, uint32_t dim, __nv_bfloat16* to, uint64_t plane,
               uint32_t pitch) {
    const uint64_t slot = blockIdx.x;
    const DrChunk c(sh, slot);
    const uint32_t words = heads * pitch / 2;
    for (uint32_t i = threadIdx.x; i < DR_CHUNK * words; i += blockDim.x) {
        const uint32_t r = i / words, w = i % words, h = w * 2 / pitch, d = w * 2 % pitch;
        float x = 0.0f, y = 0.0f;
        if (r < c.rows) {
            const T* const p = from + (c.row + r) * from_stride + (uint64_t)h * dim + d;
            if (d < dim) x = widen(p[0]);
            if (d + 1 < dim) y = widen(p[1]);
        }
        uint32_t hi, lo;
        split_bf16(x, y, hi, lo);
        uint32_t* const at = (uint32_t*)(to + (slot * DR_CHUNK + r) * (uint64_t)heads * pitch) + w;
        at[0] = hi;
        *(uint32_t*)((__nv_bfloat16*)at + plane) = lo;
    }
}

// ---- what does not depend on the state ------------------------------------------------------------
constexpr int DR_PREPARE_THREADS = 128;
constexpr int DR_PITCH = DR_CHUNK + 1;
template <int DK, int PLANES>
struct DrPrepareSmem {
    __nv_bfloat16 k[PLANES][DR_CHUNK * DK], q[PLANES][DR_CHUNK * DK];
    float near[DR_CHUNK * DR_PITCH], read[DR_CHUNK * DR_PITCH];  // k_i.k_j and q_i.k_j
    float m[DR_CHUNK * DR_PITCH], inv[DR_CHUNK * DR_PITCH], tmp[32 * 33];
    double total[DR_CHUNK];
    float beta[DR_CHUNK];
};

// inv = (I + m)^-1 of a strictly lower triangular m: the 16 x 16 blocks of the diagonal by substitution, a column a
// lane, then blocks below from ones above: [X 0; -Y m21 X, Y].
template <typename S>
__device__ __forceinline__ void dr_invert(S& s) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (lane < 16) {
        const int b = warp * 16;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v = i == lane ? 1.0f : 0.0f;
#pragma unroll
            for (int k = 0; k < i; ++k) v = fmaf(-s.m[(b + i) * DR_PITCH + b + k], x[k], v);
            x[i] = v;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s.inv[(b + i) * DR_PITCH + b + lane] = x[i];
    }
    for (int i = t; i < DR_CHUNK * DR_CHUNK; i += DR_PREPARE_THREADS) {  // above the diagonal blocks
        const int r = i >> 6, c = i & 63;
        if ((c >> 4) > (r >> 4)) s.inv[r * DR_PITCH + c] = 0.0f;
    }
    __syncthreads();
    {
        const int b = (t >> 6) * 32, r = (t & 63) >> 2, c = (t & 3) * 4;  // blocks (16, 0) and (48, 32)
        float v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float a = s.m[(b + 16 + r) * DR_PITCH + b + k];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(a, s.inv[(b + k) * DR_PITCH + b + c + j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s.tmp[((t >> 6) * 16 + r) * 33 + c + j] = v[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const float a = s.inv[(b + 16 + r) * DR_PITCH + b + 16 + k];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = fmaf(a, s.tmp[((t >> 6) * 16 + k) * 33 + c + j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s.inv[(b + 16 + r) * DR_PITCH + b + c + j] = -v[j];
    }
    __syncthreads();
    {
        const int r = t >> 2, c = (t & 3) * 8;  // block (32, 0)
        float v[8] = {};
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
            const float a = s.m[(32 + r) * DR_PITCH + k];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = fmaf(a, s.inv[k * DR_PITCH + c + j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s.tmp[r * 33 + c + j] = v[j];
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
            const float a = s.inv[(32 + r) * DR_PITCH + 32 + k];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = fmaf(a, s.tmp[k * 33 + c + j], v[j]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) s.inv[(32 + r) * DR_PITCH + c + j] = -v[j];
    }
    __syncthreads();
}

template <int DK, int PLANES, bool BACKWARD>
__global__ void __launch_bounds__(DR_PREPARE_THREADS)
dr_prepare_kernel(DrShape sh, DrOperand q, DrOperand k, const float* decay, uint64_t decay_stride, const float* beta,
                  uint64_t beta_stride, DrPrepared to) {
    extern __shared__ __align__(128) uint8_t dr_smem[];
    using Smem = DrPrepareSmem<DK, PLANES>;
    Smem& s = *(Smem*)dr_smem;
    const uint64_t slot = blockIdx.x / sh.key_heads;
    const uint32_t hk = blockIdx.x % sh.key_heads, group = sh.heads / sh.key_heads;
    const DrChunk c(sh, slot);
    if (!c.rows) return;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    uint32_t kt[PLANES], qt[PLANES];
#pragma unroll
    for (int p = 0; p < PLANES; ++p) {
        kt[p] = smem_u32(s.k[p]), qt[p] = smem_u32(s.q[p]);
        tile_load<DK>(kt[p], k.rows(slot, c, hk) + p * k.plane, k.row, DR_CHUNK, k.have(c), k.dim, t, DR_PREPARE_THREADS);
        tile_load<DK>(qt[p], q.rows(slot, c, hk) + p * q.plane, q.row, DR_CHUNK, q.have(c), q.dim, t, DR_PREPARE_THREADS);
    }
    cp_async_commit();
    cp_async_wait_all();
    __syncthreads();
    {
        float nr[8][4] = {}, rd[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t ak[PLANES][4], aq[PLANES][4];
#pragma unroll
            for (int p = 0; p < PLANES; ++p) load_a<DK>(ak[p], kt[p], warp * 16, kk * 2, lane), load_a<DK>(aq[p], qt[p], warp * 16, kk * 2, lane);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (n > warp) break;  // columns past the warp's rows are masked
                uint32_t b[4];
                load_b<DK>(b, kt[0], n * 16, kk * 2, lane);
#pragma unroll
                for (int p = 0; p < PLANES; ++p) {
                    mma_bf16(nr[2 * n], ak[p], b[0], b[1]), mma_bf16(nr[2 * n + 1], ak[p], b[2], b[3]);
                    mma_bf16(rd[2 * n], aq[p], b[0], b[1]), mma_bf16(rd[2 * n + 1], aq[p], b[2], b[3]);
                }
                if constexpr (PLANES == 2) {
                    load_b<DK>(b, kt[1], n * 16, kk * 2, lane);
                    mma_bf16(nr[2 * n], ak[0], b[0], b[1]), mma_bf16(nr[2 * n + 1], ak[0], b[2], b[3]);
                    mma_bf16(rd[2 * n], aq[0], b[0], b[1]), mma_bf16(rd[2 * n + 1], aq[0], b[2], b[3]);
                }
            }
        }
        const int r = warp * 16 + (lane >> 2), col = (lane & 3) * 2;
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = (r + (j >> 1) * 8) * DR_PITCH + n * 8 + col + (j & 1);
                s.near[at] = nr[n][j], s.read[at] = rd[n][j];
            }
    }
    for (uint32_t h = hk * group; h < (hk + 1) * group; ++h) {
        __syncthreads();
        const uint64_t at = to.at(sh, slot, h);
        float* const gates = to.gates + at * 3 * DR_CHUNK;
        if (warp == 0) {  // running sums of the decays, in 64 bits: differences of long sums matter
            double v[2];
            float b[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = lane * 2 + j;
                float d = r < c.rows && decay ? decay[(c.row + r) * decay_stride + h] : 0.0f;
                d = d < DR_LEAST_DECAY ? DR_LEAST_DECAY : d;
                v[j] = d;
                b[j] = r < c.rows ? beta[(c.row + r) * beta_stride + h] : 0.0f;
            }
            double sum = v[0] + v[1];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            const double last = __shfl_sync(0xffffffffu, sum, 31);
            const double g[2] = {sum - v[1], sum};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = lane * 2 + j;
                s.total[r] = g[j], s.beta[r] = b[j];
                gates[r] = expf((float)g[j]), gates[DR_CHUNK + r] = expf((float)(last - g[j])), gates[2 * DR_CHUNK + r] = b[j];
            }
        }
        __syncthreads();
        __nv_bfloat16* const read = to.read + at * 2 * DR_TILE;
        for (int i = t; i < DR_TILE / 2; i += DR_PREPARE_THREADS) {
            const int r = i >> 5, c0 = (i & 31) * 2;
            float rd[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = c0 + j;
                const float d = col <= r ? expf((float)(s.total[r] - s.total[col])) : 0.0f;
                const float n = col < r ? d * s.near[r * DR_PITCH + col] * s.beta[BACKWARD ? r : col] : 0.0f;
                s.m[r * DR_PITCH + col] = n;
                rd[j] = col <= r ? sh.scale * d * s.read[r * DR_PITCH + col] : 0.0f;
            }
            uint32_t hi, lo;
            split_bf16(rd[0], rd[1], hi, lo);
            ((uint32_t*)read)[i] = hi;
            ((uint32_t*)(read + DR_TILE))[i] = lo;
        }
        __syncthreads();
        dr_invert(s);
        __nv_bfloat16* const inverse = to.inverse + at * 2 * DR_TILE;
        for (int i = t; i < DR_TILE / 2; i += DR_PREPARE_THREADS) {
            const int r = i >> 5, c0 = (i & 31) * 2;
            uint32_t hi, lo;
            split_bf16(s.inv[r * DR_PITCH + c0], s.inv[r * DR_PITCH + c0 + 1], hi, lo);
            ((uint32_t*)inverse)[i] = hi;
            ((uint32_t*)(inverse + DR_TILE))[i] = lo;
        }
    }
}

// ---- chunk after chunk ----------------------------------------------------------------------------
// Rows [row, row + 2) x ... of a fragment's element pairs, to a matrix of two planes with `pitch` columns.
__device__ __forceinline__ void dr_store_planes(__nv_bfloat16* to, uint64_t plane, int pitch, int row, int col, float x, float y) {
    uint32_t hi, lo;
    split_bf16(x, y, hi, lo);
    __nv_bfloat16* const at = to + row * pitch + col;
    *(uint32_t*)at = hi;
    *(uint32_t*)(at + plane) = lo;
}

template <int DK, int PLANES, int WARPS>
struct DrChainStage {
    __nv_bfloat16 k[PLANES][DR_CHUNK * DK], q[PLANES][DR_CHUNK * DK];
    __nv_bfloat16 v[PLANES][DR_CHUNK * (WARPS > 4 ? 128 : 64)];  // V forward, dO backward: the CTA's columns
    __nv_bfloat16 inverse[2][DR_TILE], read[2][DR_TILE];
    float gates[3][DR_CHUNK];
};
template <int DK, int PLANES, int WARPS>
struct DrChainSmem {
    DrChainStage<DK, PLANES, WARPS> stage[2];
};

struct DrChain {
    DrShape sh;
    DrOperand q, k, v;  // v: dO in the backward pass
    DrPrepared prepared;
    const float* from;  // states before the first chunk (forward), gradients of the last ones (backward)
    float* to;          // the states after; gradients of the first
    void* out;          // forward
    uint64_t out_stride;
    DrPlanes states, values;  // S0 and w (forward, if saved), X and z (backward)
    uint32_t key_cols;        // columns of a saved state, key_dim up to a multiple of 16
};

template <int DK, int PLANES, int WARPS>
__device__ __forceinline__ void dr_load(DrChainStage<DK, PLANES, WARPS>& st, const DrChain& p, const DrChunk& c, uint64_t slot,
                                        uint32_t h, uint32_t hk, uint32_t v0, int t) {
    constexpr int THREADS = WARPS * 32, VC = WARPS > 4 ? 128 : 64;
#pragma unroll
    for (int i = 0; i < PLANES; ++i) {
        tile_load<DK>(smem_u32(st.k[i]), p.k.rows(slot, c, hk) + i * p.k.plane, p.k.row, DR_CHUNK, p.k.have(c), p.k.dim, t, THREADS);
        tile_load<DK>(smem_u32(st.q[i]), p.q.rows(slot, c, hk) + i * p.q.plane, p.q.row, DR_CHUNK, p.q.have(c), p.q.dim, t, THREADS);
        if (p.v.at)
            tile_load<VC>(smem_u32(st.v[i]), p.v.rows(slot, c, h) + i * p.v.plane + v0, p.v.row, DR_CHUNK, p.v.have(c),
                          (int)p.v.dim - (int)v0, t, THREADS);
    }
    const uint64_t at = p.prepared.at(p.sh, slot, h);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        tile_load<64>(smem_u32(st.inverse[i]), p.prepared.inverse + (at * 2 + i) * DR_TILE, 64, 64, 64, 64, t, THREADS);
        tile_load<64>(smem_u32(st.read[i]), p.prepared.read + (at * 2 + i) * DR_TILE, 64, 64, 64, 64, t, THREADS);
    }
    for (int i = t; i < 3 * DR_CHUNK / 4; i += THREADS)
        cp_async16(&st.gates[0][0] + i * 4, p.prepared.gates + at * 3 * DR_CHUNK + i * 4);
}

// The state's 16 rows of this warp, from or to float32 [value_dim][key_dim].
template <int NT>
__device__ __forceinline__ void dr_state_in(float (&s)[NT][4], const float* from, uint32_t row, uint32_t rows, uint32_t cols, int col) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = row + (j >> 1) * 8, c = n * 8 + col + (j & 1);
            s[n][j] = from && r < rows && c < cols ? from[(uint64_t)r * cols + c] : 0.0f;
        }
}
template <int NT>
__device__ __forceinline__ void dr_state_out(const float (&s)[NT][4], float* to, uint32_t row, uint32_t rows, uint32_t cols, int col) {
    if (!to) return;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = row + (j >> 1) * 8, c = n * 8 + col + (j & 1);
            if (r < rows && c < cols) to[(uint64_t)r * cols + c] = s[n][j];
        }
}

// c (16 x 64: value x token) += s (16 x DK) K^T
template <int DK, int PLANES>
__device__ __forceinline__ void dr_times_keys(float (&c)[8][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                              const uint32_t (&k)[PLANES], int kk, int lane) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        uint32_t b[4];
        load_b<DK>(b, k[0], n * 16, kk * 2, lane);
        mma_bf16(c[2 * n], hi, b[0], b[1]), mma_bf16(c[2 * n + 1], hi, b[2], b[3]);
        mma_bf16(c[2 * n], lo, b[0], b[1]), mma_bf16(c[2 * n + 1], lo, b[2], b[3]);
        if constexpr (PLANES == 2) {
            load_b<DK>(b, k[PLANES - 1], n * 16, kk * 2, lane);
            mma_bf16(c[2 * n], hi, b[0], b[1]), mma_bf16(c[2 * n + 1], hi, b[2], b[3]);
        }
    }
}
// s (16 x DK) += a (16 x 16 tokens: hi + lo) times rows [16 kt, 16 kt + 16) of a tile of keys or queries
template <int DK, int PLANES>
__device__ __forceinline__ void dr_add_outer(float (&s)[DK / 8][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4],
                                             const uint32_t (&tile)[PLANES], int kt, int lane) {
#pragma unroll
    for (int n = 0; n < DK / 16; ++n) {
        uint32_t b[4];
        load_b_t<DK>(b, tile[0], kt * 16, n * 2, lane);
        mma_bf16(s[2 * n], hi, b[0], b[1]), mma_bf16(s[2 * n + 1], hi, b[2], b[3]);
        mma_bf16(s[2 * n], lo, b[0], b[1]), mma_bf16(s[2 * n + 1], lo, b[2], b[3]);
        if constexpr (PLANES == 2) {
            load_b_t<DK>(b, tile[PLANES - 1], kt * 16, n * 2, lane);
            mma_bf16(s[2 * n], hi, b[0], b[1]), mma_bf16(s[2 * n + 1], hi, b[2], b[3]);
        }
    }
}

template <typename T>
__device__ __forceinline__ void dr_store_pair(T* to, uint32_t col, uint32_t cols, bool even, float x, float y) {
    if (even && col + 1 < cols) {
        if constexpr (sizeof(T) == 4) *(float2*)(to + col) = make_float2(x, y);
        else if constexpr (std::is_same_v<T, __half>) *(__half2*)(to + col) = __floats2half2_rn(x, y);
        else *(__nv_bfloat162*)(to + col) = __floats2bfloat162_rn(x, y);
    } else {
        if (col < cols) to[col] = narrow<T>(x);
        if (col + 1 < cols) to[col + 1] = narrow<T>(y);
    }
}

template <typename T, int DK, int PLANES, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1)
dr_forward_kernel(const __grid_constant__ DrChain p) {
    constexpr int NT = DK / 8, VC = WARPS > 4 ? 128 : 64;
    extern __shared__ __align__(128) uint8_t dr_smem[];
    auto& smem = *(DrChainSmem<DK, PLANES, WARPS>*)dr_smem;
    const uint32_t slices = (p.sh.value_dim + WARPS * 16 - 1) / (WARPS * 16);
    const uint32_t slice = blockIdx.x % slices, h = blockIdx.x / slices % p.sh.heads, seq = blockIdx.x / slices / p.sh.heads;
    const uint32_t hk = h / (p.sh.heads / p.sh.key_heads), v0 = slice * WARPS * 16;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, col = (lane & 3) * 2;
    const uint32_t row = v0 + warp * 16 + g;  // of the state: the thread's first
    const uint64_t start = p.sh.start(seq), end = min(p.sh.start(seq + 1), p.sh.rows), base = p.sh.base(seq);
    const uint32_t chunks = end > start ? (uint32_t)((end - start + DR_CHUNK - 1) / DR_CHUNK) : 0;
    const uint64_t state = ((uint64_t)seq * p.sh.heads + h) * p.sh.value_dim * p.sh.key_dim;
    float s[NT][4];
    dr_state_in<NT>(s, p.from ? p.from + state : nullptr, row, p.sh.value_dim, p.sh.key_dim, col);
    DrChunk c(p.sh, base);
    auto chunk = [&](uint32_t i) {
        c.row = start + (uint64_t)i * DR_CHUNK;
        c.rows = (uint32_t)min((uint64_t)DR_CHUNK, end - c.row);
        return c;
    };
    if (chunks) dr_load(smem.stage[0], p, chunk(0), base, h, hk, v0, t);
    cp_async_commit();
    T* const out = (T*)p.out;
    const bool even = ((uintptr_t)out | p.out_stride * sizeof(T) | p.sh.value_dim * sizeof(T)) % (2 * sizeof(T)) == 0;
    for (uint32_t i = 0; i < chunks; ++i) {
        if (i + 1 < chunks) dr_load(smem.stage[(i + 1) & 1], p, chunk(i + 1), base + i + 1, h, hk, v0, t);
        cp_async_commit();
        cp_async_wait_prior1();
        __syncthreads();
        const DrChunk now = chunk(i);
        auto& st = smem.stage[i & 1];
        uint32_t k[PLANES], q[PLANES];
#pragma unroll
        for (int j = 0; j < PLANES; ++j) k[j] = smem_u32(st.k[j]), q[j] = smem_u32(st.q[j]);
        const uint32_t inv[2] = {smem_u32(st.inverse[0]), smem_u32(st.inverse[1])},
                       rd[2] = {smem_u32(st.read[0]), smem_u32(st.read[1])};
        __nv_bfloat16* const saved = p.states.at ? p.states.of(p.sh, base + i, h) : nullptr;
        // r = S0 K^T (value x token) and o = Q S0^T (token x value)
        float r[8][4] = {}, o[4][2][4] = {};
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t hi[4], lo[4];
            split_block(s[2 * kk], s[2 * kk + 1], hi, lo);
            if (saved) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t rr = row + (j & 1) * 8, cc = kk * 16 + (j >> 1) * 8 + col;
                    if (rr < p.sh.value_dim && cc < p.key_cols) {
                        __nv_bfloat16* const at = saved + rr * p.key_cols + cc;
                        *(uint32_t*)at = hi[j];
                        *(uint32_t*)(at + p.states.size) = lo[j];
                    }
                }
            }
            dr_times_keys<DK, PLANES>(r, hi, lo, k, kk, lane);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                uint32_t a[4];
                load_a<DK>(a, q[0], m * 16, kk * 2, lane);
                mma_bf16(o[m][0], a, hi[0], hi[2]), mma_bf16(o[m][1], a, hi[1], hi[3]);
                mma_bf16(o[m][0], a, lo[0], lo[2]), mma_bf16(o[m][1], a, lo[1], lo[3]);
                if constexpr (PLANES == 2) {
                    load_a<DK>(a, q[PLANES - 1], m * 16, kk * 2, lane);
                    mma_bf16(o[m][0], a, hi[0], hi[2]), mma_bf16(o[m][1], a, hi[1], hi[3]);
                }
            }
        }
        // r = V - g S0 K^T
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            uint32_t v[PLANES][4];
#pragma unroll
            for (int j = 0; j < PLANES; ++j) load_a_t<VC>(v[j], smem_u32(st.v[j]), n * 16, warp * 2, lane);
#pragma unroll
            for (int x = 0; x < 4; ++x) {  // fragment register x: rows g + 8 (x & 1), tokens 16 n + 8 (x >> 1) + col
                const float2 gate = *(const float2*)&st.gates[0][n * 16 + (x >> 1) * 8 + col];
                float v0 = bf16_low(v[0][x]), v1 = bf16_high(v[0][x]);
                if constexpr (PLANES == 2) v0 += bf16_low(v[PLANES - 1][x]), v1 += bf16_high(v[PLANES - 1][x]);
                float* const d = &r[2 * n + (x >> 1)][(x & 1) * 2];
                d[0] = fmaf(-gate.x, d[0], v0), d[1] = fmaf(-gate.y, d[1], v1);
            }
        }
        // w = r inverse^T
        float w[8][4] = {};
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(r[2 * kt], r[2 * kt + 1], hi, lo);
#pragma unroll
            for (int n = kt; n < 4; ++n) {
                uint32_t b[4];
                load_b<64>(b, inv[0], n * 16, kt * 2, lane);
                mma_bf16(w[2 * n], hi, b[0], b[1]), mma_bf16(w[2 * n + 1], hi, b[2], b[3]);
                mma_bf16(w[2 * n], lo, b[0], b[1]), mma_bf16(w[2 * n + 1], lo, b[2], b[3]);
                load_b<64>(b, inv[1], n * 16, kt * 2, lane);
                mma_bf16(w[2 * n], hi, b[0], b[1]), mma_bf16(w[2 * n + 1], hi, b[2], b[3]);
            }
        }
        if (p.values.at) {
            __nv_bfloat16* const values = p.values.of(p.sh, base + i, h);
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (row + j * 8 < p.sh.value_dim)
                        dr_store_planes(values, p.values.size, DR_CHUNK, row + j * 8, n * 8 + col, w[n][2 * j], w[n][2 * j + 1]);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {  // u
            const float2 b = *(const float2*)&st.gates[2][n * 8 + col];
            w[n][0] *= b.x, w[n][1] *= b.y, w[n][2] *= b.x, w[n][3] *= b.y;
        }
        // o = scale g o + A u
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float g0 = st.gates[0][m * 16 + g] * p.sh.scale, g1 = st.gates[0][m * 16 + g + 8] * p.sh.scale;
#pragma unroll
            for (int n = 0; n < 2; ++n) o[m][n][0] *= g0, o[m][n][1] *= g0, o[m][n][2] *= g1, o[m][n][3] *= g1;
        }
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(w[2 * kt], w[2 * kt + 1], hi, lo);
#pragma unroll
            for (int m = kt; m < 4; ++m) {
                uint32_t a[4];
                load_a<64>(a, rd[0], m * 16, kt * 2, lane);
                mma_bf16(o[m][0], a, hi[0], hi[2]), mma_bf16(o[m][1], a, hi[1], hi[3]);
                mma_bf16(o[m][0], a, lo[0], lo[2]), mma_bf16(o[m][1], a, lo[1], lo[3]);
                load_a<64>(a, rd[1], m * 16, kt * 2, lane);
                mma_bf16(o[m][0], a, hi[0], hi[2]), mma_bf16(o[m][1], a, hi[1], hi[3]);
            }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t token = m * 16 + g + j * 8;
                if (token >= now.rows) continue;
                T* const to = out + (now.row + token) * p.out_stride + (uint64_t)h * p.sh.value_dim;
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    dr_store_pair(to, v0 + warp * 16 + n * 8 + col, p.sh.value_dim, even, o[m][n][2 * j], o[m][n][2 * j + 1]);
            }
        // S = g_64 S + (e u)^T K
        const float whole = st.gates[0][DR_CHUNK - 1];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[n][j] *= whole;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
            for (int n = 2 * kt; n < 2 * kt + 2; ++n) {
                const float2 e = *(const float2*)&st.gates[1][n * 8 + col];
                w[n][0] *= e.x, w[n][1] *= e.y, w[n][2] *= e.x, w[n][3] *= e.y;
            }
            uint32_t hi[4], lo[4];
            split_block(w[2 * kt], w[2 * kt + 1], hi, lo);
            dr_add_outer<DK, PLANES>(s, hi, lo, k, kt, lane);
        }
        __syncthreads();  // the stage is free
    }
    dr_state_out<NT>(s, p.to ? p.to + state : nullptr, row, p.sh.value_dim, p.sh.key_dim, col);
}

template <int DK, int PLANES, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1)
dr_backward_kernel(const __grid_constant__ DrChain p) {
    constexpr int NT = DK / 8, VC = WARPS > 4 ? 128 : 64;
    extern __shared__ __align__(128) uint8_t dr_smem[];
    auto& smem = *(DrChainSmem<DK, PLANES, WARPS>*)dr_smem;
    const uint32_t slices = (p.sh.value_dim + WARPS * 16 - 1) / (WARPS * 16);
    const uint32_t slice = blockIdx.x % slices, h = blockIdx.x / slices % p.sh.heads, seq = blockIdx.x / slices / p.sh.heads;
    const uint32_t hk = h / (p.sh.heads / p.sh.key_heads), v0 = slice * WARPS * 16;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, g = lane >> 2, col = (lane & 3) * 2;
    const uint32_t row = v0 + warp * 16 + g;
    const uint64_t start = p.sh.start(seq), end = min(p.sh.start(seq + 1), p.sh.rows), base = p.sh.base(seq);
    const uint32_t chunks = end > start ? (uint32_t)((end - start + DR_CHUNK - 1) / DR_CHUNK) : 0;
    const uint64_t state = ((uint64_t)seq * p.sh.heads + h) * p.sh.value_dim * p.sh.key_dim;
    float x[NT][4];
    dr_state_in<NT>(x, p.from ? p.from + state : nullptr, row, p.sh.value_dim, p.sh.key_dim, col);
    DrChunk c(p.sh, base);
    auto chunk = [&](uint32_t i) {
        c.row = start + (uint64_t)i * DR_CHUNK;
        c.rows = (uint32_t)min((uint64_t)DR_CHUNK, end - c.row);
        return c;
    };
    if (chunks) dr_load(smem.stage[0], p, chunk(chunks - 1), base + chunks - 1, h, hk, v0, t);
    cp_async_commit();
    for (uint32_t i = 0; i < chunks; ++i) {
        const uint64_t slot = base + chunks - 1 - i;
        if (i + 1 < chunks) dr_load(smem.stage[(i + 1) & 1], p, chunk(chunks - 2 - i), slot - 1, h, hk, v0, t);
        cp_async_commit();
        cp_async_wait_prior1();
        __syncthreads();
        auto& st = smem.stage[i & 1];
        uint32_t k[PLANES], q[PLANES], go[PLANES];
#pragma unroll
        for (int j = 0; j < PLANES; ++j) k[j] = smem_u32(st.k[j]), q[j] = smem_u32(st.q[j]), go[j] = smem_u32(st.v[j]);
        const uint32_t inv[2] = {smem_u32(st.inverse[0]), smem_u32(st.inverse[1])},
                       rd[2] = {smem_u32(st.read[0]), smem_u32(st.read[1])};
        // du = e X K^T (value x token)
        float du[8][4] = {};
        __nv_bfloat16* const states = p.states.of(p.sh, slot, h);
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t hi[4], lo[4];
            split_block(x[2 * kk], x[2 * kk + 1], hi, lo);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t rr = row + (j & 1) * 8, cc = kk * 16 + (j >> 1) * 8 + col;
                if (rr < p.sh.value_dim && cc < p.key_cols) {
                    __nv_bfloat16* const at = states + rr * p.key_cols + cc;
                    *(uint32_t*)at = hi[j];
                    *(uint32_t*)(at + p.states.size) = lo[j];
                }
            }
            dr_times_keys<DK, PLANES>(du, hi, lo, k, kk, lane);
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 e = *(const float2*)&st.gates[1][n * 8 + col];
            du[n][0] *= e.x, du[n][1] *= e.y, du[n][2] *= e.x, du[n][3] *= e.y;
        }
        // ... + dO^T A
        if (p.v.at) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t a[PLANES][4];
#pragma unroll
                for (int j = 0; j < PLANES; ++j) load_a_t<VC>(a[j], go[j], kt * 16, warp * 2, lane);
#pragma unroll
                for (int n = 0; n <= kt; ++n) {
                    uint32_t b[4];
                    load_b_t<64>(b, rd[0], kt * 16, n * 2, lane);
#pragma unroll
                    for (int j = 0; j < PLANES; ++j) mma_bf16(du[2 * n], a[j], b[0], b[1]), mma_bf16(du[2 * n + 1], a[j], b[2], b[3]);
                    load_b_t<64>(b, rd[1], kt * 16, n * 2, lane);
                    mma_bf16(du[2 * n], a[0], b[0], b[1]), mma_bf16(du[2 * n + 1], a[0], b[2], b[3]);
                }
            }
        }
        // z = du inverse
        float z[8][4] = {};
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(du[2 * kt], du[2 * kt + 1], hi, lo);
#pragma unroll
            for (int n = 0; n <= kt; ++n) {
                uint32_t b[4];
                load_b_t<64>(b, inv[0], kt * 16, n * 2, lane);
                mma_bf16(z[2 * n], hi, b[0], b[1]), mma_bf16(z[2 * n + 1], hi, b[2], b[3]);
                mma_bf16(z[2 * n], lo, b[0], b[1]), mma_bf16(z[2 * n + 1], lo, b[2], b[3]);
                load_b_t<64>(b, inv[1], kt * 16, n * 2, lane);
                mma_bf16(z[2 * n], hi, b[0], b[1]), mma_bf16(z[2 * n + 1], hi, b[2], b[3]);
            }
        }
        __nv_bfloat16* const values = p.values.of(p.sh, slot, h);
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (row + j * 8 < p.sh.value_dim)
                    dr_store_planes(values, p.values.size, DR_CHUNK, row + j * 8, n * 8 + col, z[n][2 * j], z[n][2 * j + 1]);
        // X = g_64 X + (scale g dO)^T Q - (g beta z)^T K
        const float whole = st.gates[0][DR_CHUNK - 1];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[n][j] *= whole;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            if (p.v.at) {
                uint32_t a[PLANES][4];
#pragma unroll
                for (int j = 0; j < PLANES; ++j) load_a_t<VC>(a[j], go[j], kt * 16, warp * 2, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 gate = *(const float2*)&st.gates[0][kt * 16 + (j >> 1) * 8 + col];
                    float v0 = bf16_low(a[0][j]), v1 = bf16_high(a[0][j]);
                    if constexpr (PLANES == 2) v0 += bf16_low(a[PLANES - 1][j]), v1 += bf16_high(a[PLANES - 1][j]);
                    split_bf16(v0 * gate.x * p.sh.scale, v1 * gate.y * p.sh.scale, hi[j], lo[j]);
                }
                dr_add_outer<DK, PLANES>(x, hi, lo, q, kt, lane);
            }
#pragma unroll
            for (int n = 2 * kt; n < 2 * kt + 2; ++n) {
                const float2 gate = *(const float2*)&st.gates[0][n * 8 + col], b = *(const float2*)&st.gates[2][n * 8 + col];
                const float y0 = -gate.x * b.x, y1 = -gate.y * b.y;
                z[n][0] *= y0, z[n][1] *= y1, z[n][2] *= y0, z[n][3] *= y1;
            }
            split_block(z[2 * kt], z[2 * kt + 1], hi, lo);
            dr_add_outer<DK, PLANES>(x, hi, lo, k, kt, lane);
        }
        __syncthreads();
    }
    dr_state_out<NT>(x, p.to ? p.to + state : nullptr, row, p.sh.value_dim, p.sh.key_dim, col);
}

// ---- gradients of the inputs ------------------------------------------------------------------------
constexpr int DR_GRAD_THREADS = 256;  // warps: 4 blocks of 16 tokens x 2 halves of the key columns
template <int DK, int PLANES>
struct DrGradientSmem {
    __nv_bfloat16 k[PLANES][DR_CHUNK * DK], q[PLANES][DR_CHUNK * DK];
    __nv_bfloat16 s[2][64 * DK], x[2][64 * DK];       // 64 of the value dimensions
    __nv_bfloat16 w[2][64 * DR_CHUNK], z[2][64 * DR_CHUNK], go[PLANES][DR_CHUNK * 64];
    __nv_bfloat16 da[2][DR_TILE], dn[2][DR_TILE];
    float gates[3][DR_CHUNK];
    double total[DR_CHUNK];
    float dot[2][DR_CHUNK], carry[2][DR_CHUNK], dbeta[4][DR_CHUNK], sx[8];
};

struct DrGradient {
    DrShape sh;
    DrOperand q, k, go;
    DrPrepared prepared;
    const float* decay;
    uint64_t decay_stride;
    DrPlanes s, w, x, z;
    uint32_t key_cols;
    void *dq, *dk, *dv;
    float *ddecay, *dbeta;
    bool pairs_k, pairs_v;  // elements 2 i and 2 i + 1 of a row can be stored together: of dq and dk, of dv
};

template <typename T, int DK, int PLANES>
__global__ void __launch_bounds__(DR_GRAD_THREADS, 1)
dr_gradient_kernel(const __grid_constant__ DrGradient p) {
    constexpr int NT = DK / 16, NP = DK / 32;  // tiles and pairs of tiles of 8 key columns a warp has
    extern __shared__ __align__(128) uint8_t dr_smem[];
    auto& sm = *(DrGradientSmem<DK, PLANES>*)dr_smem;
    const uint64_t slot = blockIdx.x / p.sh.key_heads;
    const uint32_t hk = blockIdx.x % p.sh.key_heads, group = p.sh.heads / p.sh.key_heads;
    const DrChunk c(p.sh, slot);
    if (!c.rows) return;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rb = warp >> 1, ch = warp & 1, g = lane >> 2, col = (lane & 3) * 2;
    uint32_t k[PLANES], q[PLANES], go[PLANES];
#pragma unroll
    for (int i = 0; i < PLANES; ++i) {
        k[i] = smem_u32(sm.k[i]), q[i] = smem_u32(sm.q[i]), go[i] = smem_u32(sm.go[i]);
        tile_load<DK>(k[i], p.k.rows(slot, c, hk) + i * p.k.plane, p.k.row, DR_CHUNK, p.k.have(c), p.k.dim, t, DR_GRAD_THREADS);
        tile_load<DK>(q[i], p.q.rows(slot, c, hk) + i * p.q.plane, p.q.row, DR_CHUNK, p.q.have(c), p.q.dim, t, DR_GRAD_THREADS);
    }
    const uint32_t s[2] = {smem_u32(sm.s[0]), smem_u32(sm.s[1])}, x[2] = {smem_u32(sm.x[0]), smem_u32(sm.x[1])},
                   w[2] = {smem_u32(sm.w[0]), smem_u32(sm.w[1])}, z[2] = {smem_u32(sm.z[0]), smem_u32(sm.z[1])},
                   da[2] = {smem_u32(sm.da[0]), smem_u32(sm.da[1])}, dn[2] = {smem_u32(sm.dn[0]), smem_u32(sm.dn[1])};
    float all_q[NT][4] = {}, all_k[NT][4] = {};  // sums over the key head's heads
    const uint32_t token = rb * 16 + g;
    for (uint32_t h = hk * group; h < (hk + 1) * group; ++h) {
        const uint64_t at = p.prepared.at(p.sh, slot, h);
        __syncthreads();
        if (t < 3 * DR_CHUNK) (&sm.gates[0][0])[t] = p.prepared.gates[at * 3 * DR_CHUNK + t];
        if (warp == 7) {
            double v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = lane * 2 + j;
                const float d = r < c.rows && p.decay ? p.decay[(c.row + r) * p.decay_stride + h] : 0.0f;
                v[j] = d < DR_LEAST_DECAY ? DR_LEAST_DECAY : d;
            }
            double sum = v[0] + v[1];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += up;
            }
            sm.total[lane * 2] = sum - v[1], sm.total[lane * 2 + 1] = sum;
        }
        float dq[NT][4] = {}, er[NT][4] = {}, wr[NT][4] = {}, a[4][4] = {}, n[4][4] = {};
        float sx = 0.0f;
        for (uint32_t v0 = 0; v0 < p.sh.value_dim; v0 += 64) {
            if (v0) __syncthreads();
            const int have = min((int)(p.sh.value_dim - v0), 64);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                tile_load<DK>(s[i], p.s.of(p.sh, slot, h) + i * p.s.size + v0 * p.key_cols, p.key_cols, 64, have, p.key_cols, t, DR_GRAD_THREADS);
                tile_load<DK>(x[i], p.x.of(p.sh, slot, h) + i * p.x.size + v0 * p.key_cols, p.key_cols, 64, have, p.key_cols, t, DR_GRAD_THREADS);
                tile_load<64>(w[i], p.w.of(p.sh, slot, h) + i * p.w.size + v0 * DR_CHUNK, DR_CHUNK, 64, have, 64, t, DR_GRAD_THREADS);
                tile_load<64>(z[i], p.z.of(p.sh, slot, h) + i * p.z.size + v0 * DR_CHUNK, DR_CHUNK, 64, have, 64, t, DR_GRAD_THREADS);
            }
#pragma unroll
            for (int i = 0; i < PLANES; ++i)
                if (p.go.at)
                    tile_load<64>(go[i], p.go.rows(slot, c, h) + i * p.go.plane + v0, p.go.row, DR_CHUNK, p.go.have(c),
                                  (int)p.go.dim - (int)v0, t, DR_GRAD_THREADS);
            cp_async_commit();
            cp_async_wait_all();
            __syncthreads();
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t ag[PLANES][4], aw[2][4], az[2][4];
                if (p.go.at) {
#pragma unroll
                    for (int i = 0; i < PLANES; ++i) load_a<64>(ag[i], go[i], rb * 16, kt * 2, lane);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) load_a_t<64>(aw[i], w[i], kt * 16, rb * 2, lane), load_a_t<64>(az[i], z[i], kt * 16, rb * 2, lane);
                if (ch == 0) {  // dv = beta z
                    T* const to = (T*)p.dv + (c.row * p.sh.heads + h) * p.sh.value_dim;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t r = token + (j & 1) * 8;
                        const float b = sm.gates[2][r];
                        if (r < c.rows)
                            dr_store_pair(to + (uint64_t)r * p.sh.heads * p.sh.value_dim, v0 + kt * 16 + (j >> 1) * 8 + col, p.sh.value_dim,
                                          p.pairs_v, b * (bf16_low(az[0][j]) + bf16_low(az[1][j])),
                                          b * (bf16_high(az[0][j]) + bf16_high(az[1][j])));
                    }
                }
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    uint32_t b[4];
                    const int piece = (ch * NP + j) * 2;
                    load_b_t<DK>(b, s[0], kt * 16, piece, lane);
                    if (p.go.at) {
#pragma unroll
                        for (int i = 0; i < PLANES; ++i) mma_bf16(dq[2 * j], ag[i], b[0], b[1]), mma_bf16(dq[2 * j + 1], ag[i], b[2], b[3]);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma_bf16(er[2 * j], az[i], b[0], b[1]), mma_bf16(er[2 * j + 1], az[i], b[2], b[3]);
                    load_b_t<DK>(b, s[1], kt * 16, piece, lane);
                    if (p.go.at) mma_bf16(dq[2 * j], ag[0], b[0], b[1]), mma_bf16(dq[2 * j + 1], ag[0], b[2], b[3]);
                    mma_bf16(er[2 * j], az[0], b[0], b[1]), mma_bf16(er[2 * j + 1], az[0], b[2], b[3]);
                    load_b_t<DK>(b, x[0], kt * 16, piece, lane);
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma_bf16(wr[2 * j], aw[i], b[0], b[1]), mma_bf16(wr[2 * j + 1], aw[i], b[2], b[3]);
                    load_b_t<DK>(b, x[1], kt * 16, piece, lane);
                    mma_bf16(wr[2 * j], aw[0], b[0], b[1]), mma_bf16(wr[2 * j + 1], aw[0], b[2], b[3]);
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // 32 of the other tokens
                    uint32_t b[4];
                    load_b_t<64>(b, w[0], kt * 16, (ch * 2 + j) * 2, lane);
                    if (p.go.at) {
#pragma unroll
                        for (int i = 0; i < PLANES; ++i) mma_bf16(a[2 * j], ag[i], b[0], b[1]), mma_bf16(a[2 * j + 1], ag[i], b[2], b[3]);
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) mma_bf16(n[2 * j], az[i], b[0], b[1]), mma_bf16(n[2 * j + 1], az[i], b[2], b[3]);
                    load_b_t<64>(b, w[1], kt * 16, (ch * 2 + j) * 2, lane);
                    if (p.go.at) mma_bf16(a[2 * j], ag[0], b[0], b[1]), mma_bf16(a[2 * j + 1], ag[0], b[2], b[3]);
                    mma_bf16(n[2 * j], az[0], b[0], b[1]), mma_bf16(n[2 * j + 1], az[0], b[2], b[3]);
                }
            }
            // <S0, X> and w.z
            for (int i = t; i < 64 * DK / 2; i += DR_GRAD_THREADS) {
                const uint32_t s0 = ((const uint32_t*)sm.s[0])[i], s1 = ((const uint32_t*)sm.s[1])[i],
                               x0 = ((const uint32_t*)sm.x[0])[i], x1 = ((const uint32_t*)sm.x[1])[i];
                sx = fmaf(bf16_low(s0) + bf16_low(s1), bf16_low(x0) + bf16_low(x1), sx);
                sx = fmaf(bf16_high(s0) + bf16_high(s1), bf16_high(x0) + bf16_high(x1), sx);
            }
            {
                const int j = (t & 31) * 2;  // two tokens, 8 of the value dimensions
                float d0 = 0.0f, d1 = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int r = warp * 8 + i;
                    const uint32_t w0 = tile_word<64>(w[0], r, j), w1 = tile_word<64>(w[1], r, j), z0 = tile_word<64>(z[0], r, j),
                                   z1 = tile_word<64>(z[1], r, j);
                    d0 = fmaf(bf16_low(w0) + bf16_low(w1), bf16_low(z0) + bf16_low(z1), d0);
                    d1 = fmaf(bf16_high(w0) + bf16_high(w1), bf16_high(z0) + bf16_high(z1), d1);
                }
                // warps 2 i and 2 i + 1 take turns with row i of the table
                if (v0 == 0 && (warp & 1) == 0) sm.dbeta[warp >> 1][j] = 0.0f, sm.dbeta[warp >> 1][j + 1] = 0.0f;
                __syncthreads();
                if ((warp & 1) == 0) sm.dbeta[warp >> 1][j] += d0, sm.dbeta[warp >> 1][j + 1] += d1;
                __syncthreads();
                if ((warp & 1) == 1) sm.dbeta[warp >> 1][j] += d0, sm.dbeta[warp >> 1][j + 1] += d1;
            }
        }
        // scale D dA and D dN as operands: dA_ij = beta_j a_ij, dN_ij = -beta_i beta_j n_ij
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int i = token + half * 8, c0 = ch * 32 + j * 8 + col;
                float va[2], vn[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int cc = c0 + e;
                    const float d = cc <= i ? expf((float)(sm.total[i] - sm.total[cc])) * sm.gates[2][cc] : 0.0f;
                    va[e] = cc <= i ? p.sh.scale * d * a[j][half * 2 + e] : 0.0f;
                    vn[e] = cc < i ? -d * sm.gates[2][i] * n[j][half * 2 + e] : 0.0f;
                }
                uint32_t hi, lo;
                const uint32_t off = tile_at<64>(0, i, c0 >> 3) + (c0 & 7) * 2;
                split_bf16(va[0], va[1], hi, lo);
                *(uint32_t*)((char*)sm.da[0] + off) = hi, *(uint32_t*)((char*)sm.da[1] + off) = lo;
                split_bf16(vn[0], vn[1], hi, lo);
                *(uint32_t*)((char*)sm.dn[0] + off) = hi, *(uint32_t*)((char*)sm.dn[1] + off) = lo;
            }
        // row factors of the products with the states; k.(e u X) is needed by itself
        float carry[2] = {0.0f, 0.0f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = token + half * 8;
            const float g0 = sm.gates[0][i], e = sm.gates[1][i] * sm.gates[2][i], b = sm.gates[2][i];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int cc = ch * (DK / 2) + j * 8 + col;
                uint32_t kw = tile_word<DK>(k[0], i, cc);
                float k0 = bf16_low(kw), k1 = bf16_high(kw);
                if constexpr (PLANES == 2) kw = tile_word<DK>(k[PLANES - 1], i, cc), k0 += bf16_low(kw), k1 += bf16_high(kw);
#pragma unroll
                for (int m = half * 2; m < half * 2 + 2; ++m) dq[j][m] *= g0 * p.sh.scale, er[j][m] *= -g0 * b, wr[j][m] *= e;
                carry[half] = fmaf(k0, wr[j][half * 2], fmaf(k1, wr[j][half * 2 + 1], carry[half]));
            }
        }
        __syncthreads();
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
#pragma unroll
            for (int side = 0; side < 2; ++side) {  // rows of dA, dN against earlier tokens; columns against later ones
                if (side == 0 ? kt > rb : kt < rb) continue;
                uint32_t fa[2][4], fn[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (side == 0) load_a<64>(fa[i], da[i], rb * 16, kt * 2, lane), load_a<64>(fn[i], dn[i], rb * 16, kt * 2, lane);
                    else load_a_t<64>(fa[i], da[i], kt * 16, rb * 2, lane), load_a_t<64>(fn[i], dn[i], kt * 16, rb * 2, lane);
                }
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int piece = (ch * NP + j) * 2;
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < PLANES; ++i) {
                        load_b_t<DK>(b, k[i], kt * 16, piece, lane);
#pragma unroll
                        for (int l = 0; l < 2 - i; ++l) {
                            if (side == 0) {
                                mma_bf16(dq[2 * j], fa[l], b[0], b[1]), mma_bf16(dq[2 * j + 1], fa[l], b[2], b[3]);
                                mma_bf16(er[2 * j], fn[l], b[0], b[1]), mma_bf16(er[2 * j + 1], fn[l], b[2], b[3]);
                            } else {
                                mma_bf16(wr[2 * j], fn[l], b[0], b[1]), mma_bf16(wr[2 * j + 1], fn[l], b[2], b[3]);
                            }
                        }
                        if (side == 1) {
                            load_b_t<DK>(b, q[i], kt * 16, piece, lane);
#pragma unroll
                            for (int l = 0; l < 2 - i; ++l) mma_bf16(wr[2 * j], fa[l], b[0], b[1]), mma_bf16(wr[2 * j + 1], fa[l], b[2], b[3]);
                        }
                    }
                }
            }
        }
        // q.dq + k.(erase - write)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = token + half * 8;
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int cc = ch * (DK / 2) + j * 8 + col;
                float kv[2] = {0, 0}, qv[2] = {0, 0};
#pragma unroll
                for (int l = 0; l < PLANES; ++l) {
                    const uint32_t kw = tile_word<DK>(k[l], i, cc), qw = tile_word<DK>(q[l], i, cc);
                    kv[0] += bf16_low(kw), kv[1] += bf16_high(kw), qv[0] += bf16_low(qw), qv[1] += bf16_high(qw);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int m = half * 2 + e;
                    dot = fmaf(qv[e], dq[j][m], fmaf(kv[e], er[j][m] - wr[j][m], dot));
                    all_q[j][m] += dq[j][m], all_k[j][m] += er[j][m] + wr[j][m];
                }
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                dot += __shfl_xor_sync(0xffffffffu, dot, o);
                carry[half] += __shfl_xor_sync(0xffffffffu, carry[half], o);
            }
            if ((lane & 3) == 0) sm.dot[ch][i] = dot, sm.carry[ch][i] = carry[half];
        }
        sx = warp_reduce<OpSum>(sx);
        if (lane == 0) sm.sx[warp] = sx;
        __syncthreads();
        if (warp == 0) {
            double d[2], extra = 0.0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = lane * 2 + j;
                d[j] = (double)sm.dot[0][r] + sm.dot[1][r];
                extra += (double)sm.carry[0][r] + sm.carry[1][r];
            }
            if (lane < 8) extra += (double)sm.sx[lane] * sm.gates[0][DR_CHUNK - 1];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) extra += __shfl_xor_sync(0xffffffffu, extra, o);
            double sum = d[0] + d[1];  // from the lane's rows to the end
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double down = __shfl_down_sync(0xffffffffu, sum, o);
                if (lane + o < 32) sum += down;
            }
            const double v[2] = {sum + extra, sum - d[0] + extra};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = lane * 2 + j;
                if (r < c.rows) {
                    const uint64_t to = (c.row + r) * p.sh.heads + h;
                    if (p.ddecay) p.ddecay[to] = (float)v[j];
                    p.dbeta[to] = (sm.dbeta[0][r] + sm.dbeta[1][r]) + (sm.dbeta[2][r] + sm.dbeta[3][r]);
                }
            }
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint32_t i = token + half * 8;
        if (i >= c.rows) continue;
        const uint64_t to = ((c.row + i) * p.sh.key_heads + hk) * p.sh.key_dim;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint32_t cc = ch * (DK / 2) + j * 8 + col;
            dr_store_pair((T*)p.dq + to, cc, p.sh.key_dim, p.pairs_k, all_q[j][half * 2], all_q[j][half * 2 + 1]);
            dr_store_pair((T*)p.dk + to, cc, p.sh.key_dim, p.pairs_k, all_k[j][half * 2], all_k[j][half * 2 + 1]);
        }
    }
}

// Rows outside all sequences: zeros.
struct DrFill {
    void* at;
    uint64_t stride, bytes;  // of a row
};
struct DrFills {
    DrFill f[5];
};
__global__ void __launch_bounds__(256) dr_padding_kernel(DrShape sh, DrFills fills) {
    const uint64_t first = min((uint64_t)sh.offsets[0], sh.rows), last = min((uint64_t)sh.offsets[sh.sequences], sh.rows);
    const uint64_t outside = first + (sh.rows - last);
    for (uint64_t i = blockIdx.x; i < outside; i += gridDim.x) {
        const uint64_t r = i < first ? i : i - first + last;
#pragma unroll
        for (int k = 0; k < 5; ++k) {
            if (!fills.f[k].at) continue;
            uint16_t* const to = (uint16_t*)((char*)fills.f[k].at + r * fills.f[k].stride);
            for (uint64_t b = threadIdx.x; b < fills.f[k].bytes / 2; b += blockDim.x) to[b] = 0;
        }
    }
}

// ---- one token ------------------------------------------------------------------------------------
constexpr int DR_STEP_WARPS = 4;
// A warp takes 8 rows of a state (value dimensions) at a time: a lane holds 4 key columns of each.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(DR_STEP_WARPS * 32)
dr_step_kernel(DrShape sh, const T* q, uint64_t q_stride, const T* k, uint64_t k_stride, const T* v, uint64_t v_stride,
               const float* decay, uint64_t decay_stride, const float* beta, uint64_t beta_stride, const float* states_in,
               uint64_t rows_in, const int32_t* parents, float* states_out, T* out, uint64_t out_stride, uint32_t parts) {
    const int lane = threadIdx.x & 31;
    const uint64_t unit = (uint64_t)blockIdx.x * DR_STEP_WARPS + (threadIdx.x >> 5);
    const uint64_t pair = unit / parts;  // row and head
    if (pair >= sh.rows * sh.heads) return;
    const uint64_t r = pair / sh.heads;
    const uint32_t h = (uint32_t)(pair % sh.heads), hk = h / (sh.heads / sh.key_heads), v0 = (uint32_t)(unit % parts) * 8;
    int64_t from = parents ? (int64_t)parents[r] : (int64_t)r;
    if (!states_in) {
        from = -1;
    } else if (from >= (int64_t)rows_in) {
        set_error(LCPP_ERR_INVALID_ARG);
        from = -1;
    }
    auto column = [&](int j) { return WIDE ? (uint32_t)lane * 4 + j : (uint32_t)lane + j * 32; };
    const uint64_t size = (uint64_t)sh.value_dim * sh.key_dim;
    float s[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool have = from >= 0 && v0 + i < sh.value_dim;
        const float* const at = states_in + ((uint64_t)from * sh.heads + h) * size + (uint64_t)(v0 + i) * sh.key_dim;
        if constexpr (WIDE) {
            float4 f = make_float4(0, 0, 0, 0);
            if (have && column(0) < sh.key_dim) f = *(const float4*)(at + column(0));
            s[i][0] = f.x, s[i][1] = f.y, s[i][2] = f.z, s[i][3] = f.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] = have && column(j) < sh.key_dim ? at[column(j)] : 0.0f;
        }
    }
    float kv[4], qv[4], qk = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const bool have = column(j) < sh.key_dim;
        kv[j] = have ? widen(k[r * k_stride + (uint64_t)hk * sh.key_dim + column(j)]) : 0.0f;
        qv[j] = have ? widen(q[r * q_stride + (uint64_t)hk * sh.key_dim + column(j)]) : 0.0f;
        qk = fmaf(qv[j], kv[j], qk);
    }
    const float factor = decay ? expf(decay[r * decay_stride + h]) : 1.0f, b = beta[r * beta_stride + h];
    // S' k and S' q by 8 rows, 16 sums over the lanes: halved at each step, so that lane i ends with the sum i & 15
    float sum[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[i][j] *= factor;
            a = fmaf(s[i][j], kv[j], a), c = fmaf(s[i][j], qv[j], c);
        }
        sum[i] = a, sum[8 + i] = c;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const bool up = lane & o;
            const float keep = up ? sum[i + o] : sum[i], give = up ? sum[i] : sum[i + o];
            sum[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
    }
    sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 16);
    qk = warp_reduce<OpSum>(qk);
    // lanes 0-7: S' k of row i; 8-15: S' q of row i - 8
    const uint32_t mine = v0 + (lane & 7);
    const bool live = mine < sh.value_dim;
    const float value = live ? widen(v[r * v_stride + (uint64_t)h * sh.value_dim + mine]) : 0.0f;
    const float sk = __shfl_sync(0xffffffffu, sum[0], lane & 7), sq = __shfl_sync(0xffffffffu, sum[0], 8 + (lane & 7));
    const float u = b * (value - sk);
    if (lane < 8 && live) out[r * out_stride + (uint64_t)h * sh.value_dim + mine] = narrow<T>(sh.scale * fmaf(u, qk, sq));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float ui = __shfl_sync(0xffffffffu, u, i);
        if (v0 + i >= sh.value_dim) continue;
        float* const at = states_out + (r * sh.heads + h) * size + (uint64_t)(v0 + i) * sh.key_dim;
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(ui, kv[j], s[i][j]);
        if constexpr (WIDE) {
            if (column(0) < sh.key_dim) *(float4*)(at + column(0)) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (column(j) < sh.key_dim) at[column(j)] = s[i][j];
        }
    }
}

// ---- host -----------------------------------------------------------------------------------------
constexpr uint64_t DR_MAX_ROWS = 0xffffffffull, DR_MAX_SEQUENCES = 1ull << 28, DR_MAX_HEADS = 1u << 16;

static lcpp_status dr_check(int dtype, const lcpp_delta_shape* sh) {
    if (!sh || !is_float_dtype(dtype) || sh->rows > DR_MAX_ROWS || sh->num_sequences > DR_MAX_SEQUENCES ||
        sh->heads > DR_MAX_HEADS || sh->key_dim > DR_MAX_DIM || sh->value_dim > DR_MAX_DIM || !sh->heads || !sh->key_heads ||
        !sh->key_dim || !sh->value_dim || sh->heads % sh->key_heads)
        return LCPP_ERR_INVALID_ARG;
    return LCPP_OK;
}
static DrShape dr_shape(const lcpp_delta_shape& sh) {
    return DrShape{sh.rows, sh.offsets ? 0 : sh.length, sh.offsets, (uint32_t)sh.num_sequences, sh.heads, sh.key_heads,
                   sh.key_dim, sh.value_dim, sh.scale};
}
static uint64_t dr_key_cols(const lcpp_delta_shape& sh) { return align_up(sh.key_dim, 16); }

struct DrLayout {
    uint64_t slots, state, value;  // chunks; elements of a plane
    size_t inverse, read, gates, x, z, q, k, v, bytes;
    uint64_t key_pitch, value_pitch;
    bool packed;
    DrLayout(const lcpp_delta_shape& sh, bool backward, bool pack) : packed(pack) {
        slots = sh.rows / DR_CHUNK + sh.num_sequences;
        state = sh.value_dim * dr_key_cols(sh), value = sh.value_dim * DR_CHUNK;
        key_pitch = align_up(sh.key_dim, 8), value_pitch = align_up(sh.value_dim, 8);
        size_t at = 0;
        auto take = [&](uint64_t n) {
            const size_t here = at;
            at += align_up(n, 256);
            return here;
        };
        const uint64_t units = slots * sh.heads;
        inverse = take(units * 2 * DR_TILE * 2), read = take(units * 2 * DR_TILE * 2), gates = take(units * 3 * DR_CHUNK * 4);
        x = z = q = k = v = 0;
        if (backward) x = take(units * 2 * state * 2), z = take(units * 2 * value * 2);
        if (pack) {
            q = take(slots * DR_CHUNK * sh.key_heads * key_pitch * 4), k = take(slots * DR_CHUNK * sh.key_heads * key_pitch * 4);
            v = take(slots * DR_CHUNK * sh.heads * value_pitch * 4);  // dO in the backward pass
        }
        bytes = max(at, (size_t)256);
    }
    DrPrepared prepared(void* temp) const {
        char* const t = (char*)temp;
        return DrPrepared{(__nv_bfloat16*)(t + inverse), (__nv_bfloat16*)(t + read), (float*)(t + gates)};
    }
};

// Rows of bf16 that can be copied in pieces of 16 bytes.
static bool dr_direct(const void* p, uint64_t stride, uint64_t rows, uint32_t dim) {
    return (uintptr_t)p % 16 == 0 && dim % 8 == 0 && (rows <= 1 || stride % 8 == 0);
}

template <typename T>
static lcpp_status dr_operand(const DrShape& sh, const DrLayout& l, const void* from, uint64_t stride, uint32_t heads, uint32_t dim,
                              uint64_t pitch, void* room, DrOperand* to, cudaStream_t s) {
    if (!from) {
        *to = DrOperand{};
        return LCPP_OK;
    }
    if (!l.packed) {
        *to = DrOperand{(const __nv_bfloat16*)from, stride, 0, dim, dim, false};
        return LCPP_OK;
    }
    const uint64_t plane = l.slots * DR_CHUNK * heads * pitch;
    *to = DrOperand{(const __nv_bfloat16*)room, heads * pitch, plane, (uint32_t)pitch, (uint32_t)pitch, true};
    ProfScope prof("dr_pack", s);
    dr_pack_kernel<T><<<(unsigned)l.slots, 256, 0, s>>>(sh, (const T*)from, stride, heads, dim, (__nv_bfloat16*)room, plane, (uint32_t)pitch);
    count_launch();
    return check_launch();
}

// Allows KERNEL `smem` bytes of shared memory on the current device.
template <auto KERNEL>
static bool dr_sized(size_t smem) {
    static std::atomic<uint64_t> sized{0};
    const uint64_t bit = 1ull << device_info().device;
    if (sized.load(std::memory_order_relaxed) & bit) return true;
    if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) return false;
    sized.fetch_or(bit, std::memory_order_relaxed);
    return true;
}
template <auto KERNEL, typename... A>
static lcpp_status dr_launch(const char* name, uint64_t grid, unsigned threads, size_t smem, cudaStream_t s, const A&... args) {
    if (grid > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    if (!dr_sized<KERNEL>(smem)) return check_launch();
    ProfScope prof(name, s);
    KERNEL<<<(unsigned)grid, threads, smem, s>>>(args...);
    count_launch();
    return check_launch();
}

// How many warps a CTA of the chain has, 16 value dimensions each: fewer where that spreads the states over more SMs.
// Two planes of 128 key columns leave shared memory for 4 warps' values.
static int dr_warps(const lcpp_delta_shape& sh, bool packed) {
    const uint64_t states = sh.num_sequences * sh.heads, sms = device_info().sms;
    int warps = packed ? 4 : 8;
    while (warps > 2 && (warps * 8u >= sh.value_dim || states * ceil_div(sh.value_dim, warps * 16) * 2 <= sms)) warps /= 2;
    return warps;
}

template <typename T, typename F>
static lcpp_status dr_dispatch(const lcpp_delta_shape& sh, bool packed, F&& f) {
    auto planes = [&](auto dk) -> lcpp_status {
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            if (!packed) return f(dk, std::integral_constant<int, 1>{});
        }
        return f(dk, std::integral_constant<int, 2>{});
    };
    return sh.key_dim <= 64 ? planes(std::integral_constant<int, 64>{}) : planes(std::integral_constant<int, 128>{});
}

// Everything that a call reads, and its checks.
struct DrCall {
    int dtype;
    const lcpp_delta_shape& sh;
    const lcpp_delta_inputs& in;
    uint64_t element() const { return dtype == LCPP_F32 ? 4 : 2; }
    uint64_t keys() const { return (uint64_t)sh.key_heads * sh.key_dim; }
    uint64_t values() const { return (uint64_t)sh.heads * sh.value_dim; }
    uint64_t state() const { return values() * sh.key_dim; }
    static bool stride_ok(uint64_t stride, uint64_t rows, uint64_t width) {
        return rows <= 1 || (stride >= width && stride < (1ull << 31));
    }
    lcpp_status check(bool sequences) const {
        if (sequences) {
            if (!sh.offsets && (sh.length > DR_MAX_ROWS || sh.num_sequences * sh.length != sh.rows)) return LCPP_ERR_INVALID_ARG;
            if ((uintptr_t)sh.offsets % 4) return LCPP_ERR_INVALID_ARG;
        }
        if (sh.rows && (!in.q || !in.k || !in.v || !in.beta)) return LCPP_ERR_INVALID_ARG;
        if (!stride_ok(in.q_stride, sh.rows, keys()) || !stride_ok(in.k_stride, sh.rows, keys()) ||
            !stride_ok(in.v_stride, sh.rows, values()) || !stride_ok(in.beta_stride, sh.rows, sh.heads) ||
            (in.decay && !stride_ok(in.decay_stride, sh.rows, sh.heads)))
            return LCPP_ERR_INVALID_ARG;
        if (!elements_aligned(dtype, in.q, in.k, in.v) || !elements_aligned(LCPP_F32, in.decay, in.beta, in.init))
            return LCPP_ERR_INVALID_ARG;
        return LCPP_OK;
    }
    Region matrix(const void* p, uint64_t stride, uint64_t width, uint64_t e) const { return Region(p, sh.rows, stride * e, width * e); }
    Region q() const { return matrix(in.q, in.q_stride, keys(), element()); }
    Region k() const { return matrix(in.k, in.k_stride, keys(), element()); }
    Region v() const { return matrix(in.v, in.v_stride, values(), element()); }
    Region decay() const { return matrix(in.decay, in.decay_stride, sh.heads, 4); }
    Region beta() const { return matrix(in.beta, in.beta_stride, sh.heads, 4); }
    Region states(const float* p) const { return Region(p, sh.num_sequences * state() * 4); }
    Region offsets() const { return Region(sh.offsets, (sh.num_sequences + 1) * 4); }
    // `w` is apart from all inputs but, where init_too is false, the first states.
    bool apart(const Region& w, bool init_too = true) const {
        return w.apart(q(), k(), v(), decay(), beta(), offsets()) && (!init_too || w.apart(states(in.init)));
    }
    bool direct() const {
        return dtype == LCPP_BF16 && dr_direct(in.q, in.q_stride, sh.rows, sh.key_dim) &&
               dr_direct(in.k, in.k_stride, sh.rows, sh.key_dim) && dr_direct(in.v, in.v_stride, sh.rows, sh.value_dim);
    }
};

static lcpp_status dr_padding(const DrShape& sh, const DrFills& fills, cudaStream_t s) {
    if (!sh.offsets || !sh.rows) return LCPP_OK;
    ProfScope prof("dr_padding", s);
    dr_padding_kernel<<<(unsigned)min(sh.rows, (uint64_t)device_info().sms * 4), 256, 0, s>>>(sh, fills);
    count_launch();
    return check_launch();
}

}  // namespace lcpp

using namespace lcpp;

extern "C" size_t lcpp_delta_rule_temp_bytes(int dtype, const lcpp_delta_shape* shape, int backward, int aligned) {
    if (dr_check(dtype, shape) != LCPP_OK) return 0;
    const bool pack = dtype != LCPP_BF16 || !aligned || shape->key_dim % 8 || shape->value_dim % 8;
    return DrLayout(*shape, backward != 0, pack).bytes;
}

extern "C" size_t lcpp_delta_rule_saved_bytes(const lcpp_delta_shape* shape) {
    if (dr_check(LCPP_F32, shape) != LCPP_OK) return 0;
    const DrLayout l(*shape, false, false);
    const uint64_t units = l.slots * shape->heads;
    return align_up(units * 2 * l.state * 2, 256) + align_up(units * 2 * l.value * 2, 256);
}

extern "C" lcpp_status lcpp_delta_rule_forward(int dtype, const lcpp_delta_shape* shape, const lcpp_delta_inputs* inputs, void* out,
                                               uint64_t out_stride, float* last, void* saved, void* temp, size_t temp_bytes,
                                               void* stream) {
    if (!inputs || dr_check(dtype, shape) != LCPP_OK) return LCPP_ERR_INVALID_ARG;
    const DrCall c{dtype, *shape, *inputs};
    const lcpp_status ok = c.check(true);
    if (ok != LCPP_OK) return ok;
    if (!shape->num_sequences && !shape->rows) return LCPP_OK;
    if (!elements_aligned(dtype, out) || !elements_aligned(LCPP_F32, last) || (uintptr_t)saved % 16 ||
        (shape->rows && (!out || !DrCall::stride_ok(out_stride, shape->rows, c.values()))))
        return LCPP_ERR_INVALID_ARG;
    const bool packed = !c.direct();
    const DrLayout l(*shape, false, packed);
    if (!temp || temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % 16) return LCPP_ERR_INVALID_ARG;
    const Region ro = c.matrix(out, out_stride, c.values(), c.element()), rl = c.states(last), rt(temp, l.bytes),
                 rs(saved, lcpp_delta_rule_saved_bytes(shape));
    if (!c.apart(ro) || !c.apart(rl, false) || !rl.apart_or_same(c.states(inputs->init)) || !c.apart(rt) || !c.apart(rs) ||
        !ro.apart(rl, rt, rs) || !rl.apart(rt, rs) || !rt.apart(rs))
        return LCPP_ERR_INVALID_ARG;
    const cudaStream_t s = (cudaStream_t)stream;
    const DrShape sh = dr_shape(*shape);
    DrFills fills{};
    fills.f[0] = {out, out_stride * c.element(), c.values() * c.element()};
    lcpp_status status = dr_padding(sh, fills, s);
    if (status != LCPP_OK || !shape->num_sequences) return status;
    return dispatch_float(dtype, [&](auto type) -> lcpp_status {
        using T = decltype(type);
        DrChain p{};
        p.sh = sh, p.prepared = l.prepared(temp), p.from = inputs->init, p.to = last, p.out = out, p.out_stride = out_stride;
        p.key_cols = (uint32_t)dr_key_cols(*shape);
        char* const t = (char*)temp;
        lcpp_status status = dr_operand<T>(sh, l, inputs->q, inputs->q_stride, sh.key_heads, sh.key_dim, l.key_pitch, t + l.q, &p.q, s);
        if (status == LCPP_OK) status = dr_operand<T>(sh, l, inputs->k, inputs->k_stride, sh.key_heads, sh.key_dim, l.key_pitch, t + l.k, &p.k, s);
        if (status == LCPP_OK) status = dr_operand<T>(sh, l, inputs->v, inputs->v_stride, sh.heads, sh.value_dim, l.value_pitch, t + l.v, &p.v, s);
        if (status != LCPP_OK) return status;
        if (saved) {
            p.states = DrPlanes{(__nv_bfloat16*)saved, l.state};
            p.values = DrPlanes{(__nv_bfloat16*)((char*)saved + align_up(l.slots * sh.heads * 2 * l.state * 2, 256)), l.value};
        }
        return dr_dispatch<T>(*shape, packed, [&](auto dk, auto planes) -> lcpp_status {
            constexpr int DK = decltype(dk)::value, PLANES = decltype(planes)::value;
            lcpp_status status = LCPP_OK;
            if (sh.rows)
                status = dr_launch<dr_prepare_kernel<DK, PLANES, false>>("dr_prepare", l.slots * sh.key_heads, DR_PREPARE_THREADS,
                                                                         sizeof(DrPrepareSmem<DK, PLANES>), s, sh, p.q, p.k, inputs->decay,
                                                                         inputs->decay_stride, inputs->beta, inputs->beta_stride, p.prepared);
            if (status != LCPP_OK) return status;
            auto chain = [&](auto warps) {
                constexpr int WARPS = decltype(warps)::value;
                const uint64_t grid = (uint64_t)sh.sequences * sh.heads * ceil_div(sh.value_dim, WARPS * 16);
                return dr_launch<dr_forward_kernel<T, DK, PLANES, WARPS>>("dr_forward", grid, WARPS * 32,
                                                                          sizeof(DrChainSmem<DK, PLANES, WARPS>), s, p);
            };
            const int warps = dr_warps(*shape, packed);
            if constexpr (PLANES == 1) {
                if (warps == 8) return chain(std::integral_constant<int, 8>{});
            }
            if (warps == 4) return chain(std::integral_constant<int, 4>{});
            return chain(std::integral_constant<int, 2>{});
        });
    });
}

extern "C" lcpp_status lcpp_delta_rule_backward(int dtype, const lcpp_delta_shape* shape, const lcpp_delta_inputs* inputs,
                                                const void* saved, const lcpp_delta_grads* grads, void* temp, size_t temp_bytes,
                                                void* stream) {
    if (!inputs || !grads || dr_check(dtype, shape) != LCPP_OK) return LCPP_ERR_INVALID_ARG;
    const DrCall c{dtype, *shape, *inputs};
    const lcpp_status ok = c.check(true);
    if (ok != LCPP_OK) return ok;
    if (!shape->num_sequences && !shape->rows) return LCPP_OK;
    if (!elements_aligned(dtype, grads->out, grads->q, grads->k, grads->v) || (uintptr_t)saved % 16 ||
        !elements_aligned(LCPP_F32, grads->last, grads->decay, grads->beta, grads->init))
        return LCPP_ERR_INVALID_ARG;
    if (shape->rows && (!saved || !grads->q || !grads->k || !grads->v || !grads->beta ||
                        (grads->out && !DrCall::stride_ok(grads->out_stride, shape->rows, c.values()))))
        return LCPP_ERR_INVALID_ARG;
    const bool packed = !c.direct() || (grads->out && !dr_direct(grads->out, grads->out_stride, shape->rows, shape->value_dim));
    const DrLayout l(*shape, true, packed);
    if (!temp || temp_bytes < l.bytes) return LCPP_ERR_TEMP_TOO_SMALL;
    if ((uintptr_t)temp % 16) return LCPP_ERR_INVALID_ARG;
    const uint64_t e = c.element(), rows = shape->rows;
    const Region ro = c.matrix(grads->out, grads->out_stride, c.values(), e), rl = c.states(grads->last),
                 rs(saved, lcpp_delta_rule_saved_bytes(shape)), rt(temp, l.bytes);
    const Region written[] = {Region(grads->q, rows * c.keys() * e), Region(grads->k, rows * c.keys() * e),
                              Region(grads->v, rows * c.values() * e), Region(grads->decay, rows * shape->heads * 4),
                              Region(grads->beta, rows * shape->heads * 4), c.states(grads->init), rt};
    for (size_t i = 0; i < sizeof(written) / sizeof(written[0]); ++i) {
        if (!c.apart(written[i]) || !written[i].apart(ro, rl, rs)) return LCPP_ERR_INVALID_ARG;
        for (size_t j = 0; j < i; ++j)
            if (!written[i].apart(written[j])) return LCPP_ERR_INVALID_ARG;
    }
    const cudaStream_t s = (cudaStream_t)stream;
    const DrShape sh = dr_shape(*shape);
    DrFills fills{};
    fills.f[0] = {grads->q, c.keys() * e, c.keys() * e}, fills.f[1] = {grads->k, c.keys() * e, c.keys() * e};
    fills.f[2] = {grads->v, c.values() * e, c.values() * e};
    fills.f[3] = {grads->decay, sh.heads * 4ull, sh.heads * 4ull}, fills.f[4] = {grads->beta, sh.heads * 4ull, sh.heads * 4ull};
    lcpp_status status = dr_padding(sh, fills, s);
    if (status != LCPP_OK || !shape->num_sequences) return status;
    return dispatch_float(dtype, [&](auto type) -> lcpp_status {
        using T = decltype(type);
        DrChain p{};
        p.sh = sh, p.prepared = l.prepared(temp), p.from = grads->last, p.to = grads->init;
        p.key_cols = (uint32_t)dr_key_cols(*shape);
        char* const t = (char*)temp;
        p.states = DrPlanes{(__nv_bfloat16*)(t + l.x), l.state}, p.values = DrPlanes{(__nv_bfloat16*)(t + l.z), l.value};
        lcpp_status status = dr_operand<T>(sh, l, inputs->q, inputs->q_stride, sh.key_heads, sh.key_dim, l.key_pitch, t + l.q, &p.q, s);
        if (status == LCPP_OK) status = dr_operand<T>(sh, l, inputs->k, inputs->k_stride, sh.key_heads, sh.key_dim, l.key_pitch, t + l.k, &p.k, s);
        if (status == LCPP_OK) status = dr_operand<T>(sh, l, grads->out, grads->out_stride, sh.heads, sh.value_dim, l.value_pitch, t + l.v, &p.v, s);
        if (status != LCPP_OK) return status;
        DrGradient gr{};
        gr.sh = sh, gr.q = p.q, gr.k = p.k, gr.go = p.v, gr.prepared = p.prepared, gr.decay = inputs->decay, gr.decay_stride = inputs->decay_stride;
        gr.s = DrPlanes{(__nv_bfloat16*)saved, l.state};
        gr.w = DrPlanes{(__nv_bfloat16*)((char*)saved + align_up(l.slots * sh.heads * 2 * l.state * 2, 256)), l.value};
        gr.x = p.states, gr.z = p.values, gr.key_cols = p.key_cols;
        gr.dq = grads->q, gr.dk = grads->k, gr.dv = grads->v, gr.ddecay = grads->decay, gr.dbeta = grads->beta;
        gr.pairs_k = sh.key_dim % 2 == 0 && ((uintptr_t)grads->q | (uintptr_t)grads->k) % (2 * sizeof(T)) == 0;
        gr.pairs_v = sh.value_dim % 2 == 0 && (uintptr_t)grads->v % (2 * sizeof(T)) == 0;
        return dr_dispatch<T>(*shape, packed, [&](auto dk, auto planes) -> lcpp_status {
            constexpr int DK = decltype(dk)::value, PLANES = decltype(planes)::value;
            lcpp_status status = LCPP_OK;
            if (sh.rows)
                status = dr_launch<dr_prepare_kernel<DK, PLANES, true>>("dr_prepare", l.slots * sh.key_heads, DR_PREPARE_THREADS,
                                                                        sizeof(DrPrepareSmem<DK, PLANES>), s, sh, p.q, p.k, inputs->decay,
                                                                        inputs->decay_stride, inputs->beta, inputs->beta_stride, p.prepared);
            if (status != LCPP_OK) return status;
            auto chain = [&](auto warps) {
                constexpr int WARPS = decltype(warps)::value;
                const uint64_t grid = (uint64_t)sh.sequences * sh.heads * ceil_div(sh.value_dim, WARPS * 16);
                return dr_launch<dr_backward_kernel<DK, PLANES, WARPS>>("dr_backward", grid, WARPS * 32,
                                                                        sizeof(DrChainSmem<DK, PLANES, WARPS>), s, p);
            };
            const int warps = dr_warps(*shape, packed);
            if (PLANES == 1 && warps == 8) {
                if constexpr (PLANES == 1) status = chain(std::integral_constant<int, 8>{});
            } else if (warps == 4) {
                status = chain(std::integral_constant<int, 4>{});
            } else {
                status = chain(std::integral_constant<int, 2>{});
            }
            if (status != LCPP_OK || !sh.rows) return status;
            return dr_launch<dr_gradient_kernel<T, DK, PLANES>>("dr_gradient", l.slots * sh.key_heads, DR_GRAD_THREADS,
                                                                sizeof(DrGradientSmem<DK, PLANES>), s, gr);
        });
    });
}

extern "C" lcpp_status lcpp_delta_rule_step(int dtype, const lcpp_delta_shape* shape, const lcpp_delta_inputs* inputs,
                                            uint64_t rows_in, const int32_t* parents, float* states_out, void* out,
                                            uint64_t out_stride, void* stream) {
    if (!inputs || dr_check(dtype, shape) != LCPP_OK || shape->rows > 0x7fffffffull || rows_in > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    const DrCall c{dtype, *shape, *inputs};
    const lcpp_status ok = c.check(false);
    if (ok != LCPP_OK || !shape->rows) return ok;
    const uint64_t rows = shape->rows, e = c.element();
    if (!states_out || !out || !DrCall::stride_ok(out_stride, rows, c.values()) || !elements_aligned(dtype, out) ||
        !elements_aligned(LCPP_F32, parents, states_out) || (inputs->init && !parents && rows_in < rows))
        return LCPP_ERR_INVALID_ARG;
    const Region ro = c.matrix(out, out_stride, c.values(), e), rn(states_out, rows * c.state() * 4),
                 rs(inputs->init, (parents ? rows_in : rows) * c.state() * 4), rp(parents, rows * 4);
    for (const Region& w : {ro, rn})
        if (!w.apart(c.q(), c.k(), c.v(), c.decay(), c.beta(), rp)) return LCPP_ERR_INVALID_ARG;
    if (!ro.apart(rn, rs) || (parents ? !rn.apart(rs) : !rn.apart_or_same(rs))) return LCPP_ERR_INVALID_ARG;
    const DrShape sh = dr_shape(*shape);
    const uint32_t parts = (uint32_t)ceil_div(sh.value_dim, 8);
    const uint64_t grid = ceil_div(rows * sh.heads * parts, DR_STEP_WARPS);
    const bool wide = sh.key_dim % 4 == 0 && ((uintptr_t)inputs->init | (uintptr_t)states_out) % 16 == 0;
    return dispatch_float(dtype, [&](auto type) -> lcpp_status {
        using T = decltype(type);
        auto launch = [&](auto kernel) -> lcpp_status {
            if (grid > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
            ProfScope prof("dr_step", (cudaStream_t)stream);
            kernel<<<(unsigned)grid, DR_STEP_WARPS * 32, 0, (cudaStream_t)stream>>>(
                sh, (const T*)inputs->q, inputs->q_stride, (const T*)inputs->k, inputs->k_stride, (const T*)inputs->v, inputs->v_stride,
                inputs->decay, inputs->decay_stride, inputs->beta, inputs->beta_stride, inputs->init, rows_in, parents, states_out, (T*)out,
                out_stride, parts);
            count_launch();
            return check_launch();
        };
        return wide ? launch(dr_step_kernel<T, true>) : launch(dr_step_kernel<T, false>);
    });
}
