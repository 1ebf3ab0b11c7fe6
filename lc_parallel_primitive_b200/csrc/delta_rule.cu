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
// Products are of float16 with float32 sums, and a float32 value enters as two float16 with a power of two taken out
// (warp_mma.cuh), so that states, which live for a whole sequence, and gradients keep float32's order of error.  q and k
// of 16 bits are exact in one float16 but for the scale of their tile; float32 ones are split too (PLANES 2).  Pairs of
// bf16, which need no scale, left errors of 5e-6 to 2e-5, these leave 2e-7 to 3e-6.
//
// mma.sync and not tcgen05: a chain's products are 16 x 64 x 16 to 16 x 128 x 16 a warp, and each needs the last one's
// result; in registers that is the next operand at once, where an accumulator in tensor memory would have to be read,
// split and written to shared memory between any two.
//
// Times at 8 sequences of 2048 tokens, 16 heads, 128 dimensions, bf16 (4096 chunks and heads): preparation 126 us, forward
// with what the backward pass wants 261, backward chain 254, gradients 579; 1353 us in all.
#include "float_types.cuh"
#include "warp_mma.cuh"

namespace lcpp {

constexpr int DR_CHUNK = 64;
constexpr int DR_MAX_DIM = 128;
constexpr int DR_BLOCK = DR_CHUNK * BLOCK_ROW;  // bytes of a 64 x 64 block
constexpr uint32_t DR_DRAIN_LIMIT = 1u << 14;    // polls of 32 ns and more that a CTA which gave up waits for its own copies
constexpr float DR_LEAST_DECAY = -150.0f;       // exp of less is 0 in float32 anyway, and -inf has no differences

struct DrShape {
    uint64_t rows, length;
    const uint32_t* offsets;
    const uint32_t* order;  // of the chains: the sequences' numbers, long ones first (null: as they come)
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
    uint32_t rows;
    __device__ __forceinline__ DrChunk(const DrShape& sh, uint64_t slot) : row(0), rows(0) {
        uint32_t lo = 0, hi = sh.sequences;  // the last sequence whose base is not past the slot
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (sh.base(mid) <= slot) lo = mid;
            else hi = mid;
        }
        const uint64_t from = sh.start(lo), to = min(sh.start(lo + 1), sh.rows), base = sh.base(lo);
        if (slot < base) return;
        row = from + (slot - base) * DR_CHUNK;
        if (row < to) rows = (uint32_t)min((uint64_t)DR_CHUNK, to - row);
    }
};

// ---- images --------------------------------------------------------------------------------------
// What the kernels leave for one another lies in blocks as shared memory holds them (warp_mma.cuh).
// Of a slot and key head: K, then Q, each PLANES x (key columns / 64) blocks of 64 rows.
template <int DK, int PLANES>
constexpr int DR_KEYS = PLANES * (DK / 64) * DR_BLOCK;  // bytes of K, and of Q
// Of a slot and head: the inverse, then A (two planes each), then the gates.
struct DrGates {
    float g[64], e[64], beta[64];
    float back_k, back_q, back_inverse, back_read;  // inverses of the scales
    float pad[60];
    float total[64], rest[64];  // running sums of the decays, in two parts
};
constexpr int DR_UNIT = 4 * DR_BLOCK + (int)sizeof(DrGates);
static_assert(DR_UNIT % 16 == 0, "a bulk copy");
// Matrices of a slot and head with a row per value dimension, by 32 rows: two planes of blocks of 32 rows.  Every 16
// rows have a scale of their own, since one warp writes them; its inverse is kept beside.
constexpr int DR_PIECE = 32 * BLOCK_ROW;  // bytes of a block
struct DrImage {
    uint8_t* at;
    float* back;        // 8 for each slot and head
    uint32_t blocks;    // of 64 columns: 1 (tokens), or the key columns'
    uint32_t rows;      // a multiple of 32
    __host__ __device__ uint64_t bytes() const { return (uint64_t)rows / 32 * 2 * blocks * DR_PIECE; }
    __device__ __forceinline__ uint8_t* of(uint64_t unit) const { return at + unit * bytes(); }
};

// Wait for a barrier's phase, with the library's cap of polls of at most a microsecond (read when the first one fails).
__device__ __forceinline__ bool dr_poll(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done;
}
__device__ __forceinline__ bool dr_wait(uint64_t* bar, uint32_t parity) {
    bool done = dr_poll(bar, parity);
    if (!done)
        for (uint32_t left = g_spin_limit; --left && !done;) done = dr_poll(bar, parity);
    return done;
}

// ---- what does not depend on the state ------------------------------------------------------------
__device__ __forceinline__ void dr_let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dr_wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

constexpr int DR_PREPARE_THREADS = 256;  // warps: 4 blocks of 16 rows x 2 halves of the columns
constexpr int DR_PITCH = 68, DR_TMP_PITCH = 40;
struct DrInvert {
    float m[64 * DR_PITCH], inv[64 * DR_PITCH], tmp[32 * DR_TMP_PITCH];
};
// The keys' blocks, then a head's triangular matrix and its inverse, then the blocks of the head's unit, one after the other
// in the same memory.
template <int DK, int PLANES>
struct DrPrepareSmem {
    union alignas(128) {
        uint8_t keys[2 * DR_KEYS<DK, PLANES>];
        DrInvert invert;
        uint8_t blocks[4 * DR_BLOCK];
    };
    alignas(128) DrGates gates;
    float most[2][8];
};

// c (16 x 8) += a (16 x 8 steps, rows `ap` floats apart) b (8 steps x 8, rows `bp` apart), all float32 in shared memory: each
// factor as two tf32 (hi hi + hi lo + lo hi: 2^-21 is left out), which have float32's range.
__device__ __forceinline__ uint32_t dr_tf32(float v) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ void dr_mma_tf32(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
template <int STEPS>
__device__ __forceinline__ void dr_product(float (&c)[4], const float* a, int ap, const float* b, int bp, int lane) {
    const int g = lane >> 2, t = lane & 3;
    a += g * ap + t, b += t * bp + g;
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
        const float av[4] = {a[k * 8], a[k * 8 + 8 * ap], a[k * 8 + 4], a[k * 8 + 8 * ap + 4]}, bv[2] = {b[k * 8 * bp], b[(k * 8 + 4) * bp]};
        uint32_t ah[4], al[4], bh[2], bl[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) ah[i] = dr_tf32(av[i]), al[i] = dr_tf32(av[i] - __uint_as_float(ah[i]));
#pragma unroll
        for (int i = 0; i < 2; ++i) bh[i] = dr_tf32(bv[i]), bl[i] = dr_tf32(bv[i] - __uint_as_float(bh[i]));
        dr_mma_tf32(c, ah, bl), dr_mma_tf32(c, al, bh), dr_mma_tf32(c, ah, bh);
    }
}
__device__ __forceinline__ void dr_put(float* to, int pitch, const float (&c)[4], float by, int lane) {
    to += (lane >> 2) * pitch + (lane & 3) * 2;
    *(float2*)to = make_float2(c[0] * by, c[1] * by);
    *(float2*)(to + 8 * pitch) = make_float2(c[2] * by, c[3] * by);
}

// inv = (I + m)^-1 of a strictly lower triangular m: the 16 x 16 blocks of the diagonal by substitution, a column a
// lane, then blocks below from ones above: [X 0; -Y m21 X, Y].
__device__ __forceinline__ void dr_invert(DrInvert& s) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    if (warp < 4) {
        if (lane < 16) {
            const int b = warp * 16;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float v = i == lane ? 1.0f : 0.0f;
#pragma unroll
                for (int k = 0; k < i; k += 4) {
                    const float4 m = *(const float4*)&s.m[(b + i) * DR_PITCH + b + k];
                    v = fmaf(-m.x, x[k], v);
                    if (k + 1 < i) v = fmaf(-m.y, x[k + 1], v);
                    if (k + 2 < i) v = fmaf(-m.z, x[k + 2], v);
                    if (k + 3 < i) v = fmaf(-m.w, x[k + 3], v);
                }
                x[i] = v;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s.inv[(b + i) * DR_PITCH + b + lane] = x[i];
        }
    } else {
        for (int i = t - 128; i < 64 * 16; i += 128) {  // above the diagonal blocks
            const int r = i >> 4, c = (i & 15) * 4;
            if ((c >> 4) > (r >> 4)) *(float4*)&s.inv[r * DR_PITCH + c] = make_float4(0, 0, 0, 0);
        }
    }
    __syncthreads();
    {  // blocks (16, 0) and (48, 32): 8 of their columns a warp
        const int b = (warp >> 1 & 1) * 32, n = (warp & 1) * 8;
        float* const tmp = s.tmp + (warp >> 1 & 1) * 16 * DR_TMP_PITCH + n;
        if (warp < 4) {
            float c[4] = {0, 0, 0, 0};
            dr_product<2>(c, &s.m[(b + 16) * DR_PITCH + b], DR_PITCH, &s.inv[b * DR_PITCH + b + n], DR_PITCH, lane);
            dr_put(tmp, DR_TMP_PITCH, c, 1.0f, lane);
            __syncwarp();  // a column of the product needs its own columns only
            c[0] = c[1] = c[2] = c[3] = 0.0f;
            dr_product<2>(c, &s.inv[(b + 16) * DR_PITCH + b + 16], DR_PITCH, tmp, DR_TMP_PITCH, lane);
            dr_put(&s.inv[(b + 16) * DR_PITCH + b + n], DR_PITCH, c, -1.0f, lane);
        }
    }
    __syncthreads();
    {  // block (32, 0): 16 x 8 of it a warp
        const int r = (warp >> 2) * 16, n = (warp & 3) * 8;
        float c[4] = {0, 0, 0, 0};
        dr_product<4>(c, &s.m[(32 + r) * DR_PITCH], DR_PITCH, &s.inv[n], DR_PITCH, lane);
        dr_put(s.tmp + r * DR_TMP_PITCH + n, DR_TMP_PITCH, c, 1.0f, lane);
        __syncthreads();
        c[0] = c[1] = c[2] = c[3] = 0.0f;
        dr_product<4>(c, &s.inv[(32 + r) * DR_PITCH + 32], DR_PITCH, s.tmp + n, DR_TMP_PITCH, lane);
        dr_put(&s.inv[(32 + r) * DR_PITCH + n], DR_PITCH, c, -1.0f, lane);
    }
    __syncthreads();
}

// The largest of the warps' values >= 0.
__device__ __forceinline__ float dr_max8(const float* of) {
    return fmaxf(fmaxf(fmaxf(of[0], of[1]), fmaxf(of[2], of[3])), fmaxf(fmaxf(of[4], of[5]), fmaxf(of[6], of[7])));
}

struct DrPrepare {
    DrShape sh;
    const void *q, *k;
    uint64_t q_stride, k_stride;
    const float *decay, *beta;
    uint64_t decay_stride, beta_stride;
    bool wide;  // rows of q and k are whole pieces of 16 bytes on 16 bytes
    uint8_t *keys, *units;
};

// A CTA a chunk and key head, the heads of which it takes in turn.  Bound by shared memory (45 % of its pipe's cycles; issue
// slots 51 %) and by the barriers between its short steps; 3 CTAs an SM (2 for float32's two planes) fill most of the
// gaps, 4 with fewer registers took the same time.  The inverse is by substitution only in its 16 x 16 diagonal blocks:
// 64 rows of it took 3 times as long as the products that join blocks.
template <typename T, int DK, bool BACKWARD>
__global__ void __launch_bounds__(DR_PREPARE_THREADS, sizeof(T) == 4 ? 2 : 3)
dr_prepare_kernel(const __grid_constant__ DrPrepare p) {
    constexpr int PLANES = sizeof(T) == 4 ? 2 : 1, NB = DK / 64, ITEMS = DR_CHUNK * DK / 8 / DR_PREPARE_THREADS;
    extern __shared__ __align__(128) uint8_t dr_smem[];
    auto& s = *(DrPrepareSmem<DK, PLANES>*)dr_smem;
    const DrShape& sh = p.sh;
    dr_let_next_start();
    dr_wait_for_last();
    const uint64_t slot = blockIdx.x / sh.key_heads;
    const uint32_t hk = blockIdx.x % sh.key_heads, group = sh.heads / sh.key_heads;
    const DrChunk c(sh, slot);
    if (!c.rows) return;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rb = warp >> 1, ch = warp & 1;
    const LaneOffsets o(lane);
    // K and Q into blocks, each with a scale
    Scale scale[2];
    {
        alignas(16) T raw[2][ITEMS][8];
        auto from = [&](int x, uint32_t r, uint32_t d) {
            return (const T*)(x ? p.q : p.k) + (c.row + r) * (x ? p.q_stride : p.k_stride) + (uint64_t)hk * sh.key_dim + d;
        };
        if (p.wide) {  // all loads before the first use: rows and columns that do not exist are read from others and cleared
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const uint32_t item = i * DR_PREPARE_THREADS + t, r = item / (DK / 8), d = item % (DK / 8) * 8;
#pragma unroll
                    for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
                        const uint32_t e = d + j * 16 / (int)sizeof(T);
                        ((uint4*)raw[x][i])[j] = __ldg((const uint4*)from(x, min(r, c.rows - 1), e < sh.key_dim ? e : 0));
                    }
                }
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint32_t item = i * DR_PREPARE_THREADS + t, r = item / (DK / 8), d = item % (DK / 8) * 8;
#pragma unroll
                for (int j = 0; j < (int)sizeof(T) / 2; ++j) {
                    if (r < c.rows && d + j * 16 / (int)sizeof(T) < sh.key_dim) continue;
#pragma unroll
                    for (int x = 0; x < 2; ++x) ((uint4*)raw[x][i])[j] = make_uint4(0, 0, 0, 0);
                }
            }
        } else {
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int i = 0; i < ITEMS; ++i) {
                    const uint32_t item = i * DR_PREPARE_THREADS + t, r = item / (DK / 8), d = item % (DK / 8) * 8;
#pragma unroll
                    for (int j = 0; j < 8; ++j) raw[x][i][j] = r < c.rows && d + j < sh.key_dim ? *from(x, r, d + j) : narrow<T>(0.0f);
                }
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) most = fmaxf(most, fabsf(widen(raw[x][i][j])));
            most = warp_max(most);
            if (lane == 0) s.most[x][warp] = most;
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            scale[x] = scale_for<40>(dr_max8(s.most[x]));
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const uint32_t item = i * DR_PREPARE_THREADS + t, r = item / (DK / 8), d = item % (DK / 8) * 8;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) split_f16(widen(raw[x][i][2 * j]), widen(raw[x][i][2 * j + 1]), scale[x].by, hi[j], lo[j]);
                uint8_t* const at = s.keys + x * DR_KEYS<DK, PLANES> + (d >> 6) * DR_BLOCK + block_at(r, d & 63);
                *(uint4*)at = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (PLANES == 2) *(uint4*)(at + NB * DR_BLOCK) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        fence_proxy_async_smem();
        __syncthreads();
    }
    if (t == 0) {
        bulk_store(p.keys + (slot * sh.key_heads + hk) * (2 * DR_KEYS<DK, PLANES>), s.keys, 2 * DR_KEYS<DK, PLANES>);
        bulk_commit();
    }
    float nr[4][4] = {}, rd[4][4] = {};  // k_i.k_j and q_i.k_j: 16 rows and 32 columns a warp
    const uint32_t kt = smem_u32(s.keys), qt = kt + DR_KEYS<DK, PLANES>;
#pragma unroll
    for (int kk = 0; kk < DK / 16; ++kk) {
        if (ch * 2 > rb) break;  // columns past the warp's rows are masked
        const uint32_t block = (kk >> 2) * DR_BLOCK;
        uint32_t ak[PLANES][4], aq[PLANES][4];
#pragma unroll
        for (int i = 0; i < PLANES; ++i) {
            load_a(ak[i], kt + i * NB * DR_BLOCK + block, rb * 16, kk & 3, o);
            load_a(aq[i], qt + i * NB * DR_BLOCK + block, rb * 16, kk & 3, o);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if (ch * 2 + n > rb) break;
#pragma unroll
            for (int i = 0; i < PLANES; ++i) {
                uint32_t b[4];
                load_b(b, kt + i * NB * DR_BLOCK + block, (ch * 2 + n) * 16, kk & 3, o);
#pragma unroll
                for (int l = 0; l < PLANES - i; ++l) mma_f16_2(nr[2 * n], nr[2 * n + 1], ak[l], b), mma_f16_2(rd[2 * n], rd[2 * n + 1], aq[l], b);
            }
        }
    }
    const int r0 = rb * 16 + (lane >> 2), col = ch * 32 + (lane & 3) * 2;
    const float back_near = scale[0].back * scale[0].back, back_read = scale[0].back * scale[1].back * sh.scale;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) nr[n][j] *= back_near, rd[n][j] *= back_read;
    DrGates& gates = s.gates;
    for (uint32_t h = hk * group; h < (hk + 1) * group; ++h) {
        if (t == 0) bulk_wait_read_all();  // the keys, the head before's unit
        __syncthreads();
        if (warp == 0) {  // running sums of the decays, in 64 bits: differences of long sums matter
            double v[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = lane * 2 + j;
                float d = r < c.rows && p.decay ? p.decay[(c.row + r) * p.decay_stride + h] : 0.0f;
                d = d < DR_LEAST_DECAY ? DR_LEAST_DECAY : d;
                v[j] = d;
                gates.beta[r] = r < c.rows ? p.beta[(c.row + r) * p.beta_stride + h] : 0.0f;
            }
            double sum = v[0] + v[1];
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, sum, i);
                if (lane >= i) sum += up;
            }
            const double last = __shfl_sync(0xffffffffu, sum, 31), total[2] = {sum - v[1], sum};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = lane * 2 + j;
                gates.total[r] = (float)total[j], gates.rest[r] = (float)(total[j] - (float)total[j]);
                gates.g[r] = __expf((float)total[j]), gates.e[r] = __expf((float)(last - total[j]));
            }
            if (lane == 0) gates.back_k = scale[0].back, gates.back_q = scale[1].back;
        }
        __syncthreads();
        float a[4][4], most = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (ch * 4 + n <= 2 * rb + 1) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int r = r0 + (j >> 1) * 8, cc = n * 8 + col + (j & 1);
                    const float d = __expf((gates.total[r] - gates.total[cc]) + (gates.rest[r] - gates.rest[cc]));
                    a[n][j] = cc <= r ? d * rd[n][j] : 0.0f;
                    most = fmaxf(most, fabsf(a[n][j]));
                    s.invert.m[r * DR_PITCH + cc] = cc < r ? d * nr[n][j] * gates.beta[BACKWARD ? r : cc] : 0.0f;
                }
            } else {  // the inversion does not look above the blocks of the diagonal
                a[n][0] = a[n][1] = a[n][2] = a[n][3] = 0.0f;
            }
        }
        most = warp_max(most);
        if (lane == 0) s.most[0][warp] = most;
        __syncthreads();
        dr_invert(s.invert);
        const Scale read = scale_for<40>(dr_max8(s.most[0]));
        float v[4][4];
        most = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 x = *(const float2*)&s.invert.inv[(r0 + j * 8) * DR_PITCH + n * 8 + col];
                v[n][2 * j] = x.x, v[n][2 * j + 1] = x.y;
                most = fmaxf(most, fmaxf(fabsf(x.x), fabsf(x.y)));
            }
        most = warp_max(most);
        if (lane == 0) s.most[1][warp] = most;
        __syncthreads();
        const Scale inverse = scale_for<40>(dr_max8(s.most[1]));
        if (t == 0) gates.back_inverse = inverse.back, gates.back_read = read.back;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                uint32_t hi, lo;
                uint8_t* const at = s.blocks + block_at(r0 + j * 8, n * 8 + col);
                split_f16(v[n][2 * j], v[n][2 * j + 1], inverse.by, hi, lo);
                *(uint32_t*)at = hi, *(uint32_t*)(at + DR_BLOCK) = lo;
                split_f16(a[n][2 * j], a[n][2 * j + 1], read.by, hi, lo);
                *(uint32_t*)(at + 2 * DR_BLOCK) = hi, *(uint32_t*)(at + 3 * DR_BLOCK) = lo;
            }
        fence_proxy_async_smem();
        __syncthreads();
        if (t == 0) {
            uint8_t* const to = p.units + (slot * sh.heads + h) * DR_UNIT;
            bulk_store(to, s.blocks, 4 * DR_BLOCK);
            bulk_store(to + 4 * DR_BLOCK, &s.gates, sizeof(DrGates));
            bulk_commit();
        }
    }
    if (t == 0) bulk_wait_read_all();
}

// ---- chunk after chunk ----------------------------------------------------------------------------
// Values as the caller has them ([rows][heads][value_dim]): 64 tokens x 16 of a warp's value dimensions.  2-byte rows of
// 32 bytes with their two pieces swapped every 4 rows, float32 rows of 80 bytes, against bank conflicts.
template <typename T>
constexpr int DR_RAW_ROW = sizeof(T) == 4 ? 80 : 32;
template <typename T>
constexpr int DR_RAW = DR_CHUNK * DR_RAW_ROW<T>;
template <typename T>
__device__ __forceinline__ uint32_t dr_raw_at(uint32_t tile, int row, int piece) {
    if constexpr (sizeof(T) == 4) return tile + row * 80 + piece * 16;
    else return tile + row * 32 + ((piece ^ (row >> 2 & 1)) << 4);
}
template <typename T>
__device__ __forceinline__ void dr_raw_load(uint32_t tile, const T* from, uint64_t stride, int rows, int cols, bool wide, int lane) {
    constexpr int PIECES = 2 * sizeof(T) / 2, E = 16 / sizeof(T);  // of a row; elements of one
#pragma unroll
    for (int i = 0; i < DR_CHUNK * PIECES / 32; ++i) {
        const int item = i * 32 + lane, r = item / PIECES, c = item % PIECES;
        const uint32_t at = dr_raw_at<T>(tile, r, c);
        if (wide) {
            const bool have = r < rows && c * E < cols;
            cp_async16_fill(at, have ? from + r * stride + c * E : from, have ? 16 : 0);
        } else {
            alignas(16) T v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = r < rows && c * E + j < cols ? from[r * stride + c * E + j] : narrow<T>(0.0f);
            const uint4 w = *(const uint4*)v;
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
        }
    }
}
// Transposed, tokens [token, token + 16): v[x] are the value dimensions g + 8 (x & 1) and the tokens 8 (x >> 1) + col, + 1.
template <typename T>
__device__ __forceinline__ void dr_raw_get(float (&v)[4][2], uint32_t tile, int token, int lane) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                v[x][j] = __uint_as_float(lds32(tile + (token + (x >> 1) * 8 + (lane & 3) * 2 + j) * 80 + ((lane >> 2) + (x & 1) * 8) * 4));
    } else {
        uint32_t r[4];
        const int row = token + (lane & 7) + (lane >> 4) * 8;
        ldmatrix4_t(r, dr_raw_at<T>(tile, row, lane >> 3 & 1));
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if constexpr (std::is_same_v<T, __half>) {
                const float2 f = unpack_f16(r[x]);
                v[x][0] = f.x, v[x][1] = f.y;
            } else {
                v[x][0] = __uint_as_float(r[x] << 16), v[x][1] = __uint_as_float(r[x] & 0xffff0000u);
            }
        }
    }
}

template <typename T, int DK, int WARPS>
struct DrChainSmem {
    static constexpr int PLANES = sizeof(T) == 4 ? 2 : 1;
    static constexpr int STAGE = 2 * DR_KEYS<DK, PLANES> + DR_UNIT;
    // two stages but where they do not fit beside the values
    static constexpr int STAGES = 2 * (STAGE + WARPS * DR_RAW<T>) + 64 <= 227 * 1024 ? 2 : 1;
    alignas(128) uint8_t stage[STAGES][STAGE];
    alignas(16) uint8_t raw[WARPS][2][DR_RAW<T>];
    uint64_t full[STAGES], empty[STAGES];
};

struct DrChain {
    DrShape sh;
    const uint8_t *keys, *units;
    const void* values;  // V forward, dO backward (null: zeros)
    uint64_t value_stride;
    bool wide;           // rows of values are whole 16-byte pieces
    // States before the first chunk (forward), gradients of the last ones (backward), and the states after (gradients of
    // the first), of the sequences' parts one after the other; parts > 1: `to` is of whole sequences, the end part's.
    const float* from;
    float* to;
    uint32_t parts;      // of a sequence, with about as many chunks each
    float *local, *map;  // DR_STATES: what a part makes of no state, and of each row of the unit matrix
    void* out;           // forward
    uint64_t out_stride;
    DrImage states, kept;  // S0 and w (forward, if saved), X and z (backward)
    float* back_values;    // backward: inverse scales of dO
};

template <typename T>
__device__ __forceinline__ void dr_store_pair(T* to, uint32_t col, uint32_t cols, bool pairs, float x, float y) {
    if (pairs && col + 1 < cols) {
        if constexpr (sizeof(T) == 4) *(float2*)(to + col) = make_float2(x, y);
        else if constexpr (std::is_same_v<T, __half>) *(__half2*)(to + col) = __floats2half2_rn(x, y);
        else *(__nv_bfloat162*)(to + col) = __floats2bfloat162_rn(x, y);
    } else {
        if (col < cols) to[col] = narrow<T>(x);
        if (col + 1 < cols) to[col + 1] = narrow<T>(y);
    }
}

// What a chain writes: everything, or only the states at the end of its part, for sequences in parts: part p's states
// are those before it times a key_dim x key_dim matrix plus what it makes of none.  The matrix comes from the same
// recurrence, with the unit matrix's rows for a state and without values.
enum { DR_ALL, DR_STATES };

// What both directions share: where a CTA's warps are, the copies of the chunks' images, and products with them.
template <typename T, int DK, int WARPS, bool BACKWARD, int WHAT>
struct DrChainCta {
    using Smem = DrChainSmem<T, DK, WARPS>;
    static constexpr int PLANES = Smem::PLANES, NB = DK / 64, NT = DK / 8, STAGES = Smem::STAGES, KEYS = DR_KEYS<DK, PLANES>;
    const DrChain& p;
    Smem& sm;
    const int lane, warp, g, col;
    const LaneOffsets o;
    uint32_t h, hk, seq, v0, live, row, dim;  // dim: rows of the state
    uint32_t asked = 0;  // stages' copies so far, by the thread that asks for them
    uint64_t start, end, base;
    uint32_t first, chunks;  // the part's
    const T* values;
    bool unit_rows = false, ok = true;
    const float* from;
    float* to;

    __device__ __forceinline__ DrChainCta(const DrChain& p_, Smem& sm_)
        : p(p_), sm(sm_), lane(threadIdx.x & 31), warp(threadIdx.x >> 5), g((threadIdx.x & 31) >> 2), col((threadIdx.x & 3) * 2),
          o(threadIdx.x & 31) {
        const DrShape& sh = p.sh;
        dr_let_next_start();
        const uint32_t value_slices = (sh.value_dim + WARPS * 16 - 1) / (WARPS * 16),
                       slices = value_slices + (WHAT == DR_STATES ? (sh.key_dim + WARPS * 16 - 1) / (WARPS * 16) : 0);
        const uint32_t parts = WHAT == DR_STATES ? p.parts - 1 : p.parts;  // nothing follows on the end part
        uint32_t slice = blockIdx.x % slices, rest = blockIdx.x / slices;
        h = rest % sh.heads, rest /= sh.heads;
        const uint32_t part = rest % parts + (WHAT == DR_STATES && BACKWARD ? 1 : 0);
        seq = rest / parts, hk = h / (sh.heads / sh.key_heads);
        dr_wait_for_last();
        if (sh.order) seq = sh.order[seq];
        unit_rows = slice >= value_slices;
        if (unit_rows) slice -= value_slices;
        dim = unit_rows ? sh.key_dim : sh.value_dim;
        v0 = slice * WARPS * 16;
        live = min((uint32_t)WARPS, (dim - v0 + 15) / 16);
        row = v0 + warp * 16 + g;
        start = sh.start(seq), end = min(sh.start(seq + 1), sh.rows), base = sh.base(seq);
        const uint32_t all = end > start ? (uint32_t)((end - start + DR_CHUNK - 1) / DR_CHUNK) : 0, each = (all + p.parts - 1) / p.parts;
        first = min(part * each, all), chunks = min(all - first, each);
        values = unit_rows ? nullptr : (const T*)p.values;
        const uint64_t state = (uint64_t)sh.value_dim * sh.key_dim, stream = (uint64_t)seq * sh.heads + h, piece = stream * p.parts + part;
        if (WHAT == DR_STATES) {
            from = nullptr;
            to = unit_rows ? p.map + piece * sh.key_dim * sh.key_dim : p.local + piece * state;
        } else {
            from = p.from ? p.from + piece * state : nullptr;
            to = p.to && part == (BACKWARD ? 0 : p.parts - 1) ? p.to + stream * state : nullptr;
        }
        if (threadIdx.x == 0) {
            for (int i = 0; i < STAGES; ++i) mbar_init(&sm.full[i], 1), mbar_init(&sm.empty[i], live);
            fence_mbar_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ uint32_t order(uint32_t it) const { return first + (BACKWARD ? chunks - 1 - it : it); }
    // The first images and values, and the state that they meet.
    __device__ __forceinline__ void open(float (&s)[NT][4]) {
        if (warp == 0 && lane == 0)
            for (uint32_t i = 0; i < (uint32_t)STAGES && i < chunks; ++i) load(i, order(i));
        __syncwarp();
        if (chunks) load_values(0, order(0));
        cp_async_commit();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t r = row + (j >> 1) * 8, c = n * 8 + col + (j & 1);
                s[n][j] = from && r < dim && c < p.sh.key_dim ? from[(uint64_t)r * p.sh.key_dim + c] : 0.0f;
                if (WHAT == DR_STATES && unit_rows && r == c && r < dim) s[n][j] = 1.0f;
            }
    }
    __device__ __forceinline__ void close(const float (&s)[NT][4], float by) {
        if (!ok) {  // copies under way land before the CTA's memory is another's
            cp_async_wait_all();
            for (uint32_t i = asked - min(asked, (uint32_t)STAGES); i < asked; ++i) mbar_wait(&sm.full[i % STAGES], (i / STAGES) & 1, DR_DRAIN_LIMIT);
            set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
        }
        if (!to) return;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t r = row + (j >> 1) * 8, c = n * 8 + col + (j & 1);
                if (r < dim && c < p.sh.key_dim) to[(uint64_t)r * p.sh.key_dim + c] = s[n][j] * by;
            }
    }
    // What is added to a state need not be finer than 2^-45 of it, and must not be much finer, or the state would not fit
    // the domain: a limit of its scale, from the state's largest value (times a domain) and that domain.
    static __device__ __forceinline__ float finest(float top, float back) {
        return top > 0.0f ? power_inverse(back) * 1073741824.0f : __int_as_float(0x7f000000);  // 2^30 times its scale; any
    }
    __device__ __forceinline__ uint64_t unit(uint32_t chunk) const { return (base + chunk) * p.sh.heads + h; }
    __device__ __forceinline__ uint32_t rows(uint32_t chunk) const {
        return (uint32_t)min((uint64_t)DR_CHUNK, end - start - (uint64_t)chunk * DR_CHUNK);
    }
    __device__ __forceinline__ void load(uint32_t stage, uint32_t chunk) {  // one thread
        ++asked;
        mbar_arrive_expect_tx(&sm.full[stage], Smem::STAGE);
        bulk_load(sm.stage[stage], p.keys + ((base + chunk) * p.sh.key_heads + hk) * (2 * KEYS), 2 * KEYS, &sm.full[stage]);
        bulk_load(sm.stage[stage] + 2 * KEYS, p.units + unit(chunk) * DR_UNIT, DR_UNIT, &sm.full[stage]);
    }
    __device__ __forceinline__ void load_values(uint32_t buffer, uint32_t chunk) {
        if (!values) return;
        const T* const at = values + (start + (uint64_t)chunk * DR_CHUNK) * p.value_stride + (uint64_t)h * p.sh.value_dim + v0 + warp * 16;
        dr_raw_load<T>(smem_u32(sm.raw[warp][buffer]), at, p.value_stride, rows(chunk), (int)(p.sh.value_dim - v0) - warp * 16, p.wide, lane);
    }
    // Step `it` is chunk order(it).  Waits for its values and images, and asks for the next values.
    __device__ __forceinline__ bool begin(uint32_t it) {
        cp_async_wait_all();
        __syncwarp();
        if (it + 1 < chunks) load_values((it + 1) & 1, order(it + 1));
        cp_async_commit();
        ok = __all_sync(0xffffffffu, dr_wait(&sm.full[it % STAGES], (it / STAGES) & 1));
        return ok;
    }
    // Two stages: the next images are asked for amid a step, when the other warps have left the step before.
    __device__ __forceinline__ void ahead(uint32_t it) {
        if (STAGES == 2 && warp == 0 && lane == 0 && it + 1 < chunks && it >= 1) {
            if (dr_wait(&sm.empty[(it + 1) & 1], ((it - 1) / 2) & 1)) load((it + 1) & 1, order(it + 1));
            else set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
        }
        __syncwarp();
    }
    __device__ __forceinline__ void finish(uint32_t it) {
        __syncwarp();
        if (lane == 0) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sm.empty[it % STAGES])) : "memory");
            if (STAGES == 1 && warp == 0 && it + 1 < chunks) {
                if (dr_wait(&sm.empty[0], it & 1)) load(0, order(it + 1));
                else set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
            }
        }
        __syncwarp();
    }
    // A sum takes its next product some 24 cycles after the last, three issues of products: all tiles take one before any
    // takes the next.
    // c (16 x 64: value x token) += s (16 x 16 kk .. 16 kk + 16) K^T
    __device__ __forceinline__ void times_keys(float (&c)[8][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], uint32_t k, int kk) const {
#pragma unroll
        for (int i = 0; i < PLANES; ++i) {
            uint32_t b[4][4];
#pragma unroll
            for (int n = 0; n < 4; ++n) load_b(b[n], k + (i * NB + (kk >> 2)) * DR_BLOCK, n * 16, kk & 3, o);
#pragma unroll
            for (int n = 0; n < 4; ++n) mma_f16_2(c[2 * n], c[2 * n + 1], hi, b[n]);
            if (i == 0) {
#pragma unroll
                for (int n = 0; n < 4; ++n) mma_f16_2(c[2 * n], c[2 * n + 1], lo, b[n]);
            }
        }
    }
    // s (16 x DK) += a (16 x tokens 16 kt .. 16 kt + 16) times the rows of K or Q
    __device__ __forceinline__ void add_outer(float (&s)[NT][4], const uint32_t (&hi)[4], const uint32_t (&lo)[4], uint32_t tile, int kt) const {
#pragma unroll
        for (int i = 0; i < PLANES; ++i)
#pragma unroll
            for (int m = 0; m < DK / 64; ++m) {
                uint32_t b[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) load_b_t(b[n], tile + (i * NB + m) * DR_BLOCK, kt * 16, n, o);
#pragma unroll
                for (int n = 0; n < 4; ++n) mma_f16_2(s[8 * m + 2 * n], s[8 * m + 2 * n + 1], hi, b[n]);
                if (i == 0) {
#pragma unroll
                    for (int n = 0; n < 4; ++n) mma_f16_2(s[8 * m + 2 * n], s[8 * m + 2 * n + 1], lo, b[n]);
                }
            }
    }
    // Where the thread's elements of an image with `blocks` blocks a row lie, but for the piece of 8 columns, whose number's
    // bits 4 .. 6 are exclusive or-ed with (its rows g and g + 8 permute alike).
    __device__ __forceinline__ uint8_t* mine(uint8_t* image, uint32_t blocks) const {
        return image + (row >> 5) * (2 * blocks * DR_PIECE) + (row & 31) * BLOCK_ROW + (g << 4) + col * 2;
    }
    static __device__ __forceinline__ uint32_t* piece(uint8_t* at, int number) { return (uint32_t*)((uintptr_t)at ^ (uintptr_t)(number << 4)); }
    // The fragment of columns 16 kk .. of the warp's 16 rows to an image, from mine().
    template <int BLOCKS>
    static __device__ __forceinline__ void keep(uint8_t* at, const uint32_t (&hi)[4], const uint32_t (&lo)[4], int kk) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t* const to = piece(at, (kk & 3) * 2 + (j >> 1)) + ((kk >> 2) * DR_PIECE + (j & 1) * 8 * BLOCK_ROW) / 4;
            to[0] = hi[j];
            to[BLOCKS * DR_PIECE / 4] = lo[j];
        }
    }
    __device__ __forceinline__ void keep_back(float* back, uint64_t unit, float v) const {
        if (lane == 0) back[unit * 8 + (v0 >> 4) + warp] = v;
    }
};

// Bound by latency: a warp's products wait for the last ones' sums (13 ns each) and for their operands, with one or two warps
// a scheduler.  Counters with 8 warps: issue slots 37 %, tensor pipe 31 %, shared memory 40 %; with 2: 29 and 12 %.  Two
// CTAs an SM, for which 64 key columns leave room with one stage of images each, took 523 us instead of 450 over 256
// packed sequences: the copies are no longer ahead.
template <typename T, int DK, int WARPS, int WHAT>
__global__ void __launch_bounds__(WARPS * 32, 1)
dr_forward_kernel(const __grid_constant__ DrChain p) {
    using Cta = DrChainCta<T, DK, WARPS, false, WHAT>;
    constexpr bool ALL = WHAT == DR_ALL;
    constexpr int NT = Cta::NT, NB = Cta::NB, PLANES = Cta::PLANES, KEYS = Cta::KEYS;
    constexpr bool FINE = !std::is_same_v<T, __nv_bfloat16>;  // outputs of 8 bits need one part of the state and of u (11 bits)
    extern __shared__ __align__(128) uint8_t dr_smem[];
    Cta cta(p, *(typename Cta::Smem*)dr_smem);
    const int lane = cta.lane, warp = cta.warp, g = cta.g, col = cta.col;
    const LaneOffsets& o = cta.o;
    if (warp >= (int)cta.live) return;
    float s[NT][4];  // the state times a power of two
    float back_domain = 1.0f;
    cta.open(s);
    T* const out = (T*)p.out + (uint64_t)cta.h * p.sh.value_dim;
    const bool pairs = ((uintptr_t)p.out | p.out_stride * sizeof(T) | p.sh.value_dim * sizeof(T)) % (2 * sizeof(T)) == 0;
    for (uint32_t it = 0; it < cta.chunks; ++it) {
        if (!cta.begin(it)) break;
        const uint32_t stage = smem_u32(cta.sm.stage[it % Cta::STAGES]), k = stage, q = stage + KEYS, inv = stage + 2 * KEYS,
                       rd = inv + 2 * DR_BLOCK;
        const DrGates& gt = *(const DrGates*)(cta.sm.stage[it % Cta::STAGES] + 2 * KEYS + 4 * DR_BLOCK);
        const uint64_t unit = cta.unit(cta.order(it));
        // r = S0 K^T (value x token) and out = Q S0^T (token x value)
        float r[8][4] = {}, y[4][2][4] = {};
        const float top = max_abs(s);
        const Scale ss = coarse_scale_for(top, back_domain);
        uint8_t* const states = ALL && p.states.at ? cta.mine(p.states.of(unit), NB) : nullptr;
        if (states) cta.keep_back(p.states.back, unit, kept_back(top, ss.back * back_domain));
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t hi[4], lo[4];
            split_block(s[2 * kk], s[2 * kk + 1], ss.by, hi, lo);
            if (states) Cta::template keep<NB>(states, hi, lo, kk);
            cta.times_keys(r, hi, lo, k, kk);
#pragma unroll
            for (int i = 0; ALL && i < PLANES; ++i) {
                uint32_t a[4][4];
#pragma unroll
                for (int m = 0; m < 4; ++m) load_a(a[m], q + (i * NB + (kk >> 2)) * DR_BLOCK, m * 16, kk & 3, o);
#pragma unroll
                for (int m = 0; m < 4; ++m) mma_f16(y[m][0], a[m], hi[0], hi[2]), mma_f16(y[m][1], a[m], hi[1], hi[3]);
                if (FINE && i == 0) {
#pragma unroll
                    for (int m = 0; m < 4; ++m) mma_f16(y[m][0], a[m], lo[0], lo[2]), mma_f16(y[m][1], a[m], lo[1], lo[3]);
                }
            }
        }
        const float back_state = ss.back * back_domain, finest = Cta::finest(top, back_state);
        // r = V - g S0 K^T
        const uint32_t raw = smem_u32(cta.sm.raw[warp][it & 1]);
        const float back_r = -back_state * gt.back_k;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            float v[4][2] = {};
            if (ALL || cta.values) dr_raw_get<T>(v, raw, n * 16, lane);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 gate = *(const float2*)&gt.g[n * 16 + (x >> 1) * 8 + col];
                float* const d = &r[2 * n + (x >> 1)][(x & 1) * 2];
                pair_split(pair_fma(pair_mul(pair_of(gate.x, gate.y), pair_of(back_r, back_r)), pair_of(d[0], d[1]), pair_of(v[x][0], v[x][1])), d[0], d[1]);
            }
        }
        cta.ahead(it);
        // w = r inverse^T
        const Scale sr = scale_for(max_abs(r));
        float w[8][4] = {};
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(r[2 * kt], r[2 * kt + 1], sr.by, hi, lo);
            uint32_t b[4][4];
#pragma unroll
            for (int n = kt; n < 4; ++n) load_b(b[n], inv, n * 16, kt, o);
#pragma unroll
            for (int n = kt; n < 4; ++n) mma_f16_2(w[2 * n], w[2 * n + 1], hi, b[n]);
#pragma unroll
            for (int n = kt; n < 4; ++n) mma_f16_2(w[2 * n], w[2 * n + 1], lo, b[n]);
#pragma unroll
            for (int n = kt; n < 4; ++n) load_b(b[n], inv + DR_BLOCK, n * 16, kt, o);
#pragma unroll
            for (int n = kt; n < 4; ++n) mma_f16_2(w[2 * n], w[2 * n + 1], hi, b[n]);
        }
        const float back_w = sr.back * gt.back_inverse;
        if (ALL && p.kept.at) {
            const float most = max_abs(w);
            const Scale sw = coarse_scale_for(most, back_w);
            uint8_t* const kept = cta.mine(p.kept.of(unit), 1);
            cta.keep_back(p.kept.back, unit, kept_back(most, sw.back * back_w));
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t hi[4], lo[4];
                split_block(w[2 * kt], w[2 * kt + 1], sw.by, hi, lo);
                Cta::template keep<1>(kept, hi, lo, kt);
            }
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {  // u
            const float2 b = *(const float2*)&gt.beta[n * 8 + col];
            const uint64_t by = pair_mul(pair_of(b.x, b.y), pair_of(back_w, back_w));
            scale_pair(w[n][0], w[n][1], by), scale_pair(w[n][2], w[n][3], by);
        }
        if constexpr (ALL) {  // out = scale g out + A u
            const Scale su = scale_up_to(scale_for(max_abs(w)), finest);
            {
                const float by = p.sh.scale * back_state * gt.back_q, into = su.by * power_inverse(gt.back_read);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const float g0 = gt.g[m * 16 + g] * by * into, g1 = gt.g[m * 16 + g + 8] * by * into;
#pragma unroll
                    for (int n = 0; n < 2; ++n) scale_pair(y[m][n][0], y[m][n][1], pair_of(g0, g0)), scale_pair(y[m][n][2], y[m][n][3], pair_of(g1, g1));
                }
            }
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t hi[4], lo[4];
                split_block(w[2 * kt], w[2 * kt + 1], su.by, hi, lo);
                uint32_t a[4][4];
#pragma unroll
                for (int m = kt; m < 4; ++m) load_a(a[m], rd, m * 16, kt, o);
#pragma unroll
                for (int m = kt; m < 4; ++m) mma_f16(y[m][0], a[m], hi[0], hi[2]), mma_f16(y[m][1], a[m], hi[1], hi[3]);
                if constexpr (FINE) {
#pragma unroll
                    for (int m = kt; m < 4; ++m) mma_f16(y[m][0], a[m], lo[0], lo[2]), mma_f16(y[m][1], a[m], lo[1], lo[3]);
#pragma unroll
                    for (int m = kt; m < 4; ++m) load_a(a[m], rd + DR_BLOCK, m * 16, kt, o);
#pragma unroll
                    for (int m = kt; m < 4; ++m) mma_f16(y[m][0], a[m], hi[0], hi[2]), mma_f16(y[m][1], a[m], hi[1], hi[3]);
                }
            }
            {
                const float back = su.back * gt.back_read;
                const uint32_t have = cta.rows(cta.order(it));
                T* const first = out + (cta.start + (uint64_t)cta.order(it) * DR_CHUNK + g) * p.out_stride;
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (m * 16 + j * 8 + g >= have) continue;
                        T* const to = first + (m * 16 + j * 8) * p.out_stride;
#pragma unroll
                        for (int n = 0; n < 2; ++n)
                            dr_store_pair(to, cta.v0 + warp * 16 + n * 8 + col, p.sh.value_dim, pairs, y[m][n][2 * j] * back, y[m][n][2 * j + 1] * back);
                    }
            }
        }
        // S = g_64 S + (e u)^T K, in the domain of the product
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 e = *(const float2*)&gt.e[n * 8 + col];
            scale_pair(w[n][0], w[n][1], pair_of(e.x, e.y)), scale_pair(w[n][2], w[n][3], pair_of(e.x, e.y));
        }
        const Scale se = scale_up_to(scale_for(max_abs(w)), finest);
        const float into = se.by * power_inverse(gt.back_k), whole = gt.g[DR_CHUNK - 1] * (back_domain * into);
        back_domain = se.back * gt.back_k;
        scale_all(s, whole);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(w[2 * kt], w[2 * kt + 1], se.by, hi, lo);
            cta.add_outer(s, hi, lo, k, kt);
        }
        cta.finish(it);
    }
    cta.close(s, back_domain);
}

// As the forward chain (issue slots 35 %, tensor pipe 36 %).
template <typename T, int DK, int WARPS, int WHAT>
__global__ void __launch_bounds__(WARPS * 32, 1)
dr_backward_kernel(const __grid_constant__ DrChain p) {
    using Cta = DrChainCta<T, DK, WARPS, true, WHAT>;
    constexpr bool ALL = WHAT == DR_ALL;
    constexpr int NT = Cta::NT, KEYS = Cta::KEYS;
    constexpr bool EXACT = sizeof(T) == 2;  // dO in one part
    extern __shared__ __align__(128) uint8_t dr_smem[];
    Cta cta(p, *(typename Cta::Smem*)dr_smem);
    const int lane = cta.lane, warp = cta.warp, col = cta.col;
    const LaneOffsets& o = cta.o;
    if (warp >= (int)cta.live) return;
    float x[NT][4];  // the state's gradient times a power of two
    float back_domain = 1.0f;
    cta.open(x);
    for (uint32_t it = 0; it < cta.chunks; ++it) {
        if (!cta.begin(it)) break;
        const uint32_t stage = smem_u32(cta.sm.stage[it % Cta::STAGES]), k = stage, q = stage + KEYS, inv = stage + 2 * KEYS,
                       rd = inv + 2 * DR_BLOCK;
        const DrGates& gt = *(const DrGates*)(cta.sm.stage[it % Cta::STAGES] + 2 * KEYS + 4 * DR_BLOCK);
        const uint64_t unit = cta.unit(cta.order(it));
        const uint32_t raw = smem_u32(cta.sm.raw[warp][it & 1]);
        // du = e X K^T (value x token)
        float du[8][4] = {};
        const float top = max_abs(x);
        const Scale sx = coarse_scale_for(top, back_domain);
        const float finest = Cta::finest(top, sx.back * back_domain);
        uint8_t* const states = ALL ? cta.mine(p.states.of(unit), Cta::NB) : nullptr;
        if constexpr (ALL) cta.keep_back(p.states.back, unit, kept_back(top, sx.back * back_domain));
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t hi[4], lo[4];
            split_block(x[2 * kk], x[2 * kk + 1], sx.by, hi, lo);
            if constexpr (ALL) Cta::template keep<Cta::NB>(states, hi, lo, kk);
            cta.times_keys(du, hi, lo, k, kk);
        }
        // ... + dO^T A
        float most = 0.0f, most_g = 0.0f;
        if (cta.values) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                float v[4][2];
                dr_raw_get<T>(v, raw, kt * 16, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 gate = *(const float2*)&gt.g[kt * 16 + (j >> 1) * 8 + col];
                    most = fmaxf(most, fmaxf(fabsf(v[j][0]), fabsf(v[j][1])));
                    most_g = fmaxf(most_g, fmaxf(fabsf(v[j][0] * gate.x), fabsf(v[j][1] * gate.y)));
                }
            }
        }
        most = warp_max(most);
        // beside X only what may be added to it counts; the gradients of q, which have dO alone, want its own scale
        const Scale own = coarse_scale_for(most), so = scale_up_to(own, finest), sg = scale_up_to(scale_for(warp_max(most_g) * fabsf(p.sh.scale)), finest);
        if constexpr (ALL) cta.keep_back(p.back_values, unit, kept_back(most, own.back));
        {
            const float back = (sx.back * back_domain * gt.back_k) * (so.by * power_inverse(gt.back_read));
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const float2 e = *(const float2*)&gt.e[n * 8 + col];
                const uint64_t by = pair_mul(pair_of(e.x, e.y), pair_of(back, back));
                scale_pair(du[n][0], du[n][1], by), scale_pair(du[n][2], du[n][3], by);
            }
        }
        if (cta.values) {
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                float v[4][2];
                uint32_t hi[4], lo[4];
                dr_raw_get<T>(v, raw, kt * 16, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) split_f16(v[j][0], v[j][1], so.by, hi[j], lo[j]);
                uint32_t b[4][4];
#pragma unroll
                for (int n = 0; n <= kt; ++n) load_b_t(b[n], rd, kt * 16, n, o);
#pragma unroll
                for (int n = 0; n <= kt; ++n) mma_f16_2(du[2 * n], du[2 * n + 1], hi, b[n]);
                if constexpr (!EXACT) {
#pragma unroll
                    for (int n = 0; n <= kt; ++n) mma_f16_2(du[2 * n], du[2 * n + 1], lo, b[n]);
                }
#pragma unroll
                for (int n = 0; n <= kt; ++n) load_b_t(b[n], rd + DR_BLOCK, kt * 16, n, o);
#pragma unroll
                for (int n = 0; n <= kt; ++n) mma_f16_2(du[2 * n], du[2 * n + 1], hi, b[n]);
            }
        }
        cta.ahead(it);
        // z = du inverse
        const Scale sd = scale_for(max_abs(du));
        float z[8][4] = {};
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(du[2 * kt], du[2 * kt + 1], sd.by, hi, lo);
            uint32_t b[4][4];
#pragma unroll
            for (int n = 0; n <= kt; ++n) load_b_t(b[n], inv, kt * 16, n, o);
#pragma unroll
            for (int n = 0; n <= kt; ++n) mma_f16_2(z[2 * n], z[2 * n + 1], hi, b[n]);
#pragma unroll
            for (int n = 0; n <= kt; ++n) mma_f16_2(z[2 * n], z[2 * n + 1], lo, b[n]);
#pragma unroll
            for (int n = 0; n <= kt; ++n) load_b_t(b[n], inv + DR_BLOCK, kt * 16, n, o);
#pragma unroll
            for (int n = 0; n <= kt; ++n) mma_f16_2(z[2 * n], z[2 * n + 1], hi, b[n]);
        }
        const float back_z = sd.back * gt.back_inverse * so.back * gt.back_read;
        if constexpr (ALL) {
            const float most_z = max_abs(z);
            const Scale sz = coarse_scale_for(most_z, back_z);
            uint8_t* const kept = cta.mine(p.kept.of(unit), 1);
            cta.keep_back(p.kept.back, unit, kept_back(most_z, sz.back * back_z));
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                uint32_t hi[4], lo[4];
                split_block(z[2 * kt], z[2 * kt + 1], sz.by, hi, lo);
                Cta::template keep<1>(kept, hi, lo, kt);
            }
        }
        // X = g_64 X + (scale g dO)^T Q - (g beta z)^T K, each in the domain of its product
        float into = back_domain;
        if (cta.values) {
            into = gt.g[DR_CHUNK - 1] * (into * (sg.by * power_inverse(gt.back_q)));
            scale_all(x, into);
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                float v[4][2];
                uint32_t hi[4], lo[4];
                dr_raw_get<T>(v, raw, kt * 16, lane);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 gate = *(const float2*)&gt.g[kt * 16 + (j >> 1) * 8 + col];
                    split_f16(v[j][0] * (gate.x * p.sh.scale), v[j][1] * (gate.y * p.sh.scale), sg.by, hi[j], lo[j]);
                }
                cta.add_outer(x, hi, lo, q, kt);
            }
            into = sg.back * gt.back_q;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const float2 gate = *(const float2*)&gt.g[n * 8 + col], b = *(const float2*)&gt.beta[n * 8 + col];
            const uint64_t by = pair_of(-gate.x * b.x * back_z, -gate.y * b.y * back_z);
            scale_pair(z[n][0], z[n][1], by), scale_pair(z[n][2], z[n][3], by);
        }
        const Scale sy = scale_up_to(scale_for(max_abs(z)), finest);
        into *= sy.by * power_inverse(gt.back_k);
        if (!cta.values) into *= gt.g[DR_CHUNK - 1];
        back_domain = sy.back * gt.back_k;
        scale_all(x, into);
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) {
            uint32_t hi[4], lo[4];
            split_block(z[2 * kt], z[2 * kt + 1], sy.by, hi, lo);
            cta.add_outer(x, hi, lo, k, kt);
        }
        cta.finish(it);
    }
    cta.close(x, back_domain);
}

// The states before each part of a sequence: through the parts in order, a CTA with 8 rows of a state and all its columns.
// The maps come from L2, 16 loads ahead: 16 heads of one sequence of 65536 tokens 78 us (32 loads ahead in registers of
// their own 141; rows of the state by 16-byte reads 113).
constexpr int DR_JOIN_ROWS = 8;
struct DrJoin {
    const float *first, *local, *map;  // first: null for zeros
    float* before;
    uint32_t heads, key_dim, value_dim, parts, slices;
    bool backward;  // the end part first
};
__global__ void __launch_bounds__(128) dr_join_kernel(const __grid_constant__ DrJoin p) {
    __shared__ float s[DR_JOIN_ROWS][DR_MAX_DIM];
    dr_let_next_start();
    dr_wait_for_last();
    const uint32_t slice = blockIdx.x % p.slices, r0 = slice * DR_JOIN_ROWS, c = threadIdx.x;
    const uint64_t stream = blockIdx.x / p.slices, size = (uint64_t)p.value_dim * p.key_dim;
    float mine[DR_JOIN_ROWS];
#pragma unroll
    for (int i = 0; i < DR_JOIN_ROWS; ++i)
        mine[i] = p.first && c < p.key_dim && r0 + i < p.value_dim ? p.first[stream * size + (uint64_t)(r0 + i) * p.key_dim + c] : 0.0f;
    for (uint32_t k = 0; k < p.parts; ++k) {
        const uint64_t piece = stream * p.parts + (p.backward ? p.parts - 1 - k : k);
#pragma unroll
        for (int i = 0; i < DR_JOIN_ROWS; ++i)
            if (c < p.key_dim && r0 + i < p.value_dim) p.before[piece * size + (uint64_t)(r0 + i) * p.key_dim + c] = mine[i];
        if (k + 1 == p.parts) break;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < DR_JOIN_ROWS; ++i) s[i][c] = mine[i];
        __syncthreads();
        if (c < p.key_dim) {
#pragma unroll
            for (int i = 0; i < DR_JOIN_ROWS; ++i) mine[i] = r0 + i < p.value_dim ? p.local[piece * size + (uint64_t)(r0 + i) * p.key_dim + c] : 0.0f;
            const float* const map = p.map + piece * p.key_dim * p.key_dim + c;
#pragma unroll 16
            for (uint32_t j = 0; j < p.key_dim; ++j) {
                const float m = map[(uint64_t)j * p.key_dim];
#pragma unroll
                for (int i = 0; i < DR_JOIN_ROWS; ++i) mine[i] = fmaf(s[i][j], m, mine[i]);
            }
        }
    }
}

// ---- gradients of the inputs ------------------------------------------------------------------------
constexpr int DR_GRAD_THREADS = 512;  // warps: 4 blocks of 16 tokens x 4 parts of the key columns
// 64 tokens x 32 of the value dimensions of dO: rows of 64 bytes with permuted pieces, float32 rows of 144 bytes.
template <typename T>
constexpr int DR_SLAB_ROW = sizeof(T) == 4 ? 144 : 64;
template <typename T>
__device__ __forceinline__ uint32_t dr_slab_at(uint32_t slab, int row, int piece) {
    if constexpr (sizeof(T) == 4) return slab + row * 144 + piece * 16;
    else return slab + row * 64 + ((piece ^ (row >> 1 & 3)) << 4);
}
template <typename T, int DK>
struct DrGradientSmem {
    static constexpr int PLANES = sizeof(T) == 4 ? 2 : 1, NB = DK / 64;
    static constexpr int STATE = 2 * NB * DR_PIECE, KEPT = 2 * DR_PIECE, STEP = 2 * STATE + 2 * KEPT;  // S, X, w, z
    alignas(128) uint8_t keys[2 * DR_KEYS<DK, PLANES>];
    alignas(128) uint8_t step[2][STEP];
    alignas(128) uint8_t slab[2][DR_CHUNK * DR_SLAB_ROW<T>];
    alignas(128) uint8_t da[2 * DR_BLOCK];  // two planes
    uint8_t dn[2 * DR_BLOCK];
    alignas(128) DrGates gates[2];     // of a head and the next
    alignas(32) float back[2][5][8];   // inverse scales of S, X, w, z and dO by 16 value dimensions
    float dbeta[2][DR_CHUNK];
    float scales[16][5];               // of a warp's products over the value dimensions
    float dot[4][DR_CHUNK], carry[4][DR_CHUNK], sx[16];
    alignas(16) float most[2][16];
    uint64_t full[2], empty[2], keys_full;
    uint32_t asked;  // steps whose copies were asked for
};

struct DrGradient {
    DrShape sh;
    const uint8_t *keys, *units;
    const void* out;  // dO, or null
    uint64_t out_stride;
    bool wide;
    DrImage s, w, x, z;
    const float* back_out;
    void *dq, *dk, *dv;
    float *ddecay, *dbeta;
    bool pairs_k, pairs_v;  // elements 2 i and 2 i + 1 of a row can be stored together: of dq and dk, of dv
};

// A CTA a chunk and key head: 32 value dimensions a step with the next step's images on their way (a step's two buffers are
// handed over by barriers in memory, so that warps need not meet), then what the key columns need of all of them.  Bound by
// shared memory (46 % of its pipe's cycles), the tensor pipe (32 %) and what each warp waits between: 579 us for 8 x 2048
// tokens and 16 heads of 128 x 128, of which about 235 are outside the steps.  16 warps were chosen when warps met after each
// step (1424 us for the whole pass, 1515 with 8 warps of twice the columns); as the buffers are handed over now 8 have not been
// compared.
template <typename T, int DK, bool SHARED>  // SHARED: several heads a key head
__global__ void __launch_bounds__(DR_GRAD_THREADS, 1)
dr_gradient_kernel(const __grid_constant__ DrGradient p) {
    using Smem = DrGradientSmem<T, DK>;
    constexpr int PLANES = Smem::PLANES, NB = Smem::NB, NT = DK / 32, NP = DK / 64;  // (pairs of) tiles of 8 key columns a warp has
    constexpr bool EXACT = sizeof(T) == 2;
    extern __shared__ __align__(128) uint8_t dr_smem[];
    auto& sm = *(Smem*)dr_smem;
    const DrShape& sh = p.sh;
    dr_let_next_start();
    dr_wait_for_last();
    const uint64_t slot = blockIdx.x / sh.key_heads;
    const uint32_t hk = blockIdx.x % sh.key_heads, group = sh.heads / sh.key_heads, h0 = hk * group;
    const DrChunk c(sh, slot);
    if (!c.rows) return;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, rb = warp >> 2, cq = warp & 3, g = lane >> 2, col = (lane & 3) * 2;
    const LaneOffsets o(lane);
    const uint32_t groups = (sh.value_dim + 15) / 16, steps = (groups + 1) / 2, total = steps * group;
    bool ok = true;
    auto load = [&](uint32_t it) {  // one thread
        const uint64_t unit = slot * sh.heads + h0 + it / steps;
        const uint32_t v = it % steps;
        uint8_t* const to = sm.step[it & 1];
        sm.asked = it + 1;
        const bool first = v == 0;  // the head's gates and scales come along
        mbar_arrive_expect_tx(&sm.full[it & 1], Smem::STEP + (first ? (uint32_t)sizeof(DrGates) + 5 * 32 : 0));
        if (first) {
            const uint32_t at = it / steps & 1;
            bulk_load(&sm.gates[at], p.units + unit * DR_UNIT + 4 * DR_BLOCK, sizeof(DrGates), &sm.full[it & 1]);
            const float* const back[5] = {p.s.back, p.x.back, p.w.back, p.z.back, p.back_out};
#pragma unroll
            for (int i = 0; i < 5; ++i) bulk_load(sm.back[at][i], back[i] + unit * 8, 32, &sm.full[it & 1]);
        }
        bulk_load(to, p.s.of(unit) + v * Smem::STATE, Smem::STATE, &sm.full[it & 1]);
        bulk_load(to + Smem::STATE, p.x.of(unit) + v * Smem::STATE, Smem::STATE, &sm.full[it & 1]);
        bulk_load(to + 2 * Smem::STATE, p.w.of(unit) + v * Smem::KEPT, Smem::KEPT, &sm.full[it & 1]);
        bulk_load(to + 2 * Smem::STATE + Smem::KEPT, p.z.of(unit) + v * Smem::KEPT, Smem::KEPT, &sm.full[it & 1]);
    };
    auto load_out = [&](uint32_t it) {
        if (!p.out) return;
        constexpr int E = 16 / sizeof(T), PIECES = 32 / E;
        const uint32_t v0 = it % steps * 32, slab = smem_u32(sm.slab[it & 1]);
        const T* const from = (const T*)p.out + c.row * p.out_stride + (uint64_t)(h0 + it / steps) * sh.value_dim + v0;
        for (int item = t; item < DR_CHUNK * PIECES; item += DR_GRAD_THREADS) {
            const uint32_t r = item / PIECES, e = item % PIECES * E;
            const uint32_t at = dr_slab_at<T>(slab, r, item % PIECES);
            if (p.wide) {
                const bool have = r < c.rows && v0 + e < sh.value_dim;
                cp_async16_fill(at, have ? from + r * p.out_stride + e : from, have ? 16 : 0);
            } else {
                alignas(16) T w[E];
#pragma unroll
                for (int j = 0; j < E; ++j) w[j] = r < c.rows && v0 + e + j < sh.value_dim ? from[r * p.out_stride + e + j] : narrow<T>(0.0f);
                const uint4 q = *(const uint4*)w;
                asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(q.x), "r"(q.y), "r"(q.z), "r"(q.w) : "memory");
            }
        }
        // arrives when the thread's copies have landed, or now that it has stored
        const uint32_t bar = smem_u32(&sm.full[it & 1]);
        if (p.wide) asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
        else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
    };
    if (t == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(&sm.full[i], 1 + (p.out ? DR_GRAD_THREADS : 0)), mbar_init(&sm.empty[i], DR_GRAD_THREADS / 32);
        mbar_init(&sm.keys_full, 1);
        fence_mbar_init();
    }
    __syncthreads();
    if (t == 0) {
        mbar_arrive_expect_tx(&sm.keys_full, 2 * DR_KEYS<DK, PLANES>);
        bulk_load(sm.keys, p.keys + (slot * sh.key_heads + hk) * (2 * DR_KEYS<DK, PLANES>), 2 * DR_KEYS<DK, PLANES>, &sm.keys_full);
        load(0);
    }
    load_out(0);
    const uint32_t k = smem_u32(sm.keys), q = k + DR_KEYS<DK, PLANES>, da = smem_u32(sm.da), dn = smem_u32(sm.dn);
    float all_q[SHARED ? NT : 1][4] = {}, all_k[SHARED ? NT : 1][4] = {};  // sums over the key head's heads
    const uint32_t token = rb * 16 + g;
    uint32_t it = 0;
    for (uint32_t h = h0; h < h0 + group; ++h) {
        const DrGates& gates = sm.gates[(h - h0) & 1];
        const float(&back)[5][8] = sm.back[(h - h0) & 1];
        enum { S, X, W, Z, GO };
        // The scales of dO S0, z S0, w X, dO w and z w: that of all 16 value dimensions which have any, or 1 where they differ
        // (uneven): their products are added in float32 then, each by its own.
        float* const unit = sm.scales[warp];
        uint32_t uneven = 0;
        float dq[NT][4] = {}, er[NT][4] = {}, wr[NT][4] = {}, a[2][4] = {}, n[2][4] = {};
        float sx = 0.0f;
        for (uint32_t v = 0; v < steps; ++v, ++it) {
            if (it + 1 < total) {  // into the buffers that the warps left a step ago
                if (it) ok = ok && dr_wait(&sm.empty[(it + 1) & 1], ((it - 1) >> 1) & 1);
                if (ok) {  // a thread that gave up asks for nothing more and waits for nothing; the others give up in their turn
                    if (t == 0) load(it + 1);
                    load_out(it + 1);
                }
            }
            if (it == 0) ok = ok && dr_wait(&sm.keys_full, 0);
            ok = ok && dr_wait(&sm.full[it & 1], (it >> 1) & 1);
            __syncwarp();
            if (v == 0) {
                const int at = lane & 7;
                const bool have = at < (int)groups;
                const float x[5] = {back[GO][at], back[Z][at], back[W][at], back[GO][at], back[Z][at]},
                            y[5] = {back[S][at], back[S][at], back[X][at], back[W][at], back[W][at]};
#pragma unroll
                for (int i = 0; i < 5; ++i) {
                    const float mine = x[i] * y[i], largest = warp_max(have ? mine : 0.0f);
                    const bool differ = __any_sync(0xffffffffu, have && x[i] != 0.0f && y[i] != 0.0f && mine != largest);
                    if (lane == 0) unit[i] = differ ? 1.0f : largest;
                    uneven |= (uint32_t)differ << i;
                }
                __syncwarp();
            }
            // c0, c1 += the i-th product over the value dimensions 16 at .. with the scales of x and y
            auto add = [&](int i, float (&c0)[4], float (&c1)[4], int x, int y, uint32_t at, auto&& products) {
                if (!(uneven >> i & 1)) {
                    products(c0, c1);
                    return;
                }
                float d0[4] = {}, d1[4] = {};
                products(d0, d1);
                const float by = back[x][at], then = back[y][at];
#pragma unroll
                for (int j = 0; j < 4; ++j) c0[j] = fmaf(d0[j] * by, then, c0[j]), c1[j] = fmaf(d1[j] * by, then, c1[j]);
            };
            const uint8_t* const step = sm.step[it & 1];
            const float beta0 = gates.beta[token], beta1 = gates.beta[token + 8];
            T* const dv0 = (T*)p.dv + ((c.row + token) * sh.heads + h) * sh.value_dim;
            T* const dv1 = dv0 + 8ull * sh.heads * sh.value_dim;
            const uint32_t s = smem_u32(step), x = s + Smem::STATE, w = x + Smem::STATE, z = w + Smem::KEPT,
                           slab = smem_u32(sm.slab[it & 1]);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const uint32_t at = v * 2 + kt;  // 16 value dimensions
                if (at >= groups) break;
                uint32_t go[2][4], aw[2][4], zt[2][4];
                if (p.out) {
                    const float by = power_inverse(back[GO][at]);
                    if constexpr (EXACT) {
                        uint32_t r[4];
                        ldmatrix4(r, dr_slab_at<T>(slab, rb * 16 + (lane & 15), kt * 2 + (lane >> 4)));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float2 f;
                            if constexpr (std::is_same_v<T, __half>) f = unpack_f16(r[j]);
                            else f = make_float2(__uint_as_float(r[j] << 16), __uint_as_float(r[j] & 0xffff0000u));
                            go[0][j] = pack_f16(f.x * by, f.y * by);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t f = slab + (rb * 16 + g + (j & 1) * 8) * 144 + (kt * 16 + (j >> 1) * 8 + col) * 4;
                            split_f16(__uint_as_float(lds32(f)), __uint_as_float(lds32(f + 4)), by, go[0][j], go[1][j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    load_a_t(aw[i], w + i * DR_PIECE, kt * 16, rb, o);
                    load_a_t(zt[i], z + i * DR_PIECE, kt * 16, rb, o);
                }
                if (cq == (int)(at & 3)) {  // dv = beta z
                    const float back_z = back[Z][at];
                    const uint32_t vcol = at * 16 + col;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t r = token + (j & 1) * 8;
                        const float b = (j & 1 ? beta1 : beta0) * back_z;
                        const float2 hi = unpack_f16(zt[0][j]), lo = unpack_f16(zt[1][j]);
                        if (r < c.rows)
                            dr_store_pair((j & 1) ? dv1 : dv0, vcol + (j >> 1) * 8, sh.value_dim, p.pairs_v, b * (hi.x + lo.x), b * (hi.y + lo.y));
                    }
                }
                if (cq <= rb) {  // 16 of the other tokens
                    uint32_t b[2][4];
                    load_b_t(b[0], w, kt * 16, cq, o);
                    load_b_t(b[1], w + DR_PIECE, kt * 16, cq, o);
                    if (p.out)
                        add(3, a[0], a[1], GO, W, at, [&](float(&c0)[4], float(&c1)[4]) {
                            mma_f16_2(c0, c1, go[0], b[0]);
                            if constexpr (!EXACT) mma_f16_2(c0, c1, go[1], b[0]);
                            mma_f16_2(c0, c1, go[0], b[1]);
                        });
                    add(4, n[0], n[1], Z, W, at, [&](float(&c0)[4], float(&c1)[4]) {
                        mma_f16_2(c0, c1, zt[0], b[0]);
                        mma_f16_2(c0, c1, zt[1], b[0]);
                        mma_f16_2(c0, c1, zt[0], b[1]);
                    });
                }
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int first = cq * (DK / 4) + j * 16, block = first / 64 * DR_PIECE, jj = first % 64 / 16;
                    uint32_t b[2][4];
                    load_b_t(b[0], s + block, kt * 16, jj, o);
                    load_b_t(b[1], s + NB * DR_PIECE + block, kt * 16, jj, o);
                    if (p.out)
                        add(0, dq[2 * j], dq[2 * j + 1], GO, S, at, [&](float(&c0)[4], float(&c1)[4]) {
                            mma_f16_2(c0, c1, go[0], b[0]);
                            if constexpr (!EXACT) mma_f16_2(c0, c1, go[1], b[0]);
                            mma_f16_2(c0, c1, go[0], b[1]);
                        });
                    add(1, er[2 * j], er[2 * j + 1], Z, S, at, [&](float(&c0)[4], float(&c1)[4]) {
                        mma_f16_2(c0, c1, zt[0], b[0]);
                        mma_f16_2(c0, c1, zt[1], b[0]);
                        mma_f16_2(c0, c1, zt[0], b[1]);
                    });
                    load_b_t(b[0], x + block, kt * 16, jj, o);
                    load_b_t(b[1], x + NB * DR_PIECE + block, kt * 16, jj, o);
                    add(2, wr[2 * j], wr[2 * j + 1], W, X, at, [&](float(&c0)[4], float(&c1)[4]) {
                        mma_f16_2(c0, c1, aw[0], b[0]);
                        mma_f16_2(c0, c1, aw[1], b[0]);
                        mma_f16_2(c0, c1, aw[0], b[1]);
                    });
                }
            }
            // <S0, X> of the step's 32 rows: the diagonal of S0 X^T, 16 rows and 16 key columns a warp
            if (warp < DK / 8) {
                const int kt = warp & 1, first = (warp >> 1) * 16;
                const uint32_t at = v * 2 + kt, block = first / 64 * DR_PIECE;
                if (at < groups) {
                    float d[2][4] = {};  // the diagonal's 8 x 8 blocks
                    uint32_t s0[4], s1[4], x0[4], x1[4];
                    const int j = first % 64 / 16;
                    const uint32_t rows = ((2 * j + (lane >> 4)) ^ (lane & 7)) * 16 + (lane & 15) * BLOCK_ROW,
                                   cols = ((2 * j + (lane >> 3 & 1)) ^ (lane & 7)) * 16 + ((lane & 7) + (lane >> 4) * 8) * BLOCK_ROW;
                    ldmatrix4(s0, s + block + kt * 2048 + rows), ldmatrix4(s1, s + NB * DR_PIECE + block + kt * 2048 + rows);
                    ldmatrix4(x0, x + block + kt * 2048 + cols), ldmatrix4(x1, x + NB * DR_PIECE + block + kt * 2048 + cols);
                    mma_f16_2(d[0], d[1], s0, x0), mma_f16_2(d[0], d[1], s1, x0), mma_f16_2(d[0], d[1], s0, x1);
                    // rows g (d[0]) and g + 8 (d[1]) against columns col, col + 1 of their block
                    const float mine = g == col ? d[0][0] + d[1][2] : g == col + 1 ? d[0][1] + d[1][3] : 0.0f;
                    sx = fmaf(mine, back[S][at] * back[X][at], sx);
                }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&sm.empty[it & 1])) : "memory");
        }
        // dbeta_i = w_i.z_i is the diagonal of n
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int m = 0; m < 4; ++m)
                if (cq * 16 + j * 8 + col + (m & 1) == (int)token + (m >> 1) * 8) sm.dbeta[(h - h0) & 1][token + (m >> 1) * 8] = n[j][m] * unit[4];
        // scale D dA and D dN: dA_ij = beta_j a_ij, dN_ij = -beta_i beta_j n_ij
        float most_a = 0.0f, most_n = 0.0f;
        {
            const float back_a = unit[3] * sh.scale, back_n = -unit[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (cq > rb) break;  // zeros
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const int i = token + (m >> 1) * 8, cc = cq * 16 + j * 8 + col + (m & 1);
                    const float d = __expf((gates.total[i] - gates.total[cc]) + (gates.rest[i] - gates.rest[cc])) * gates.beta[cc];
                    a[j][m] = cc <= i ? a[j][m] * back_a * d : 0.0f;
                    n[j][m] = cc < i ? n[j][m] * back_n * d * gates.beta[i] : 0.0f;
                    most_a = fmaxf(most_a, fabsf(a[j][m])), most_n = fmaxf(most_n, fabsf(n[j][m]));
                }
            }
        }
        most_a = warp_max(most_a), most_n = warp_max(most_n);
        if (lane == 0) sm.most[0][warp] = most_a, sm.most[1][warp] = most_n;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 x = *(const float4*)&sm.most[0][i], y = *(const float4*)&sm.most[1][i];
            most_a = fmaxf(fmaxf(fmaxf(most_a, x.x), fmaxf(x.y, x.z)), x.w), most_n = fmaxf(fmaxf(fmaxf(most_n, y.x), fmaxf(y.y, y.z)), y.w);
        }
        const Scale sa = scale_for(most_a), sn = scale_for(most_n);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t hi, lo;
                const uint32_t off = block_at(token + half * 8, cq * 16 + j * 8 + col);
                split_f16(a[j][half * 2], a[j][half * 2 + 1], sa.by, hi, lo);
                sts32(da + off, hi), sts32(da + DR_BLOCK + off, lo);
                split_f16(n[j][half * 2], n[j][half * 2 + 1], sn.by, hi, lo);
                sts32(dn + off, hi), sts32(dn + DR_BLOCK + off, lo);
            }
        // row factors of the products with the states, into the domains of the products that follow; k.(e u X) is needed by
        // itself
        const float back_k = gates.back_k, back_q = gates.back_q;
        const float by_k = power_inverse(back_k), into_q = sa.by * by_k, into_n = sn.by * by_k;
        float carry[2] = {0.0f, 0.0f};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = token + half * 8;
            const float g0 = gates.g[i], b = gates.beta[i];
            const float fq = g0 * sh.scale * unit[0] * into_q, fe = -g0 * b * unit[1] * into_n, fw = gates.e[i] * b * unit[2];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int first = cq * (DK / 4) + j * 8 + col;
                const uint32_t off = first / 64 * DR_BLOCK + block_at(i, first % 64);
                float2 kv = unpack_f16(lds32(k + off));
                if constexpr (PLANES == 2) {
                    const float2 lo = unpack_f16(lds32(k + NB * DR_BLOCK + off));
                    kv.x += lo.x, kv.y += lo.y;
                }
#pragma unroll
                for (int m = half * 2; m < half * 2 + 2; ++m) dq[j][m] *= fq, er[j][m] *= fe, wr[j][m] *= fw;
                carry[half] = fmaf(kv.x * back_k, wr[j][half * 2], fmaf(kv.y * back_k, wr[j][half * 2 + 1], carry[half]));
                wr[j][half * 2] *= into_n, wr[j][half * 2 + 1] *= into_n;
            }
        }
        __syncthreads();
        // rows of dA and dN against the keys before; then columns against the later ones: dN^T K, and in dA^T Q's domain that
#pragma unroll
        for (int part = 0; part < 3; ++part) {
            if (part == 2) {
                const float turn = sa.by * power_inverse(back_q) * sn.back * back_k;
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int m = 0; m < 4; ++m) wr[j][m] *= turn;
            }
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                if (part == 0 ? kt > rb : kt < rb) continue;
                uint32_t fa[2][4], fn[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (part == 0) load_a(fa[i], da + i * DR_BLOCK, rb * 16, kt, o), load_a(fn[i], dn + i * DR_BLOCK, rb * 16, kt, o);
                    if (part == 1) load_a_t(fn[i], dn + i * DR_BLOCK, kt * 16, rb, o);
                    if (part == 2) load_a_t(fa[i], da + i * DR_BLOCK, kt * 16, rb, o);
                }
#pragma unroll
                for (int j = 0; j < NP; ++j) {
                    const int first = cq * (DK / 4) + j * 16, block = first / 64 * DR_BLOCK, jj = first % 64 / 16;
#pragma unroll
                    for (int i = 0; i < PLANES; ++i) {
                        uint32_t b[4];
                        load_b_t(b, (part == 2 ? q : k) + i * NB * DR_BLOCK + block, kt * 16, jj, o);
#pragma unroll
                        for (int l = 0; l < 2 - i; ++l) {
                            if (part == 0) mma_f16_2(dq[2 * j], dq[2 * j + 1], fa[l], b), mma_f16_2(er[2 * j], er[2 * j + 1], fn[l], b);
                            if (part == 1) mma_f16_2(wr[2 * j], wr[2 * j + 1], fn[l], b);
                            if (part == 2) mma_f16_2(wr[2 * j], wr[2 * j + 1], fa[l], b);
                        }
                    }
                }
            }
        }
        // q.dq + k.(erase - write)
        const float out_q = sa.back * back_k, out_e = sn.back * back_k, out_w = sa.back * back_q;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = token + half * 8;
            float dot = 0.0f;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int first = cq * (DK / 4) + j * 8 + col;
                const uint32_t off = first / 64 * DR_BLOCK + block_at(i, first % 64);
                float kv[2] = {0, 0}, qv[2] = {0, 0};
#pragma unroll
                for (int l = 0; l < PLANES; ++l) {
                    const float2 kw = unpack_f16(lds32(k + l * NB * DR_BLOCK + off)), qw = unpack_f16(lds32(q + l * NB * DR_BLOCK + off));
                    kv[0] += kw.x, kv[1] += kw.y, qv[0] += qw.x, qv[1] += qw.y;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int m = half * 2 + e;
                    const float fq = dq[j][m] * out_q, fe = er[j][m] * out_e, fw = wr[j][m] * out_w;
                    dot = fmaf(qv[e] * back_q, fq, fmaf(kv[e] * back_k, fe - fw, dot));
                    dq[j][m] = fq, er[j][m] = fe + fw;
                    if constexpr (SHARED) all_q[j][m] += fq, all_k[j][m] += fe + fw;
                }
            }
#pragma unroll
            for (int i2 = 1; i2 < 4; i2 <<= 1) {
                dot += __shfl_xor_sync(0xffffffffu, dot, i2);
                carry[half] += __shfl_xor_sync(0xffffffffu, carry[half], i2);
            }
            if ((lane & 3) == 0) sm.dot[cq][i] = dot, sm.carry[cq][i] = carry[half];
        }
        sx = warp_reduce<OpSum>(sx);
        if (lane == 0) sm.sx[warp] = sx;
        if (!SHARED || h + 1 == h0 + group) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t i = token + half * 8;
                if (i >= c.rows) continue;
                const uint64_t to = ((c.row + i) * sh.key_heads + hk) * sh.key_dim;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const uint32_t cc = cq * (DK / 4) + j * 8 + col;
                    const float* const fq = SHARED ? all_q[SHARED ? j : 0] : dq[j];
                    const float* const fk = SHARED ? all_k[SHARED ? j : 0] : er[j];
                    dr_store_pair((T*)p.dq + to, cc, sh.key_dim, p.pairs_k, fq[half * 2], fq[half * 2 + 1]);
                    dr_store_pair((T*)p.dk + to, cc, sh.key_dim, p.pairs_k, fk[half * 2], fk[half * 2 + 1]);
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            float d[2], extra = 0.0f;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = lane * 2 + j;
                d[j] = (sm.dot[0][r] + sm.dot[1][r]) + (sm.dot[2][r] + sm.dot[3][r]);
                extra += (sm.carry[0][r] + sm.carry[1][r]) + (sm.carry[2][r] + sm.carry[3][r]);
            }
            if (lane < 16) extra = fmaf(sm.sx[lane], gates.g[DR_CHUNK - 1], extra);
            extra = warp_reduce<OpSum>(extra);
            float sum = d[0] + d[1];  // from the lane's rows to the end
#pragma unroll
            for (int i = 1; i < 32; i <<= 1) {
                const float down = __shfl_down_sync(0xffffffffu, sum, i);
                if (lane + i < 32) sum += down;
            }
            const float after = __shfl_down_sync(0xffffffffu, sum, 1), rest = lane < 31 ? after : 0.0f;
            const float v[2] = {sum + extra, (d[1] + rest) + extra};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t r = lane * 2 + j;
                if (r < c.rows) {
                    const uint64_t to = (c.row + r) * sh.heads + h;
                    if (p.ddecay) p.ddecay[to] = v[j];
                    p.dbeta[to] = sm.dbeta[(h - h0) & 1][r];
                }
            }
        }
        // the next head's first barrier comes before it writes anything that is read here, but for its gates, scales and dbeta
    }
    if (!ok) {  // copies under way land before the CTA's memory is another's
        cp_async_wait_all();
        if (t == 0) {
            mbar_wait(&sm.keys_full, 0, DR_DRAIN_LIMIT);
            for (uint32_t i = sm.asked - min(sm.asked, 2u); i < sm.asked; ++i) mbar_wait(&sm.full[i & 1], (i >> 1) & 1, DR_DRAIN_LIMIT);
        }
        set_error(LCPP_ERR_LOOKBACK_TIMEOUT);
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
    dr_let_next_start();
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

// Sequences by their numbers of chunks, the longest first (by powers of two): a chain takes as long as its sequence, and a
// long one that starts last is waited for.  One CTA; which order equals have changes no result.
constexpr int DR_ORDER_THREADS = 1024;
struct DrOrder {
    DrShape sh;
    uint32_t* order;
};
__global__ void __launch_bounds__(DR_ORDER_THREADS) dr_order_kernel(const __grid_constant__ DrOrder p) {
    __shared__ uint32_t next[33];
    dr_let_next_start();
    dr_wait_for_last();
    auto size = [&](uint32_t s) -> uint32_t {  // 0 the longest
        const uint64_t from = p.sh.start(s), to = p.sh.start(s + 1);
        return to > from ? __clz((uint32_t)((to - from + DR_CHUNK - 1) / DR_CHUNK)) : 32;
    };
    if (threadIdx.x < 33) next[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < p.sh.sequences; s += DR_ORDER_THREADS) atomicAdd(&next[size(s)], 1u);
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t sum = 0;
        for (int i = 0; i < 33; ++i) {
            const uint32_t n = next[i];
            next[i] = sum, sum += n;
        }
    }
    __syncthreads();
    for (uint32_t s = threadIdx.x; s < p.sh.sequences; s += DR_ORDER_THREADS) p.order[atomicAdd(&next[size(s)], 1u)] = s;
}

// ---- one token ------------------------------------------------------------------------------------
constexpr int DR_STEP_WARPS = 4;
// A warp takes 8 rows of a state (value dimensions) at a time: a lane holds 4 key columns of each.  All loads come before the
// first sum, and one pass serves S' k and S' q, since S q = S' q + u (k.q).  Bound by HBM: 256 rows of 32 heads of
// 128 x 128, 1.07 GB read and written, in 150 us, 7.1 TB/s.
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
    return DrShape{sh.rows, sh.offsets ? 0 : sh.length, sh.offsets, nullptr, (uint32_t)sh.num_sequences, sh.heads, sh.key_heads,
                   sh.key_dim, sh.value_dim, sh.scale};
}

// Into how many parts the sequences are cut, so that the chains have work for all SMs: the number with the least time, by
// the sequences' average length and the waves of CTAs with 8 warps (16 value dimensions each) that both passes take.  A
// chunk takes such a CTA 5.8 us in the second pass, 3.9 us in the first, and a chain of 2 warps alone on its SM 5.1 us
// (bf16, 128 dimensions; other types and sizes, whose times were not taken, go by the same).  A part has 8 chunks at least.
static uint64_t dr_parts(const lcpp_delta_shape& sh) {
    const uint64_t sms = device_info().sms, streams = sh.num_sequences * sh.heads;
    if (!streams || streams * ceil_div(sh.value_dim, 32) > sms) return 1;
    const uint64_t chunks = ceil_div(sh.rows / sh.num_sequences, DR_CHUNK), values = ceil_div(sh.value_dim, 128), keys = ceil_div(sh.key_dim, 128);
    uint64_t best = 1;
    double least = 5.1 * chunks;
    for (uint64_t parts = 2; parts <= 64 && parts * 8 <= chunks; ++parts) {
        const double each = (double)ceil_div(chunks, parts), first = (double)ceil_div(streams * (parts - 1) * (values + keys), sms),
                     second = (double)ceil_div(streams * parts * values, sms), time = each * (3.9 * first + 5.8 * second) + 4.0 * parts;
        if (time < 0.9 * least) best = parts, least = time;
    }
    return best;
}

struct DrLayout {
    uint64_t slots, units;
    uint32_t planes, key_cols, rows;  // rows of an image
    uint64_t parts;                   // of a sequence
    size_t keys, unit, x, back_x, z, back_z, back_out, local, map, before, order, bytes;
    // room: bytes that there are.  A buffer for more rows and sequences serves fewer, which may want more parts than it holds:
    // they get those that it does.
    DrLayout(int dtype, const lcpp_delta_shape& sh, bool backward, size_t room = SIZE_MAX) {
        slots = sh.rows / DR_CHUNK + sh.num_sequences, units = slots * sh.heads;
        planes = dtype == LCPP_F32 ? 2 : 1, key_cols = sh.key_dim <= 64 ? 64 : 128, rows = (uint32_t)align_up(sh.value_dim, 32);
        size_t at = 0;
        auto take = [&](uint64_t n) {
            const size_t here = at;
            at += align_up(n, 256);
            return here;
        };
        keys = take(slots * sh.key_heads * 2 * planes * (key_cols / 64) * DR_BLOCK), unit = take(units * DR_UNIT);
        x = back_x = z = back_z = back_out = 0;
        if (backward) {
            x = take(units * states(nullptr, 0, 0).bytes()), back_x = take(units * 32);
            z = take(units * kept(nullptr, 0, 0).bytes()), back_z = take(units * 32);
            back_out = take(units * 32);
        }
        order = take(sh.num_sequences * 4);
        const size_t whole = at;
        for (parts = dr_parts(sh);; --parts) {
            local = map = before = 0, at = whole;
            if (parts > 1) {
                const uint64_t pieces = sh.num_sequences * sh.heads * parts, state = (uint64_t)sh.value_dim * sh.key_dim;
                local = take(pieces * state * 4), map = take(pieces * sh.key_dim * sh.key_dim * 4), before = take(pieces * state * 4);
            }
            if (parts == 1 || at <= room) break;
        }
        bytes = max(at, (size_t)256);
    }
    DrImage states(void* room, size_t at, size_t back) const { return DrImage{(uint8_t*)room + at, (float*)((char*)room + back), key_cols / 64, rows}; }
    DrImage kept(void* room, size_t at, size_t back) const { return DrImage{(uint8_t*)room + at, (float*)((char*)room + back), 1, rows}; }
    // What the forward call saves: S0 and w.
    size_t saved_w() const { return align_up(units * states(nullptr, 0, 0).bytes(), 256); }
    size_t saved_back() const { return saved_w() + align_up(units * kept(nullptr, 0, 0).bytes(), 256); }
    size_t saved_bytes() const { return saved_back() + 2 * align_up(units * 32, 256); }
    DrImage saved_states(void* saved) const { return states(saved, 0, saved_back()); }
    DrImage saved_kept(void* saved) const { return kept(saved, saved_w(), saved_back() + align_up(units * 32, 256)); }
};

// Rows that are whole pieces of 16 bytes on 16 bytes.
static bool dr_wide(const void* p, uint64_t stride, uint64_t rows, uint32_t dim, size_t element) {
    return (uintptr_t)p % 16 == 0 && dim * element % 16 == 0 && (rows <= 1 || stride * element % 16 == 0);
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
// follows: the kernel starts while the call's one before ends (programmatic dependent launch); every kernel lets the next
// one in when it starts itself, and waits for the end of the one before ahead of its first access to memory.
template <auto KERNEL, typename A>
static lcpp_status dr_launch(const char* name, uint64_t grid, unsigned threads, size_t smem, bool follows, cudaStream_t s, const A& args) {
    if (grid > 0x7fffffffull) return LCPP_ERR_INVALID_ARG;
    if (!dr_sized<KERNEL>(smem)) return check_launch();
    cudaLaunchAttribute how[1];
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = how;
    if (follows) {
        how[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        how[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs = 1;
    }
    ProfScope prof(name, s);
    if (cudaLaunchKernelEx(&cfg, KERNEL, args) != cudaSuccess) return check_launch();
    count_launch();
    return LCPP_OK;
}

// How many warps a CTA of the chain has, 16 value dimensions each: fewer where that spreads `streams` over more SMs.
static int dr_warps(uint64_t streams, uint32_t dim) {
    const uint64_t sms = device_info().sms;
    int warps = 8;
    while (warps > 2 && (warps * 8u >= dim || streams * ceil_div(dim, warps * 16) * 2 <= sms)) warps /= 2;
    return warps;
}
template <typename F>
static lcpp_status dr_dispatch(const lcpp_delta_shape& sh, F&& f) {
    return sh.key_dim <= 64 ? f(std::integral_constant<int, 64>{}) : f(std::integral_constant<int, 128>{});
}
template <typename T, int DK, bool BACKWARD, int WHAT>
static lcpp_status dr_chain_pass(const DrChain& p, cudaStream_t s) {
    const uint64_t streams = (uint64_t)p.sh.sequences * p.sh.heads * (WHAT == DR_STATES ? p.parts - 1 : p.parts);
    auto chain = [&](auto warps) {
        constexpr int WARPS = decltype(warps)::value;
        const uint64_t grid = streams * (ceil_div(p.sh.value_dim, WARPS * 16) + (WHAT == DR_STATES ? ceil_div(p.sh.key_dim, WARPS * 16) : 0));
        constexpr size_t smem = sizeof(DrChainSmem<T, DK, WARPS>);
        static_assert(smem <= 227 * 1024, "shared memory of a CTA");
        if constexpr (BACKWARD) return dr_launch<dr_backward_kernel<T, DK, WARPS, WHAT>>(WHAT == DR_ALL ? "dr_backward" : "dr_states", grid, WARPS * 32, smem, p.sh.rows > 0, s, p);
        else return dr_launch<dr_forward_kernel<T, DK, WARPS, WHAT>>(WHAT == DR_ALL ? "dr_forward" : "dr_states", grid, WARPS * 32, smem, p.sh.rows > 0, s, p);
    };
    if constexpr (WHAT == DR_STATES) return chain(std::integral_constant<int, 8>{});  // there are parts enough
    else {
        const int warps = dr_warps(streams, p.sh.value_dim);
        if (warps == 8) return chain(std::integral_constant<int, 8>{});
        if (warps == 4) return chain(std::integral_constant<int, 4>{});
        return chain(std::integral_constant<int, 2>{});
    }
}
template <typename T, int DK, bool BACKWARD>
static lcpp_status dr_chain(DrChain p, const DrLayout& l, void* temp, cudaStream_t s) {
    p.parts = (uint32_t)l.parts;
    // more chains than SMs, of different lengths: the order matters
    if (p.sh.offsets && p.sh.sequences > 1 && (uint64_t)p.sh.sequences * p.sh.heads * ceil_div(p.sh.value_dim, 128) > (uint64_t)device_info().sms) {
        const DrOrder o{p.sh, (uint32_t*)((char*)temp + l.order)};
        const lcpp_status status = dr_launch<dr_order_kernel>("dr_order", 1, DR_ORDER_THREADS, 0, true, s, o);
        if (status != LCPP_OK) return status;
        p.sh.order = o.order;
    }
    if (l.parts > 1) {
        char* const t = (char*)temp;
        p.local = (float*)(t + l.local), p.map = (float*)(t + l.map);
        lcpp_status status = dr_chain_pass<T, DK, BACKWARD, DR_STATES>(p, s);
        if (status != LCPP_OK) return status;
        const DrJoin j{p.from, p.local, p.map, (float*)(t + l.before), p.sh.heads, p.sh.key_dim, p.sh.value_dim, p.parts,
                       (uint32_t)ceil_div(p.sh.value_dim, DR_JOIN_ROWS), BACKWARD};
        status = dr_launch<dr_join_kernel>("dr_join", (uint64_t)p.sh.sequences * p.sh.heads * j.slices, 128, 0, true, s, j);
        if (status != LCPP_OK) return status;
        p.from = j.before;
    }
    return dr_chain_pass<T, DK, BACKWARD, DR_ALL>(p, s);
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
    DrPrepare prepare(const DrShape& shape, const DrLayout& l, void* temp) const {
        return DrPrepare{shape, in.q, in.k, in.q_stride, in.k_stride, in.decay, in.beta, in.decay_stride, in.beta_stride,
                         dr_wide(in.q, in.q_stride, sh.rows, sh.key_dim, element()) &&
                             dr_wide(in.k, in.k_stride, sh.rows, sh.key_dim, element()),
                         (uint8_t*)temp + l.keys, (uint8_t*)temp + l.unit};
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

extern "C" size_t lcpp_delta_rule_temp_bytes(int dtype, const lcpp_delta_shape* shape, int backward) {
    return dr_check(dtype, shape) == LCPP_OK ? DrLayout(dtype, *shape, backward != 0).bytes : 0;
}

extern "C" size_t lcpp_delta_rule_saved_bytes(const lcpp_delta_shape* shape) {
    return dr_check(LCPP_F32, shape) == LCPP_OK ? DrLayout(LCPP_F32, *shape, false).saved_bytes() : 0;
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
    const DrLayout l(dtype, *shape, false, temp_bytes);
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
        const DrPrepare pr = c.prepare(sh, l, temp);
        DrChain p{};
        p.sh = sh, p.keys = pr.keys, p.units = pr.units, p.values = inputs->v, p.value_stride = inputs->v_stride;
        p.wide = dr_wide(inputs->v, inputs->v_stride, sh.rows, sh.value_dim, sizeof(T));
        p.from = inputs->init, p.to = last, p.out = out, p.out_stride = out_stride;
        if (saved) p.states = l.saved_states(saved), p.kept = l.saved_kept(saved);
        return dr_dispatch(*shape, [&](auto dk) -> lcpp_status {
            constexpr int DK = decltype(dk)::value, PLANES = sizeof(T) == 4 ? 2 : 1;
            lcpp_status status = LCPP_OK;
            if (sh.rows)
                status = dr_launch<dr_prepare_kernel<T, DK, false>>("dr_prepare", l.slots * sh.key_heads, DR_PREPARE_THREADS,
                                                                    sizeof(DrPrepareSmem<DK, PLANES>), sh.offsets != nullptr, s, pr);
            return status != LCPP_OK ? status : dr_chain<T, DK, false>(p, l, temp, s);
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
    const DrLayout l(dtype, *shape, true, temp_bytes);
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
        const DrPrepare pr = c.prepare(sh, l, temp);
        DrChain p{};
        p.sh = sh, p.keys = pr.keys, p.units = pr.units, p.values = grads->out, p.value_stride = grads->out_stride;
        p.wide = dr_wide(grads->out, grads->out_stride, sh.rows, sh.value_dim, sizeof(T));
        p.from = grads->last, p.to = grads->init;
        p.states = l.states(temp, l.x, l.back_x), p.kept = l.kept(temp, l.z, l.back_z);
        p.back_values = (float*)((char*)temp + l.back_out);
        DrGradient gr{};
        gr.sh = sh, gr.keys = pr.keys, gr.units = pr.units, gr.out = p.values, gr.out_stride = p.value_stride, gr.wide = p.wide;
        gr.s = l.saved_states((void*)saved), gr.w = l.saved_kept((void*)saved), gr.x = p.states, gr.z = p.kept, gr.back_out = p.back_values;
        gr.dq = grads->q, gr.dk = grads->k, gr.dv = grads->v, gr.ddecay = grads->decay, gr.dbeta = grads->beta;
        gr.pairs_k = sh.key_dim % 2 == 0 && ((uintptr_t)grads->q | (uintptr_t)grads->k) % (2 * sizeof(T)) == 0;
        gr.pairs_v = sh.value_dim % 2 == 0 && (uintptr_t)grads->v % (2 * sizeof(T)) == 0;
        return dr_dispatch(*shape, [&](auto dk) -> lcpp_status {
            constexpr int DK = decltype(dk)::value, PLANES = sizeof(T) == 4 ? 2 : 1;
            constexpr size_t smem = sizeof(DrGradientSmem<T, DK>);
            static_assert(smem <= 227 * 1024, "shared memory of a CTA");
            lcpp_status status = LCPP_OK;
            if (sh.rows)
                status = dr_launch<dr_prepare_kernel<T, DK, true>>("dr_prepare", l.slots * sh.key_heads, DR_PREPARE_THREADS,
                                                                   sizeof(DrPrepareSmem<DK, PLANES>), sh.offsets != nullptr, s, pr);
            if (status == LCPP_OK) status = dr_chain<T, DK, true>(p, l, temp, s);
            if (status != LCPP_OK || !sh.rows) return status;
            const uint64_t grid = l.slots * sh.key_heads;
            if (sh.heads > sh.key_heads) return dr_launch<dr_gradient_kernel<T, DK, true>>("dr_gradient", grid, DR_GRAD_THREADS, smem, true, s, gr);
            return dr_launch<dr_gradient_kernel<T, DK, false>>("dr_gradient", grid, DR_GRAD_THREADS, smem, true, s, gr);
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
