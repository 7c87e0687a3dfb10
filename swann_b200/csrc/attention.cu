// attention.cu -- attention of one new token a sequence over a paged key-value
// cache.
//
// For a query row of the token at slot i = length - 1, over the slots j it sees
// (j <= i and, with a window w, j > i - w or j < sinks; slots whose page the
// table does not name are not seen):
//   x_j = scale <q, k_j>,  lse = log sum_j e^x_j,  out = sum_j e^(x_j - lse) v_j
// in one pass over K and V, with the running maximum m and sum l of a softmax
// in base 2:  m' = max(m, x), l' = l 2^(m - m') + 2^(x - m'), and the
// accumulated rows scaled by the same 2^(m - m').  Where nothing is seen the
// row is 0 and lse is -inf.
//
// One warp owns up to 16 query rows that share a key head and walks blocks of
// 16 keys on its own: keys and values arrive by cp.async in a ring of shared
// memory stages (128-byte swizzle, rows that are not seen filled with zeros, so
// nothing that lies in them reaches a product), logits and the weighted sum run
// on mma.sync with fp32 accumulators.  Weights are rounded to the cache's 16
// bits for the second product, as its other operand is; their sum l is taken
// before that rounding.  The warps of a CTA interleave the blocks of one stretch
// of the sequence and join through shared memory at the end; the stretches of a
// long sequence are joined by a second kernel.

#include "attn.cuh"

namespace swb {
namespace attn {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int ROWS = 16;      // query rows of a tile
constexpr int KEYS = 16;      // keys a warp scores at a time
constexpr int STAGES = 3;

struct Walk {
    Cache c;
    const void* q;
    int64_t q_seq_stride, q_head_stride;
    int q_heads, group;       // query heads; of them per key head
    int head_tiles, tile_heads;
    int splits;
    float scale2;             // scale * log2(e)
    int window, sinks;
    const void* prior_out;    // [seqs, q_heads, D] and [seqs, q_heads]; null: none
    const float* prior_lse;
    void* out;
    float* lse;
    float* part_out;          // [rows][splits][D]
    float2* part_ml;          // [rows][splits]
    float* logits;            // [seqs * q_heads][capacity], for the weights; null: not wanted
};

// the slots that the token at slot `pos` can see, as one range of virtual
// places: the first tokens, then everything from `lo` on
struct Range {
    int first, lo, n;
    __device__ __forceinline__ int slot(int u) const { return u < first ? u : lo + (u - first); }
};
__device__ __forceinline__ Range visible(int pos, int window, int sinks, int64_t capacity) {
    Range r;
    const int end = (int)min((int64_t)pos + 1, capacity);     // nothing is held beyond the table
    r.lo = window > 0 ? min(max(0, pos - window + 1), max(0, end)) : 0;
    r.first = min(sinks, r.lo);
    r.n = max(0, r.first + end - r.lo);
    return r;
}

template <int D>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {
    return (uint32_t)(row * D * 2 + ((chunk ^ (row & 7)) << 4));
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS) walk_kernel(const __grid_constant__ Walk P) {
    constexpr int CH = D / 8;                          // 16-byte chunks of a row
    constexpr int STAGE = 2 * KEYS * D * 2;            // K and V of a block of keys
    constexpr int NT = D / 8;                          // 8-wide output tiles
    extern __shared__ __align__(128) char smem[];
    __shared__ unsigned s_seen[WARPS][STAGES];
    __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // -- which sequence, heads and stretch
    int64_t item = blockIdx.x;
    const int split = (int)(item % P.splits);
    item /= P.splits;
    const int ht = (int)(item % P.head_tiles);
    item /= P.head_tiles;
    const int g = (int)(item % P.c.kv_heads), b = (int)(item / P.c.kv_heads);
    const int heads = min(P.tile_heads, P.group - ht * P.tile_heads);
    const int64_t row0 = (int64_t)b * P.q_heads + g * P.group + ht * P.tile_heads;   // first output row
    const Range rg = visible(P.c.lengths[b] - 1, P.window, P.sinks, P.c.capacity());

    // this CTA's stretch: a whole number of blocks for every warp
    const int per = ((rg.n + P.splits - 1) / P.splits + WARPS * KEYS - 1) / (WARPS * KEYS) * (WARPS * KEYS);
    const int u0 = min(rg.n, split * per), u1 = min(rg.n, u0 + per);
    const int nblk = (u1 - u0 + KEYS - 1) / KEYS;                // blocks of the stretch; warp w has w, w + WARPS, ..
    const int mine = nblk > warp ? (nblk - warp - 1) / WARPS + 1 : 0;

    // -- the query rows as matrix fragments: row r is head r of the tile
    const T* q = static_cast<const T*>(P.q) + b * P.q_seq_stride + (int64_t)(g * P.group + ht * P.tile_heads) * P.q_head_stride;
    const int r0 = lane >> 2, r1 = r0 + 8;
    const bool ok0 = r0 < heads, ok1 = r1 < heads;
    const T* q0 = q + r0 * P.q_head_stride;
    const T* q1 = q + r1 * P.q_head_stride;
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        const int c = kk * 16 + (lane & 3) * 2;
        qf[kk][0] = ok0 ? *reinterpret_cast<const uint32_t*>(q0 + c) : 0u;
        qf[kk][1] = ok1 ? *reinterpret_cast<const uint32_t*>(q1 + c) : 0u;
        qf[kk][2] = ok0 ? *reinterpret_cast<const uint32_t*>(q0 + c + 8) : 0u;
        qf[kk][3] = ok1 ? *reinterpret_cast<const uint32_t*>(q1 + c + 8) : 0u;
    }
    float* lg0 = P.logits && ok0 ? P.logits + (row0 + r0) * P.c.capacity() : nullptr;
    float* lg1 = P.logits && ok1 ? P.logits + (row0 + r1) * P.c.capacity() : nullptr;

    const T* kp = static_cast<const T*>(P.c.k) + (int64_t)g * P.c.head_stride;
    const T* vp = static_cast<const T*>(P.c.v) + (int64_t)g * P.c.head_stride;
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * STAGE);

    // lane < 16: the row of key `lane` of this warp's block i, or -1
    auto find = [&](int i) -> int64_t {
        const int u = u0 + (i * WARPS + warp) * KEYS + lane;
        return (lane < KEYS && i < mine && u < u1) ? P.c.row(b, rg.slot(u)) : -1;
    };
    auto issue = [&](int i, int64_t off) {
        const uint32_t st = ring + (i % STAGES) * STAGE;
        if (i < mine) {
            const unsigned seen = __ballot_sync(FULL, off >= 0);
            if (lane == 0) s_seen[warp][i % STAGES] = seen;
#pragma unroll
            for (int it = 0; it < KEYS * CH / 32; ++it) {
                const int r = (it * 32 + lane) / CH, c = (it * 32 + lane) % CH;
                const int64_t o = __shfl_sync(FULL, (long long)off, r);
                const bool real = o >= 0;
                const int64_t e = real ? o + c * 8 : 0;
                cp_async16_or_zero(st + swz<D>(r, c), kp + e, real);
                cp_async16_or_zero(st + KEYS * D * 2 + swz<D>(r, c), vp + e, real);
            }
        }
        cp_async_commit();
    };

    float o[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m0 = NEG_INF, m1 = NEG_INF, l0 = 0.f, l1 = 0.f;

#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i, find(i));
    int64_t next = find(STAGES - 1);
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<STAGES - 2>();
        __syncwarp();
        issue(i + STAGES - 1, next);      // the stage that block i - 1 has left
        next = find(i + STAGES);
        const uint32_t st = ring + (i % STAGES) * STAGE;
        const unsigned seen = s_seen[warp][i % STAGES];

        float x[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t f[4];
            ldmatrix4(f, st + swz<D>((lane >> 4) * 8 + (lane & 7), 2 * kk + ((lane >> 3) & 1)));
            Elem<T>::mma(x[0], qf[kk], f[0], f[1]);
            Elem<T>::mma(x[1], qf[kk], f[2], f[3]);
        }
        const int ub = u0 + (i * WARPS + warp) * KEYS;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int kx = n * 8 + (lane & 3) * 2 + (e & 1);
                x[n][e] = (seen >> kx) & 1u ? x[n][e] * P.scale2 : NEG_INF;
                float* lg = e < 2 ? lg0 : lg1;
                if (lg && ub + kx < u1) lg[rg.slot(ub + kx)] = x[n][e];
            }
        float a0 = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[1][0], x[1][1]));
        float a1 = fmaxf(fmaxf(x[0][2], x[0][3]), fmaxf(x[1][2], x[1][3]));
#pragma unroll
        for (int s = 1; s <= 2; s <<= 1) {
            a0 = fmaxf(a0, __shfl_xor_sync(FULL, a0, s));
            a1 = fmaxf(a1, __shfl_xor_sync(FULL, a1, s));
        }
        if (__any_sync(FULL, a0 > m0 || a1 > m1)) {
            const float n0 = fmaxf(m0, a0), n1 = fmaxf(m1, a1);
            const float f0 = n0 == NEG_INF ? 1.f : exp2_fast(m0 - n0), f1 = n1 == NEG_INF ? 1.f : exp2_fast(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                o[j][0] *= f0;
                o[j][1] *= f0;
                o[j][2] *= f1;
                o[j][3] *= f1;
            }
        }
        const float s0 = m0 == NEG_INF ? 0.f : m0, s1 = m1 == NEG_INF ? 0.f : m1;
        uint32_t pf[4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float w0 = exp2_fast(x[n][0] - s0), w1 = exp2_fast(x[n][1] - s0);
            const float w2 = exp2_fast(x[n][2] - s1), w3 = exp2_fast(x[n][3] - s1);
            l0 += w0 + w1;
            l1 += w2 + w3;
            pf[2 * n] = Elem<T>::pack(w0, w1);
            pf[2 * n + 1] = Elem<T>::pack(w2, w3);
        }
        const uint32_t sv = st + KEYS * D * 2;
#pragma unroll
        for (int j = 0; j < NT / 2; ++j) {
            uint32_t f[4];
            ldmatrix4_t(f, sv + swz<D>(((lane >> 3) & 1) * 8 + (lane & 7), 2 * j + (lane >> 4)));
            Elem<T>::mma(o[2 * j], pf, f[0], f[1]);
            Elem<T>::mma(o[2 * j + 1], pf, f[2], f[3]);
        }
        __syncwarp();
    }
    cp_async_wait<0>();
#pragma unroll
    for (int s = 1; s <= 2; s <<= 1) {
        l0 += __shfl_xor_sync(FULL, l0, s);
        l1 += __shfl_xor_sync(FULL, l1, s);
    }

    // -- join the warps
    if ((lane & 3) == 0) {
        s_m[warp][r0] = m0;
        s_m[warp][r1] = m1;
        s_l[warp][r0] = l0;
        s_l[warp][r1] = l1;
    }
    __syncthreads();      // the ring is free too
    float M0 = NEG_INF, M1 = NEG_INF;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        M0 = fmaxf(M0, s_m[w][r0]);
        M1 = fmaxf(M1, s_m[w][r1]);
    }
    const float f0 = l0 == 0.f ? 0.f : exp2_fast(m0 - M0), f1 = l1 == 0.f ? 0.f : exp2_fast(m1 - M1);
    float* so = reinterpret_cast<float*>(smem);       // [WARPS][ROWS][D]
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int c = j * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(so + (warp * ROWS + r0) * D + c) = make_float2(o[j][0] * f0, o[j][1] * f0);
        *reinterpret_cast<float2*>(so + (warp * ROWS + r1) * D + c) = make_float2(o[j][2] * f1, o[j][3] * f1);
    }
    __syncthreads();
    constexpr int TPR = THREADS / ROWS;                // threads of a row
    constexpr int DPT = D / TPR;                       // dimensions of a thread
    const int r = threadIdx.x / TPR, d0 = (threadIdx.x % TPR) * 2;
    if (r >= heads) return;
    float M = NEG_INF, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
        if (s_l[w][r] != 0.f) l += s_l[w][r] * exp2_fast(s_m[w][r] - M);
    const int64_t row = row0 + r;
    float2 acc[DPT / 2];
#pragma unroll
    for (int i = 0; i < DPT / 2; ++i) {
        acc[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float2 y = *reinterpret_cast<const float2*>(so + (w * ROWS + r) * D + d0 + i * 2 * TPR);
            acc[i].x += y.x;
            acc[i].y += y.y;
        }
    }
    if (P.splits > 1 || P.logits) {
        float* po = P.part_out + (row * P.splits + split) * D;
#pragma unroll
        for (int i = 0; i < DPT / 2; ++i) *reinterpret_cast<float2*>(po + d0 + i * 2 * TPR) = acc[i];
        if (threadIdx.x % TPR == 0) P.part_ml[row * P.splits + split] = make_float2(M, l);
        return;
    }
    // one stretch: this is the answer, up to the prior part
    float pm = P.prior_lse ? P.prior_lse[row] * LOG2E : NEG_INF;
    const float top = fmaxf(M, pm);
    const float fa = l == 0.f ? 0.f : exp2_fast(M - top), fb = pm == NEG_INF ? 0.f : exp2_fast(pm - top);
    const float sum = l * fa + fb;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(P.out) + row * D);
    const uint32_t* po = fb > 0.f ? reinterpret_cast<const uint32_t*>(static_cast<const T*>(P.prior_out) + row * D) : nullptr;
#pragma unroll
    for (int i = 0; i < DPT / 2; ++i) {
        float2 y = make_float2(acc[i].x * fa, acc[i].y * fa);
        if (po) {
            const float2 z = Elem<T>::wide(po[(d0 + i * 2 * TPR) / 2]);
            y.x += fb * z.x;
            y.y += fb * z.y;
        }
        out[(d0 + i * 2 * TPR) / 2] = Elem<T>::pack(y.x * inv, y.y * inv);
    }
    if (threadIdx.x % TPR == 0) P.lse[row] = sum == 0.f ? NEG_INF : (top + log2f(sum)) * LN2;
}

// -- the join of a row's stretches, and the weights of the slots ----------------

struct Join {
    Cache c;
    int q_heads, group, splits;
    int64_t rows;             // seqs * q_heads
    int window, sinks;
    const float* part_out;
    const float2* part_ml;
    const void* prior_out;
    const float* prior_lse;
    void* out;
    float* lse;
    const float* logits;
    float* weights;           // [seqs][kv_heads][width]; null: not wanted
    int64_t width;
    int accumulate;
    int chunks;               // blocks of JOIN_SLOTS slots of a row of weights
};

constexpr int JOIN_THREADS = 128;
constexpr int JOIN_SLOTS = 1024;

// maximum and sum of a row's stretches and its prior part, by one warp
__device__ __forceinline__ float2 row_total(const Join& P, int64_t row, int lane) {
    float m = NEG_INF;
    for (int s = lane; s < P.splits; s += 32) m = fmaxf(m, P.part_ml[row * P.splits + s].x);
    if (P.prior_lse && lane == 0) m = fmaxf(m, P.prior_lse[row] * LOG2E);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, x));
    float l = 0.f;
    for (int s = lane; s < P.splits; s += 32) {
        const float2 y = P.part_ml[row * P.splits + s];
        if (y.y != 0.f) l += y.y * exp2_fast(y.x - m);
    }
    if (P.prior_lse && lane == 0) {
        const float p = P.prior_lse[row] * LOG2E;
        if (p != NEG_INF) l += exp2_fast(p - m);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(FULL, l, x);
    return make_float2(m, l);
}

template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Join P) {
    dependency_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int W = JOIN_THREADS / 32, E = D / 32;
    if ((int64_t)blockIdx.x < P.rows) {
        __shared__ float s_o[W][D];
        const int64_t row = blockIdx.x;
        const float2 ml = row_total(P, row, lane);
        float acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
        for (int s = warp; s < P.splits; s += W) {
            const float2 mine = P.part_ml[row * P.splits + s];
            if (mine.y == 0.f) continue;      // nothing seen there: its rows are not read
            const float f = exp2_fast(mine.x - ml.x);
            const float* po = P.part_out + (row * P.splits + s) * D;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * po[lane + 32 * e];
        }
        if (warp == 0 && P.prior_lse) {
            const float p = P.prior_lse[row] * LOG2E;
            if (p != NEG_INF) {
                const float f = exp2_fast(p - ml.x);
                const T* po = static_cast<const T*>(P.prior_out) + row * D;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += f * (float)po[lane + 32 * e];
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = acc[e];
        __syncthreads();
        const float inv = ml.y == 0.f ? 0.f : 1.f / ml.y;
        for (int d = threadIdx.x; d < D; d += JOIN_THREADS) {
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) y += s_o[w][d];
            static_cast<T*>(P.out)[row * D + d] = T(y * inv);
        }
        if (threadIdx.x == 0) P.lse[row] = ml.y == 0.f ? NEG_INF : (ml.x + log2f(ml.y)) * LN2;
        return;
    }
    // the weights of JOIN_SLOTS slots of one key head, summed over its query heads
    int64_t item = blockIdx.x - P.rows;
    const int chunk = (int)(item % P.chunks);
    item /= P.chunks;
    const int g = (int)(item % P.c.kv_heads), b = (int)(item / P.c.kv_heads);
    const int far = P.window > 0 ? max(0, P.c.lengths[b] - P.window) : 0;
    const int L = P.c.length(b);
    float acc[JOIN_SLOTS / JOIN_THREADS];
#pragma unroll
    for (int i = 0; i < JOIN_SLOTS / JOIN_THREADS; ++i) acc[i] = 0.f;
    const int64_t s0 = (int64_t)chunk * JOIN_SLOTS + threadIdx.x;
    for (int h = 0; h < P.group; ++h) {
        const int64_t row = (int64_t)b * P.q_heads + g * P.group + h;
        const float2 ml = row_total(P, row, lane);
        const float lse2 = ml.y == 0.f ? __int_as_float(0x7f800000) : ml.x + log2f(ml.y);
#pragma unroll
        for (int i = 0; i < JOIN_SLOTS / JOIN_THREADS; ++i) {
            const int64_t j = s0 + i * JOIN_THREADS;
            if (j < L && (j >= far || j < P.sinks)) acc[i] += exp2_fast(P.logits[row * P.c.capacity() + j] - lse2);
        }
    }
    float* w = P.weights + ((int64_t)b * P.c.kv_heads + g) * P.width;
#pragma unroll
    for (int i = 0; i < JOIN_SLOTS / JOIN_THREADS; ++i) {
        const int64_t j = s0 + i * JOIN_THREADS;
        if (j < P.width) w[j] = P.accumulate ? w[j] + acc[i] : acc[i];
    }
}

// -- host side --------------------------------------------------------------

// How many stretches a sequence is cut into: enough CTAs for two rounds of the
// two that an SM holds, no stretch planned below 256 slots of a full sequence.
inline int plan_splits(const Cache& c, int64_t tiles) {
    if (tiles <= 0) return 1;
    const int64_t want = (4ll * abi::num_sms() + tiles - 1) / tiles;
    const int64_t most = (c.capacity() + 255) / 256;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 512 ? 512 : s);
}

template <typename T, int D>
int launch_walk(const Walk& w, int64_t items, cudaStream_t st) {
    constexpr int smem = WARPS * STAGES * 2 * KEYS * D * 2;
    cudaError_t e = cudaFuncSetAttribute(walk_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return abi::cuda_fail(e, "cudaFuncSetAttribute(attention)");
    walk_kernel<T, D><<<(unsigned)items, THREADS, smem, st>>>(w);
    return abi::cuda_check("attention launch");
}

template <typename T, int D>
int launch_join(const Join& j, int64_t blocks, cudaStream_t st) {
    const cudaError_t e = launch_after(join_kernel<T, D>, dim3((unsigned)blocks), dim3(JOIN_THREADS), 0, st, j);
    if (e != cudaSuccess) return abi::cuda_fail(e, "attention join launch");
    return abi::cuda_check("attention join launch");
}

inline int run_walk(const Walk& w, int64_t items, int dtype, int d, cudaStream_t st) {
    if (dtype == SWB_F16)
        return d == 64 ? launch_walk<__half, 64>(w, items, st) : launch_walk<__half, 128>(w, items, st);
    return d == 64 ? launch_walk<__nv_bfloat16, 64>(w, items, st) : launch_walk<__nv_bfloat16, 128>(w, items, st);
}

inline int run_join(const Join& j, int64_t blocks, int dtype, int d, cudaStream_t st) {
    if (dtype == SWB_F16)
        return d == 64 ? launch_join<__half, 64>(j, blocks, st) : launch_join<__half, 128>(j, blocks, st);
    return d == 64 ? launch_join<__nv_bfloat16, 64>(j, blocks, st) : launch_join<__nv_bfloat16, 128>(j, blocks, st);
}

inline Walk make_walk(const Cache& c, const void* q, int64_t ts, int64_t hs, int q_heads, float scale, int window,
                      int sinks) {
    Walk w = {};
    w.c = c;
    w.q = q;
    w.q_seq_stride = ts;
    w.q_head_stride = hs;
    w.q_heads = q_heads;
    w.group = q_heads / c.kv_heads;
    w.tile_heads = w.group < ROWS ? w.group : ROWS;
    w.head_tiles = (w.group + w.tile_heads - 1) / w.tile_heads;
    w.splits = 1;
    w.scale2 = scale * LOG2E;
    w.window = window;
    w.sinks = sinks;
    return w;
}

struct DecodeSpace {
    int splits;
    uint64_t ml, out, logits, total;   // byte offsets
};
inline DecodeSpace decode_space(const Cache& c, int d, int q_heads, bool weights) {
    DecodeSpace s;
    const int group = q_heads / c.kv_heads, tiles = (group + ROWS - 1) / ROWS;
    s.splits = plan_splits(c, (int64_t)c.seqs * c.kv_heads * tiles);
    const uint64_t rows = (uint64_t)c.seqs * q_heads;
    const bool join = s.splits > 1 || weights;
    s.out = 0;
    s.ml = join ? rows * s.splits * d * 4 : 0;
    s.logits = s.ml + (join ? rows * s.splits * 8 : 0);
    s.total = s.logits + (weights ? rows * (uint64_t)c.capacity() * 4 : 0);
    return s;
}

}  // namespace attn
}  // namespace swb

using namespace swb;
using namespace swb::attn;

extern "C" uint64_t swb_attn_decode_workspace(const swb_kv_cache* cache, int q_heads, int with_weights) {
    Cache c;
    if (check_cache(cache, &c) || q_heads < 1 || q_heads % c.kv_heads) return ~(uint64_t)0;
    return decode_space(c, cache->head_dim, q_heads, with_weights != 0).total;
}

extern "C" int swb_attn_decode(const void* q, int64_t q_seq_stride, int64_t q_head_stride, int q_heads,
                               const swb_kv_cache* cache, float scale, int window, int sinks, const void* prior_out,
                               const float* prior_lse, void* out, float* lse, float* weights, int64_t weights_width,
                               int accumulate, void* workspace, uint64_t ws_bytes, void* stream) {
    Cache c;
    int rc = check_cache(cache, &c);
    if (rc) return rc;
    if (c.seqs == 0) return SWB_OK;
    rc = check_query(q, q_seq_stride, q_head_stride, q_heads, c);
    if (rc) return rc;
    if (!out || !lse) return abi::fail(SWB_ERR_ARG, "null output");
    if (window < 0 || sinks < 0) return abi::fail(SWB_ERR_ARG, "window and sinks must not be negative");
    if (!prior_out != !prior_lse) return abi::fail(SWB_ERR_ARG, "a prior part needs its rows and its lse");
    if (weights && weights_width < c.capacity())
        return abi::fail(SWB_ERR_ARG, "weights are narrower than the page table's slots");
    const int d = cache->head_dim;
    const DecodeSpace sp = decode_space(c, d, q_heads, weights != nullptr);
    if (sp.total && (!workspace || ws_bytes < sp.total)) return abi::fail(SWB_ERR_ARG, "workspace too small");
    cudaStream_t st = (cudaStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    Walk w = make_walk(c, q, q_seq_stride, q_head_stride, q_heads, scale, window, sinks);
    const int64_t items = (int64_t)c.seqs * c.kv_heads * w.head_tiles * sp.splits;
    if (items >= ((int64_t)1 << 31)) return abi::fail(SWB_ERR_ARG, "too many sequences in one call");
    w.splits = sp.splits;
    w.prior_out = prior_out;
    w.prior_lse = prior_lse;
    w.out = out;
    w.lse = lse;
    w.part_out = reinterpret_cast<float*>(ws + sp.out);
    w.part_ml = reinterpret_cast<float2*>(ws + sp.ml);
    w.logits = weights ? reinterpret_cast<float*>(ws + sp.logits) : nullptr;
    rc = run_walk(w, items, cache->dtype, d, st);
    if (rc || (sp.splits == 1 && !weights)) return rc;
    Join j = {};
    j.c = c;
    j.q_heads = q_heads;
    j.group = w.group;
    j.splits = sp.splits;
    j.rows = (int64_t)c.seqs * q_heads;
    j.window = window;
    j.sinks = sinks;
    j.part_out = w.part_out;
    j.part_ml = w.part_ml;
    j.prior_out = prior_out;
    j.prior_lse = prior_lse;
    j.out = out;
    j.lse = lse;
    j.logits = w.logits;
    j.weights = weights;
    j.width = weights_width;
    j.accumulate = accumulate;
    j.chunks = (int)((weights_width + JOIN_SLOTS - 1) / JOIN_SLOTS);
    const int64_t blocks = j.rows + (weights ? (int64_t)c.seqs * c.kv_heads * j.chunks : 0);
    if (blocks >= ((int64_t)1 << 31)) return abi::fail(SWB_ERR_ARG, "too many sequences in one call");
    return run_join(j, blocks, cache->dtype, d, st);
}
