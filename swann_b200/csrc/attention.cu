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
// row is 0 and lse is -inf.  The bytes of K and V bound it.
//
// One warp owns up to 16 query rows that share a key head (a pair: a sequence
// and those rows) and walks blocks of 16 keys on its own: keys and values arrive
// by cp.async in a ring of shared memory stages (128-byte swizzle, rows that are
// not seen filled with zeros, so nothing that lies in them reaches a product),
// logits and the weighted sum run on mma.sync with fp32 accumulators (16 rows at
// most: a tcgen05 tile of 128 would be seven eighths empty, and the tensor pipe
// is not what bounds this).  Weights are rounded to the cache's 16 bits for the
// second product, as its other operand is; their sum l is taken before that.
//
// Who walks what.  Few pairs: the pairs' units of 64 keys are laid end to end
// and every CTA of a grid that the SMs hold at once takes an equal run of them,
// whatever the sequences' lengths are; a pair cut by the end of a run leaves
// parts (m, l, unnormalised rows), at most two a CTA, which a second kernel
// joins.  Very many pairs: a one-warp CTA each.

#include "attn.cuh"

namespace swb {
namespace attn {

constexpr int WARPS = 4;      // of a CTA that takes a run of units
constexpr int ROWS = 16;      // query rows of a tile
constexpr int KEYS = 16;      // keys a warp scores at a time
constexpr int UNIT = WARPS * KEYS;
constexpr int STAGES = 3;

struct Walk {
    Cache c;
    const void* q;
    int64_t q_seq_stride, q_head_stride;
    int q_heads, group;       // query heads; of them per key head
    int head_tiles, tile_heads;
    float scale2;             // scale * log2(e)
    int window, sinks;
    const void* prior_out;    // [seqs, q_heads, D] and [seqs, q_heads]; null: none
    const float* prior_lse;
    void* out;
    float* lse;
    int runs;                 // CTAs that share the units; 0: a CTA a pair
    float* part_out;          // [2 * runs][ROWS][D]
    float2* part_ml;          // [2 * runs][ROWS]
    float* logits;            // [seqs * q_heads][capacity], for the weights; null: not wanted
    float* lse2;              // [seqs * q_heads] in base 2, with logits
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

__device__ __forceinline__ int units_of(const Walk& P, int b) {
    const Range r = visible(P.c.lengths[b] - 1, P.window, P.sinks, P.c.capacity());
    return max(1, (r.n + UNIT - 1) / UNIT);
}

// The sequences' units laid end to end, counted by all threads of a CTA: thread t
// sums a stretch of sequences.
template <int THREADS>
struct Layout {
    int64_t before;           // units of a pair row (one key head) ahead of this thread's stretch
    int64_t mine;
    int64_t total;            // of all sequences, one key head tile
    int per;                  // sequences of a stretch
    __device__ __forceinline__ void count(const Walk& P, int64_t* s_sum) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        per = (P.c.seqs + THREADS - 1) / THREADS;
        const int b0 = min(P.c.seqs, (int)threadIdx.x * per), b1 = min(P.c.seqs, b0 + per);
        mine = 0;
        for (int b = b0; b < b1; ++b) mine += units_of(P, b);
        int64_t sum = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int64_t y = __shfl_up_sync(FULL, (long long)sum, s);
            if (lane >= s) sum += y;
        }
        if (lane == 31) s_sum[warp] = sum;
        __syncthreads();
        before = sum - mine;
        total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) {
            before += w < warp ? s_sum[w] : 0;
            total += s_sum[w];
        }
        __syncthreads();
    }
};

// a place among the units: a pair, its key head tile and the unit inside it
struct Spot {
    int b, h;                 // sequence; key head * head_tiles + tile
    int unit, units;          // of the pair
};

// CTA-wide: where unit x of the whole lies.  Sequence-major: all head tiles of a
// sequence, then the next.
template <int THREADS>
__device__ __forceinline__ Spot spot_of(const Walk& P, const Layout<THREADS>& L, int64_t x, Spot* s_spot) {
    const int tiles = P.c.kv_heads * P.head_tiles;
    int64_t left = x - L.before * tiles;
    if (left >= 0 && left < L.mine * tiles) {
        int b = threadIdx.x * L.per;
        for (;; ++b) {
            const int n = units_of(P, b);
            if (left < (int64_t)n * tiles) {
                s_spot->b = b;
                s_spot->h = (int)(left / n);
                s_spot->unit = (int)(left % n);
                s_spot->units = n;
                break;
            }
            left -= (int64_t)n * tiles;
        }
    }
    __syncthreads();
    return *s_spot;
}

// CTAs that take a run, and where a run begins
__device__ __forceinline__ int64_t runs_used(const Walk& P, int64_t all) { return min((int64_t)P.runs, all); }

// CTAs of a run that an SM holds, by their shared memory and registers
constexpr int cta_per_sm(int d) { return d == 128 ? 2 : 4; }

template <typename T, int D, int W>
__global__ void __launch_bounds__(W * 32, W > 1 ? cta_per_sm(D) : 8) walk_kernel(const __grid_constant__ Walk P) {
    constexpr int THREADS = W * 32;
    constexpr bool RUNS = W > 1;                       // an equal run of units a CTA, or a pair a warp
    constexpr int CH = D / 8;                          // 16-byte chunks of a row
    constexpr int STAGE = 2 * KEYS * D * 2;            // K and V of a block of keys
    constexpr int NT = D / 8;                          // 8-wide output tiles
    extern __shared__ __align__(128) char smem[];
    __shared__ unsigned s_seen[W][STAGES];
    __shared__ float s_m[W][ROWS], s_l[W][ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const uint32_t ring = smem_u32(smem) + warp * (STAGES * STAGE);

    // -- which pairs, and which of their keys
    Spot at;
    int64_t left = 1;                                  // units still to walk
    if constexpr (RUNS) {
        __shared__ int64_t s_sum[W];
        __shared__ Spot s_spot;
        Layout<THREADS> lay;
        lay.count(P, s_sum);
        const int64_t all = lay.total * P.c.kv_heads * P.head_tiles, used = runs_used(P, all);
        if (blockIdx.x >= used) return;
        const int64_t x0 = all * blockIdx.x / used;
        left = all * (blockIdx.x + 1) / used - x0;
        at = spot_of(P, lay, x0, &s_spot);
    } else {
        const int tiles = P.c.kv_heads * P.head_tiles;
        at.b = (int)(blockIdx.x / tiles);
        at.h = (int)(blockIdx.x % tiles);
        at.unit = 0;
        at.units = 1;
    }

    for (bool first = true; left > 0; first = false) {
    const int b = at.b, g = at.h / P.head_tiles, ht = at.h % P.head_tiles;
    const int heads = min(P.tile_heads, P.group - ht * P.tile_heads);
    const int64_t row0 = (int64_t)b * P.q_heads + g * P.group + ht * P.tile_heads;   // first output row
    const Range rg = visible(P.c.lengths[b] - 1, P.window, P.sinks, P.c.capacity());
    const int take = (int)min(left, (int64_t)(at.units - at.unit));
    const int u0 = RUNS ? min(rg.n, at.unit * UNIT) : 0, u1 = RUNS ? min(rg.n, u0 + take * UNIT) : rg.n;
    const bool entire = take == at.units;              // nothing of the pair is left to others
    const int nblk = (u1 - u0 + KEYS - 1) / KEYS;      // blocks of the stretch; warp w has w, w + W, ..
    const int mine = nblk > warp ? (nblk - warp - 1) / W + 1 : 0;

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
    // lane < 16: the row of key `lane` of this warp's block i, or -1
    auto find = [&](int i) -> int64_t {
        const int u = u0 + (i * W + warp) * KEYS + lane;
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
        const int ub = u0 + (i * W + warp) * KEYS;
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
    for (int w = 0; w < W; ++w) {
        M0 = fmaxf(M0, s_m[w][r0]);
        M1 = fmaxf(M1, s_m[w][r1]);
    }
    const float f0 = l0 == 0.f ? 0.f : exp2_fast(m0 - M0), f1 = l1 == 0.f ? 0.f : exp2_fast(m1 - M1);
    float* so = reinterpret_cast<float*>(smem);       // [W][ROWS][D]
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
    if (r < heads) {
    float M = NEG_INF, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) M = fmaxf(M, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < W; ++w)
        if (s_l[w][r] != 0.f) l += s_l[w][r] * exp2_fast(s_m[w][r] - M);
    const int64_t row = row0 + r;
    float2 acc[DPT / 2];
#pragma unroll
    for (int i = 0; i < DPT / 2; ++i) {
        acc[i] = make_float2(0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float2 y = *reinterpret_cast<const float2*>(so + (w * ROWS + r) * D + d0 + i * 2 * TPR);
            acc[i].x += y.x;
            acc[i].y += y.y;
        }
    }
    if (!entire) {
        const int64_t part = 2 * (int64_t)blockIdx.x + (first ? 0 : 1);
        float* po = P.part_out + (part * ROWS + r) * D;
#pragma unroll
        for (int i = 0; i < DPT / 2; ++i) *reinterpret_cast<float2*>(po + d0 + i * 2 * TPR) = acc[i];
        if (threadIdx.x % TPR == 0) P.part_ml[part * ROWS + r] = make_float2(M, l);
    } else {
    // the whole pair: this is the answer, up to the prior part
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
    if (threadIdx.x % TPR == 0) {
        const float x = sum == 0.f ? NEG_INF : top + log2f(sum);
        P.lse[row] = x * LN2;
        if (P.lse2) P.lse2[row] = x;
    }
    }
    }
    left -= take;
    at.unit = 0;
    if (left > 0) {
        if (++at.h == P.c.kv_heads * P.head_tiles) {
            at.h = 0;
            ++at.b;
            at.units = units_of(P, at.b);
        }
        __syncthreads();      // the joined rows have been read: the ring is free
    }
    }
}

// -- the join of a pair's parts ------------------------------------------------

constexpr int JOIN_THREADS = 256;

// CTA (i, r): row r of the pair that the end of run i cuts, if no earlier end cuts it
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Walk P) {
    constexpr int W = JOIN_THREADS / 32, E = D / 32;
    __shared__ int64_t s_sum[W];
    __shared__ Spot s_spot;
    __shared__ float s_o[W][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y;
    Layout<JOIN_THREADS> lay;
    lay.count(P, s_sum);       // lengths are not what the kernel before this one writes
    const int64_t all = lay.total * P.c.kv_heads * P.head_tiles, used = runs_used(P, all);
    const int64_t i = blockIdx.x, cut = all * (i + 1) / used;
    const bool inside = i + 1 < used;
    const Spot at = spot_of(P, lay, inside ? cut : 0, &s_spot);
    // every CTA waits, also those without work: a kernel after this one may then
    // rely on the one before it
    dependency_wait();
    if (!inside || at.unit == 0) return;                                       // the cut lies between two pairs
    const int64_t p0 = cut - at.unit, p1 = p0 + at.units;           // the pair's units
    if (p0 < all * i / used) return;                                // run i does not begin it: an earlier cut has it
    const int g = at.h / P.head_tiles, ht = at.h % P.head_tiles;
    if (r >= min(P.tile_heads, P.group - ht * P.tile_heads)) return;
    const int64_t row = (int64_t)at.b * P.q_heads + g * P.group + ht * P.tile_heads + r;
    // runs i .. i + n - 1 hold parts: run i in its first place if the pair begins it, else in its second
    int64_t n = 1;
    while (all * (i + n) / used < p1) ++n;
    const int64_t part0 = 2 * i + (all * i / used == p0 ? 0 : 1);

    const float prior = P.prior_lse ? P.prior_lse[row] * LOG2E : NEG_INF;
    float m = prior;
    for (int64_t s = lane; s < n; s += 32) m = fmaxf(m, P.part_ml[(s ? 2 * (i + s) : part0) * ROWS + r].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, x));
    float l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int64_t s = warp; s < n; s += W) {
        const int64_t part = (s ? 2 * (i + s) : part0) * ROWS + r;
        const float2 ml = P.part_ml[part];
        float x[E];
        if constexpr (E == 4) {
            const float4 y = *reinterpret_cast<const float4*>(P.part_out + part * D + lane * 4);
            x[0] = y.x;
            x[1] = y.y;
            x[2] = y.z;
            x[3] = y.w;
        } else {
            const float2 y = *reinterpret_cast<const float2*>(P.part_out + part * D + lane * 2);
            x[0] = y.x;
            x[1] = y.y;
        }
        const float f = ml.y == 0.f ? 0.f : exp2_fast(ml.x - m);    // nothing seen there: 0
        l += ml.y * f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += x[e] * f;
    }
    if (warp == W - 1 && prior != NEG_INF) {
        const float f = exp2_fast(prior - m);
        l += f;
        const T* po = static_cast<const T*>(P.prior_out) + row * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += f * (float)po[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = acc[e];
    __shared__ float s_l[W];
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += s_l[w];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (threadIdx.x < D) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) y += s_o[w][threadIdx.x];
        static_cast<T*>(P.out)[row * D + threadIdx.x] = T(y * inv);
    }
    if (threadIdx.x == 0) {
        const float x = sum == 0.f ? NEG_INF : m + log2f(sum);
        P.lse[row] = x * LN2;
        if (P.lse2) P.lse2[row] = x;
    }
}

// -- the slots' weights ----------------------------------------------------------

struct Shares {
    Cache c;
    int q_heads, group, window, sinks;
    const float* logits;
    const float* lse2;
    float* weights;           // [seqs][kv_heads][width]
    int64_t width;
    int accumulate;
    int chunks;               // blocks of SHARE_SLOTS slots of a row of weights
};

constexpr int SHARE_THREADS = 256;
constexpr int SHARE_SLOTS = 1024;

// a slot's share of the softmax, summed over the query heads of its key head
__global__ void __launch_bounds__(SHARE_THREADS) share_kernel(const __grid_constant__ Shares P) {
    constexpr int PER = SHARE_SLOTS / SHARE_THREADS;
    int64_t item = blockIdx.x;
    const int chunk = (int)(item % P.chunks);
    item /= P.chunks;
    const int g = (int)(item % P.c.kv_heads), b = (int)(item / P.c.kv_heads);
    const int far = P.window > 0 ? max(0, P.c.lengths[b] - P.window) : 0;
    const int L = P.c.length(b);
    const int64_t s0 = (int64_t)chunk * SHARE_SLOTS + threadIdx.x;
    float acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    dependency_wait();
    const int64_t row0 = (int64_t)b * P.q_heads + (int64_t)g * P.group;
#pragma unroll 4
    for (int h = 0; h < P.group; ++h) {
        const float lse2 = P.lse2[row0 + h];
        const float off = lse2 == NEG_INF ? 0.f : lse2;             // nothing seen: every logit is -inf
        const float* x = P.logits + (row0 + h) * P.c.capacity();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t j = s0 + i * SHARE_THREADS;
            if (j < L && (j >= far || j < P.sinks)) acc[i] += exp2_fast(x[j] - off);
        }
    }
    float* w = P.weights + ((int64_t)b * P.c.kv_heads + g) * P.width;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int64_t j = s0 + i * SHARE_THREADS;
        if (j < P.width) w[j] = P.accumulate ? w[j] + acc[i] : acc[i];
    }
}

// -- host side --------------------------------------------------------------

// Whether every pair gets a warp of its own.  With short tables (search results)
// a run would be many short pairs one after the other, each a chain of dependent
// reads; a warp a pair has as many chains in flight as the SMs hold warps.  With
// long ones it needs enough pairs that the last round of unequal lengths is short.
inline bool warp_a_pair(const Cache& c, int64_t pairs) {
    const int64_t warps = 8ll * abi::num_sms();
    return c.capacity() <= 512 ? pairs >= warps / 2 : pairs >= 16 * warps;
}

template <typename T, int D, int W>
int launch_walk(const Walk& w, int64_t ctas, cudaStream_t st) {
    constexpr int ring = W * STAGES * 2 * KEYS * D * 2, joined = W * ROWS * D * 4;
    constexpr int smem = ring > joined ? ring : joined;
    cudaError_t e = cudaFuncSetAttribute(walk_kernel<T, D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return abi::cuda_fail(e, "cudaFuncSetAttribute(attention)");
    walk_kernel<T, D, W><<<(unsigned)ctas, W * 32, smem, st>>>(w);
    return abi::cuda_check("attention launch");
}

template <typename T, int D>
int launch_decode(const Walk& w, int64_t pairs, cudaStream_t st) {
    if (!w.runs) return launch_walk<T, D, 1>(w, pairs, st);
    const int rc = launch_walk<T, D, WARPS>(w, w.runs, st);
    if (rc || w.runs == 1) return rc;
    const cudaError_t e = launch_after(join_kernel<T, D>, dim3((unsigned)(w.runs - 1), (unsigned)w.tile_heads),
                                       dim3(JOIN_THREADS), 0, st, w);
    if (e != cudaSuccess) return abi::cuda_fail(e, "attention join launch");
    return abi::cuda_check("attention join launch");
}

struct Space {
    int runs;
    uint64_t out, ml, lse2, logits, total;   // byte offsets
};
inline int tiles_of(int group) { return (group + ROWS - 1) / ROWS; }
inline Space decode_space(const Cache& c, int d, int q_heads, bool weights) {
    Space s;
    const int64_t pairs = (int64_t)c.seqs * c.kv_heads * tiles_of(q_heads / c.kv_heads);
    s.runs = warp_a_pair(c, pairs) ? 0 : cta_per_sm(d) * abi::num_sms();
    // no more runs than there can be units
    const int64_t most = pairs * ((c.capacity() + UNIT - 1) / UNIT + 1);
    if (s.runs > most) s.runs = (int)most;
    const uint64_t rows = (uint64_t)c.seqs * q_heads;
    s.out = 0;
    s.ml = (uint64_t)s.runs * 2 * ROWS * d * 4;
    s.lse2 = s.ml + (uint64_t)s.runs * 2 * ROWS * 8;
    s.logits = s.lse2 + (weights ? (rows * 4 + 15) / 16 * 16 : 0);
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
    Walk w = {};
    int rc = check_cache(cache, &w.c);
    if (rc) return rc;
    const Cache& c = w.c;
    if (c.seqs == 0) return SWB_OK;
    rc = check_query(q, q_seq_stride, q_head_stride, q_heads, c);
    if (rc) return rc;
    if (!out || !lse) return abi::fail(SWB_ERR_ARG, "null output");
    if (window < 0 || sinks < 0) return abi::fail(SWB_ERR_ARG, "window and sinks must not be negative");
    if (!prior_out != !prior_lse) return abi::fail(SWB_ERR_ARG, "a prior part needs its rows and its lse");
    if (weights && weights_width < c.capacity())
        return abi::fail(SWB_ERR_ARG, "weights are narrower than the page table's slots");
    const int d = cache->head_dim;
    const Space sp = decode_space(c, d, q_heads, weights != nullptr);
    if (sp.total && (!workspace || ws_bytes < sp.total)) return abi::fail(SWB_ERR_ARG, "workspace too small");
    cudaStream_t st = (cudaStream_t)stream;
    char* ws = static_cast<char*>(workspace);
    w.q = q;
    w.q_seq_stride = q_seq_stride;
    w.q_head_stride = q_head_stride;
    w.q_heads = q_heads;
    w.group = q_heads / c.kv_heads;
    w.tile_heads = w.group < ROWS ? w.group : ROWS;
    w.head_tiles = tiles_of(w.group);
    w.scale2 = scale * LOG2E;
    w.window = window;
    w.sinks = sinks;
    w.prior_out = prior_out;
    w.prior_lse = prior_lse;
    w.out = out;
    w.lse = lse;
    w.runs = sp.runs;
    w.part_out = reinterpret_cast<float*>(ws + sp.out);
    w.part_ml = reinterpret_cast<float2*>(ws + sp.ml);
    w.lse2 = weights ? reinterpret_cast<float*>(ws + sp.lse2) : nullptr;
    w.logits = weights ? reinterpret_cast<float*>(ws + sp.logits) : nullptr;
    const int64_t pairs = (int64_t)c.seqs * c.kv_heads * w.head_tiles;
    const int64_t chunks = (weights_width + SHARE_SLOTS - 1) / SHARE_SLOTS;
    const int64_t shares = weights ? chunks * c.seqs * c.kv_heads : 0;
    if (pairs >= ((int64_t)1 << 31) || shares >= ((int64_t)1 << 31))
        return abi::fail(SWB_ERR_ARG, "too many sequences in one call");
    if (cache->dtype == SWB_F16)
        rc = d == 64 ? launch_decode<__half, 64>(w, pairs, st) : launch_decode<__half, 128>(w, pairs, st);
    else
        rc = d == 64 ? launch_decode<__nv_bfloat16, 64>(w, pairs, st) : launch_decode<__nv_bfloat16, 128>(w, pairs, st);
    if (rc || !weights) return rc;
    Shares h = {};
    h.c = c;
    h.q_heads = q_heads;
    h.group = w.group;
    h.window = window;
    h.sinks = sinks;
    h.logits = w.logits;
    h.lse2 = w.lse2;
    h.weights = weights;
    h.width = weights_width;
    h.accumulate = accumulate;
    h.chunks = (int)chunks;
    const cudaError_t e = launch_after(share_kernel, dim3((unsigned)shares), dim3(SHARE_THREADS), 0, st, h);
    if (e != cudaSuccess) return abi::cuda_fail(e, "attention weights launch");
    return abi::cuda_check("attention weights launch");
}
