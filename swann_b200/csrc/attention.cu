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
// not seen filled with zeros, so nothing that lies in them reaches a product).
// Logits and the weighted sum run on mma.sync with fp32 accumulators, as K Q^T and
// V^T P^T: keys and dimensions fill the 16 rows of a product and the query rows
// its 8 columns, so a group of up to 8 heads wastes little (a tcgen05 tile of 128
// would be nine tenths empty, and the tensor pipe is not what bounds this).
// Weights are rounded to the cache's 16 bits for the second product, as its other
// operand is; their sum l is taken before that.  In fp16 they and l are 2^15 times
// what they are against the running maximum, so that those of a long flat tail
// beside one strong key stay far above fp16's smallest steps.
//
// Who walks what.  Few pairs: the pairs' units of 64 keys are laid end to end
// and every CTA of a grid that the SMs hold at once takes an equal run of them,
// whatever the sequences' lengths are; a pair cut by the end of a run leaves
// parts (m, l, unnormalised rows), at most two a CTA, which a second kernel
// joins.  Many short pairs: a warp a pair.
//
// Measured: 48 sequences of up to 8191 slots, 32 heads of 128 over 8: 95 us, 6.1 TB/s
// (94% of a copy's rate); one of 131071 slots with 4 key heads and weights: 62 us, of
// which 46 walk; one of 1027: 7 us, launch and latency.

#include "attn.cuh"

namespace swb {
namespace attn {

constexpr int WARPS = 4;      // of a CTA that takes a run of units
constexpr int ROWS = 16;      // query rows of a tile, at most
constexpr int KEYS = 16;      // keys a warp scores at a time
constexpr int UNIT = WARPS * KEYS;

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
    int4* cuts;               // [runs] the pair that run i begins and leaves to others: its first
                              // output row, rows, parts, first part
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

// the slot of sequence b's newest token, -1 without one
__device__ __forceinline__ int newest(const Cache& c, int b) { return max(c.lengths[b], 0) - 1; }

template <int D>
__device__ __forceinline__ uint32_t swz(int row, int chunk) {
    return (uint32_t)(row * D * 2 + ((chunk ^ (row & 7)) << 4));
}

__device__ __forceinline__ int units_of(const Walk& P, int b) {
    const Range r = visible(newest(P.c, b), P.window, P.sinks, P.c.capacity());
    return max(1, (r.n + UNIT - 1) / UNIT);
}

// The sequences' units laid end to end, counted by every warp for itself (no
// barrier): lane t sums a stretch of sequences.
struct Units {
    int before, mine;         // units of one head tile ahead of this lane's stretch, and in it
    int total;                // of one head tile
    int per;                  // sequences of a stretch
    __device__ __forceinline__ void count(const Walk& P) {
        const int lane = threadIdx.x & 31;
        per = (P.c.seqs + 31) / 32;
        const int b0 = min(P.c.seqs, lane * per), b1 = min(P.c.seqs, b0 + per);
        mine = 0;
#pragma unroll 4
        for (int b = b0; b < b1; ++b) mine += units_of(P, b);
        int sum = mine;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int y = __shfl_up_sync(FULL, sum, s);
            if (lane >= s) sum += y;
        }
        before = sum - mine;
        total = __shfl_sync(FULL, sum, 31);
    }
};

// a place among the units: a pair, its key head tile and the unit inside it
struct Spot {
    int b, h;                 // sequence; key head * head_tiles + tile
    int unit, units;          // of the pair
};

// where unit x of the whole lies, by every warp for itself.  Sequence-major: all
// head tiles of a sequence, then the next.
__device__ __forceinline__ Spot spot_of(const Walk& P, const Units& U, int x) {
    const int tiles = P.c.kv_heads * P.head_tiles, lane = threadIdx.x & 31;
    int left = x - U.before * tiles;
    const bool here = left >= 0 && left < U.mine * tiles;
    Spot at = {0, 0, 0, 1};
    if (here) {
        int n;
        for (at.b = lane * U.per;; ++at.b) {
            n = units_of(P, at.b);
            if (left < n * tiles) break;
            left -= n * tiles;
        }
        at.units = n;
        at.h = left / n;
        at.unit = left - at.h * n;
    }
    const int src = __ffs(__ballot_sync(FULL, here)) - 1;
    at.b = __shfl_sync(FULL, at.b, src);
    at.h = __shfl_sync(FULL, at.h, src);
    at.unit = __shfl_sync(FULL, at.unit, src);
    at.units = __shfl_sync(FULL, at.units, src);
    return at;
}

// `all` units in `used` runs that differ by one unit at most
struct Runs {
    int used, size, more;     // the first `more` runs have size + 1 units
    __device__ __forceinline__ Runs(int all, int runs) : used(min(runs, all)), size(all / used), more(all - used * size) {}
    __device__ __forceinline__ int begin(int i) const { return i * size + min(i, more); }
    __device__ __forceinline__ int owner(int x) const {
        const int big = more * (size + 1);
        return x < big ? x / (size + 1) : more + (x - big) / size;
    }
};

// 8 x 8 16-bit elements across a warp, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

constexpr int STAGES = 3;                              // of a warp's ring
// CTAs of a run that an SM holds, by shared memory and registers
constexpr int cta_per_sm(int d) { return d == 128 ? 2 : 4; }

// What a warp keeps of the rows of a pair: this thread's columns of the products
// are the heads n * 8 + (lane & 3) * 2 + e, its keys lane / 4 and lane / 4 + 8, its
// dimensions j * 16 + lane / 4 and + 8.
template <typename T, int D, int NT>
struct Rows {
    static constexpr int MT = D / 16;
    static constexpr float LIFT = Elem<T>::TOP;        // log2 of what weights are multiplied by
    float o[MT][NT][4], m[NT][2], l[NT][2];
    uint32_t q[D / 16][NT][2];                         // the query rows as fragments of the second operand

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < MT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[j][n][e] = 0.f;
            m[n][0] = m[n][1] = NEG_INF;
            l[n][0] = l[n][1] = 0.f;
        }
    }
    // q: the first row; rows from `heads` on are zeros
    __device__ __forceinline__ void load_q(const T* q0, int64_t stride, int heads, int lane) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = n * 8 + (lane >> 2);
            const T* qr = q0 + r * stride + (lane & 3) * 2;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                q[kk][n][0] = r < heads ? *reinterpret_cast<const uint32_t*>(qr + kk * 16) : 0u;
                q[kk][n][1] = r < heads ? *reinterpret_cast<const uint32_t*>(qr + kk * 16 + 8) : 0u;
            }
        }
    }
    // one block of 16 keys: K at `st`, V behind it; bit k of `seen`: key k counts.
    // logit(n, e, value) is told every logit.
    template <typename F>
    __device__ __forceinline__ void block(uint32_t st, unsigned seen, float scale2, int lane, F logit) {
        float y[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[n][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t f[4];
            ldmatrix4(f, st + swz<D>(((lane >> 3) & 1) * 8 + (lane & 7), 2 * kk + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < NT; ++n) Elem<T>::mma(y[n], f, q[kk][n][0], q[kk][n][1]);
        }
        const bool see0 = (seen >> (lane >> 2)) & 1u, see1 = (seen >> ((lane >> 2) + 8)) & 1u;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[n][e] = (e < 2 ? see0 : see1) ? y[n][e] * scale2 : NEG_INF;
                logit(n, e, y[n][e]);
            }
        bool grows = false;
        float a[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                a[n][e] = fmaxf(y[n][e], y[n][e + 2]);
#pragma unroll
                for (int s = 4; s <= 16; s <<= 1) a[n][e] = fmaxf(a[n][e], __shfl_xor_sync(FULL, a[n][e], s));
                grows = grows || a[n][e] > m[n][e];
            }
        if (__any_sync(FULL, grows)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float t = fmaxf(m[n][e], a[n][e]);
                    f[e] = t == NEG_INF ? 1.f : exp2_fast(m[n][e] - t);
                    m[n][e] = t;
                    l[n][e] *= f[e];
                }
#pragma unroll
                for (int j = 0; j < MT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][n][e] *= f[e & 1];
            }
        }
        uint32_t pf[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float s0 = m[n][0] == NEG_INF ? 0.f : m[n][0] - LIFT, s1 = m[n][1] == NEG_INF ? 0.f : m[n][1] - LIFT;
            const float w0 = exp2_fast(y[n][0] - s0), w1 = exp2_fast(y[n][1] - s1);
            const float w2 = exp2_fast(y[n][2] - s0), w3 = exp2_fast(y[n][3] - s1);
            l[n][0] += w0 + w2;
            l[n][1] += w1 + w3;
            pf[n][0] = transposed(Elem<T>::pack(w0, w1));
            pf[n][1] = transposed(Elem<T>::pack(w2, w3));
        }
        const uint32_t sv = st + KEYS * D * 2;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            uint32_t f[4];
            ldmatrix4_t(f, sv + swz<D>((lane >> 4) * 8 + (lane & 7), 2 * j + ((lane >> 3) & 1)));
#pragma unroll
            for (int n = 0; n < NT; ++n) Elem<T>::mma(o[j][n], f, pf[n][0], pf[n][1]);
        }
    }
    // the sums over all keys: l of a column in every lane that has it; from here on m is
    // what l and o are weights against, LIFT below the maximum
    __device__ __forceinline__ void sum() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int s = 4; s <= 16; s <<= 1) l[n][e] += __shfl_xor_sync(FULL, l[n][e], s);
                m[n][e] -= LIFT;
            }
    }
};

// 16 rows of K and of V into a stage; lane < 16 has the element offset of row
// `lane`, -1 for zeros.  Which rows are there.
template <typename T, int D>
__device__ __forceinline__ unsigned copy_block(uint32_t st, const T* kp, const T* vp, int64_t off, int lane) {
    constexpr int CH = D / 8;
#pragma unroll
    for (int it = 0; it < KEYS * CH / 32; ++it) {
        const int r = (it * 32 + lane) / CH, c = (it * 32 + lane) % CH;
        const int64_t o = __shfl_sync(FULL, (long long)off, r);
        const bool real = o >= 0;
        const int64_t e = real ? o + c * 8 : 0;
        cp_async16_or_zero(st + swz<D>(r, c), kp + e, real);
        cp_async16_or_zero(st + KEYS * D * 2 + swz<D>(r, c), vp + e, real);
    }
    return __ballot_sync(FULL, off >= 0);
}

// four dimensions of a row that is whole but for the prior part: joined and written
template <typename T, int D>
__device__ __forceinline__ void write_row(const Walk& P, int64_t row, int d, float4 acc, float top, float sum) {
    const float pm = P.prior_lse ? P.prior_lse[row] * LOG2E : NEG_INF;
    const float most = fmaxf(top, pm);
    const float fa = sum == 0.f ? 0.f : exp2_fast(top - most), fb = pm == NEG_INF ? 0.f : exp2_fast(pm - most);
    const float whole = sum * fa + fb;
    const float inv = whole == 0.f ? 0.f : 1.f / whole;
    acc = make_float4(acc.x * fa, acc.y * fa, acc.z * fa, acc.w * fa);
    if (pm != NEG_INF) {
        const uint2 z = *reinterpret_cast<const uint2*>(static_cast<const T*>(P.prior_out) + row * D + d);
        const float2 z0 = Elem<T>::wide(z.x), z1 = Elem<T>::wide(z.y);
        acc.x += fb * z0.x;
        acc.y += fb * z0.y;
        acc.z += fb * z1.x;
        acc.w += fb * z1.y;
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(P.out) + row * D + d) =
        make_uint2(Elem<T>::pack(acc.x * inv, acc.y * inv), Elem<T>::pack(acc.z * inv, acc.w * inv));
    if (d == 0) {
        const float z = whole == 0.f ? NEG_INF : most + log2f(whole);
        P.lse[row] = z * LN2;
        if (P.lse2) P.lse2[row] = z;
    }
}

// An equal run of units a CTA; up to 8 * NT query rows
template <typename T, int D, int NT>
__global__ void __launch_bounds__(WARPS * 32, cta_per_sm(D)) walk_kernel(const __grid_constant__ Walk P) {
    constexpr int W = WARPS, THREADS = W * 32;
    constexpr int STAGE = 2 * KEYS * D * 2;            // K and V of a block of keys
    constexpr int R = 8 * NT;
    constexpr int LD = D + 4;                          // of the joined rows: no two of a warp's stores meet in a bank
    extern __shared__ __align__(128) char smem[];
    __shared__ unsigned s_seen[W][STAGES];
    __shared__ float s_m[W][R], s_l[W][R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = smem_u32(smem) + warp * (STAGES * STAGE);
    const int tiles = P.c.kv_heads * P.head_tiles;

    // -- which pairs, and which of their keys
    Units U;
    U.count(P);
    const Runs runs(U.total * tiles, P.runs);
    if (threadIdx.x == 0) P.cuts[blockIdx.x] = make_int4(0, 0, 0, 0);
    if ((int)blockIdx.x >= runs.used) return;
    int x = runs.begin(blockIdx.x), left = runs.begin(blockIdx.x + 1) - x;    // the next unit; units still to walk
    Spot at = spot_of(P, U, x);

    for (bool first = true; left > 0; first = false) {
        const int b = at.b, g = at.h / P.head_tiles, ht = at.h % P.head_tiles;
        const int heads = min(P.tile_heads, P.group - ht * P.tile_heads);
        const int64_t row0 = (int64_t)b * P.q_heads + g * P.group + ht * P.tile_heads;   // first output row
        const Range rg = visible(newest(P.c, b), P.window, P.sinks, P.c.capacity());
        const int take = min(left, at.units - at.unit);
        const int u0 = min(rg.n, at.unit * UNIT), u1 = min(rg.n, u0 + take * UNIT);
        const bool entire = take == at.units;          // nothing of the pair is left to others
        const int nblk = (u1 - u0 + KEYS - 1) / KEYS;  // blocks of the stretch; warp w has w, w + W, ..
        const int mine = nblk > warp ? (nblk - warp - 1) / W + 1 : 0;

        const T* kp = static_cast<const T*>(P.c.k) + (int64_t)g * P.c.head_stride;
        const T* vp = static_cast<const T*>(P.c.v) + (int64_t)g * P.c.head_stride;
        // lane < 16: the row of key `lane` of this warp's block i, or -1
        auto find = [&](int i) -> int64_t {
            const int u = u0 + (i * W + warp) * KEYS + lane;
            return (lane < KEYS && i < mine && u < u1) ? P.c.row(b, rg.slot(u)) : -1;
        };
        auto issue = [&](int i, int64_t off) {
            if (i < mine) {
                const unsigned seen = copy_block<T, D>(ring + (i % STAGES) * STAGE, kp, vp, off, lane);
                if (lane == 0) s_seen[warp][i % STAGES] = seen;
            }
            cp_async_commit();
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) issue(i, find(i));
        int64_t next = find(STAGES - 1);

        Rows<T, D, NT> rows;
        rows.load_q(static_cast<const T*>(P.q) + b * P.q_seq_stride +
                        (int64_t)(g * P.group + ht * P.tile_heads) * P.q_head_stride,
                    P.q_head_stride, heads, lane);
        rows.clear();
        for (int i = 0; i < mine; ++i) {
            cp_async_wait<STAGES - 2>();
            __syncwarp();
            issue(i + STAGES - 1, next);      // into the stage that block i - 1 has left
            next = find(i + STAGES);
            rows.block(ring + (i % STAGES) * STAGE, s_seen[warp][i % STAGES], P.scale2, lane, [&](int n, int e, float y) {
                if (!P.logits) return;
                const int r = n * 8 + (lane & 3) * 2 + (e & 1);
                const int u = u0 + (i * W + warp) * KEYS + (lane >> 2) + (e < 2 ? 0 : 8);
                if (r < heads && u < u1) P.logits[(row0 + r) * P.c.capacity() + rg.slot(u)] = y;
            });
            __syncwarp();
        }
        cp_async_wait<0>();

        // -- join the warps
        rows.sum();
        if (lane < 4)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s_m[warp][n * 8 + lane * 2 + e] = rows.m[n][e];
                    s_l[warp][n * 8 + lane * 2 + e] = rows.l[n][e];
                }
        __syncthreads();      // the ring is free too
        float* so = reinterpret_cast<float*>(smem);    // [W][R][LD]
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = n * 8 + (lane & 3) * 2 + e;
                float top = NEG_INF;
#pragma unroll
                for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][r]);
                const float f = rows.l[n][e] == 0.f ? 0.f : exp2_fast(rows.m[n][e] - top);
                float* dst = so + (warp * R + r) * LD + (lane >> 2);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    dst[j * 16] = rows.o[j][n][e] * f;
                    dst[j * 16 + 8] = rows.o[j][n][e + 2] * f;
                }
            }
        __syncthreads();
        for (int i = threadIdx.x; i < heads * (D / 4); i += THREADS) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float top = NEG_INF, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][r]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (s_l[w][r] != 0.f) sum += s_l[w][r] * exp2_fast(s_m[w][r] - top);
                const float4 z = *reinterpret_cast<const float4*>(so + (w * R + r) * LD + d);
                acc.x += z.x;
                acc.y += z.y;
                acc.z += z.z;
                acc.w += z.w;
            }
            if (entire) {
                write_row<T, D>(P, row0 + r, d, acc, top, sum);
            } else {
                const int64_t part = (2 * (int64_t)blockIdx.x + (first ? 0 : 1)) * ROWS + r;
                *reinterpret_cast<float4*>(P.part_out + part * D + d) = acc;
                if (d == 0) P.part_ml[part] = make_float2(top, sum);
            }
        }
        if (!entire && at.unit == 0 && threadIdx.x == 0) {
            // the pair begins here and goes on in the runs that follow
            const int last = runs.owner(x + at.units - 1);
            P.cuts[blockIdx.x] = make_int4((int)row0, heads, last - (int)blockIdx.x + 1, 2 * blockIdx.x + (first ? 0 : 1));
        }
        left -= take;
        x += take;
        if (left > 0) {
            at.unit = 0;
            if (++at.h == tiles) {
                at.h = 0;
                ++at.b;
                at.units = units_of(P, at.b);
            }
            __syncthreads();      // the joined rows have been read: the ring is free
        }
    }
}

// -- many short pairs -----------------------------------------------------------

constexpr int PAIR_STAGES = 2;
// one-warp CTAs that an SM holds: with short pairs what counts is how many chains of
// dependent reads (length, table, rows) are under way, so few stages and many warps
constexpr int pair_ctas(int d) { return d == 128 ? 12 : 16; }

// A warp a pair.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(32, pair_ctas(D)) pair_kernel(const __grid_constant__ Walk P) {
    constexpr int STAGE = 2 * KEYS * D * 2, LD = D + 4;
    extern __shared__ __align__(128) char smem[];      // the stages; then the rows on their way out
    const int lane = threadIdx.x;
    const uint32_t ring = smem_u32(smem);
    const int tiles = P.c.kv_heads * P.head_tiles;
    const int b = (int)(blockIdx.x / tiles), h = (int)(blockIdx.x % tiles), g = h / P.head_tiles, ht = h % P.head_tiles;
    const int heads = min(P.tile_heads, P.group - ht * P.tile_heads), head0 = g * P.group + ht * P.tile_heads;
    const int64_t row0 = (int64_t)b * P.q_heads + head0;
    const Range rg = visible(newest(P.c, b), P.window, P.sinks, P.c.capacity());
    const int blocks = (rg.n + KEYS - 1) / KEYS;
    const T* kp = static_cast<const T*>(P.c.k) + (int64_t)g * P.c.head_stride;
    const T* vp = static_cast<const T*>(P.c.v) + (int64_t)g * P.c.head_stride;
    unsigned seen[PAIR_STAGES];
    auto find = [&](int i) -> int64_t {
        const int u = i * KEYS + lane;
        return lane < KEYS && u < rg.n ? P.c.row(b, rg.slot(u)) : -1;
    };
    seen[1] = blocks > 0 ? copy_block<T, D>(ring, kp, vp, find(0), lane) : 0u;
    cp_async_commit();
    int64_t next = find(1);
    Rows<T, D, NT> rows;
    rows.load_q(static_cast<const T*>(P.q) + b * P.q_seq_stride + (int64_t)head0 * P.q_head_stride, P.q_head_stride, heads, lane);
    rows.clear();
    for (int i = 0; i < blocks; ++i) {
        cp_async_wait<0>();
        __syncwarp();
        seen[0] = seen[1];
        if (i + 1 < blocks) seen[1] = copy_block<T, D>(ring + ((i + 1) & 1) * STAGE, kp, vp, next, lane);
        cp_async_commit();
        next = find(i + 2);
        if (seen[0] || P.logits) rows.block(ring + (i & 1) * STAGE, seen[0], P.scale2, lane, [&](int n, int e, float y) {
            if (!P.logits) return;
            const int r = n * 8 + (lane & 3) * 2 + (e & 1), u = i * KEYS + (lane >> 2) + (e < 2 ? 0 : 8);
            if (r < heads && u < rg.n) P.logits[(row0 + r) * P.c.capacity() + rg.slot(u)] = y;
        });
        __syncwarp();
    }
    cp_async_wait<0>();
    rows.sum();
    float* out = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = n * 8 + (lane & 3) * 2 + e;
            if (r >= heads) continue;
            float* dst = out + r * LD + (lane >> 2);
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
                dst[j * 16] = rows.o[j][n][e];
                dst[j * 16 + 8] = rows.o[j][n][e + 2];
            }
            if (lane < 4) {
                out[r * LD + D] = rows.m[n][e];
                out[r * LD + D + 1] = rows.l[n][e];
            }
        }
    __syncwarp();
    for (int c = lane; c < heads * (D / 4); c += 32) {
        const int r = c / (D / 4), d = c % (D / 4) * 4;
        const float* src = out + r * LD;
        write_row<T, D>(P, row0 + r, d, *reinterpret_cast<const float4*>(src + d), src[D], src[D + 1]);
    }
}

// A warp a pair of one query row: what a search of each head's keys gives.  There a
// matrix product would be seven eighths empty and most of its instructions spent on
// bringing operands into place (35 us against 26 for 4096 queries of up to 100 rows),
// so rows go straight into registers: D / 8 lanes have a row's 16-byte chunks, 32 / (D
// / 8) rows at a time, and a row's sum is folded over its lanes.
// Eight rows at a time keep its registers low (7 CTAs an SM): all warps of 4096 pairs
// are resident and wait for their rows side by side (26 us; 16 rows and 5 CTAs 30, 4
// rows and 9 CTAs 32).
constexpr int ROW_WARPS = 4, ROW_KEYS = 8;
template <typename T, int D>
__global__ void __launch_bounds__(ROW_WARPS * 32, 7) row_kernel(const __grid_constant__ Walk P, int64_t pairs) {
    constexpr int CH = D / 8, AT = 32 / CH, NI = ROW_KEYS / AT;     // lanes of a row; rows at a time; times
    const int lane = threadIdx.x & 31, c = lane % CH, sub = lane / CH;
    const int64_t pair = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5);
    if (pair >= pairs) return;                                   // whole warps; nothing below is the CTA's
    const int b = (int)(pair / P.c.kv_heads), g = (int)(pair % P.c.kv_heads);
    const Range rg = visible(newest(P.c, b), P.window, P.sinks, P.c.capacity());
    const int64_t head = (int64_t)g * P.c.head_stride + c * 8;
    const T* kp = static_cast<const T*>(P.c.k) + head;
    const T* vp = static_cast<const T*>(P.c.v) + head;
    auto find = [&](int u) -> int64_t { return u < rg.n ? P.c.row(b, rg.slot(u)) : -1; };
    int64_t next = find(lane);                                   // rows are looked up 32 at a time, one time ahead
    float q[8];
    {
        const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const T*>(P.q) + b * P.q_seq_stride + g * P.q_head_stride + c * 8);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = Elem<T>::wide(w[e]);
            q[2 * e] = f.x;
            q[2 * e + 1] = f.y;
        }
    }
    float m = NEG_INF, l = 0.f, acc[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int u1 = 0; u1 < rg.n; u1 += 32) {
        const int64_t off = next;
        next = find(u1 + 32 + lane);
        const unsigned there = __ballot_sync(FULL, off >= 0);
        for (int k0 = 0; k0 < 32 && u1 + k0 < rg.n; k0 += ROW_KEYS) {
            // a search pads with -1 what it did not find
            if (!P.logits && !((there >> k0) & ((1u << ROW_KEYS) - 1u))) continue;
            const int u0 = u1 + k0;
            uint4 k[NI], v[NI];
            bool real[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int64_t o = __shfl_sync(FULL, (long long)off, k0 + i * AT + sub);
                real[i] = o >= 0;
                k[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
                if (real[i]) {
                    k[i] = ld_row16(reinterpret_cast<const uint4*>(kp + o));
                    v[i] = ld_row16(reinterpret_cast<const uint4*>(vp + o));
                }
            }
            float x[NI], top = NEG_INF;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const uint32_t w[4] = {k[i].x, k[i].y, k[i].z, k[i].w};
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = Elem<T>::wide(w[e]);
                    s = fmaf(q[2 * e], f.x, s);
                    s = fmaf(q[2 * e + 1], f.y, s);
                }
                x[i] = s;
            }
#pragma unroll
            for (int s = CH / 2; s > 0; s >>= 1)
#pragma unroll
                for (int i = 0; i < NI; ++i) x[i] += __shfl_xor_sync(FULL, x[i], s);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                x[i] = real[i] ? x[i] * P.scale2 : NEG_INF;
                top = fmaxf(top, x[i]);
                const int u = u0 + i * AT + sub;
                if (P.logits && c == 0 && u < rg.n) P.logits[((int64_t)b * P.q_heads + g) * P.c.capacity() + rg.slot(u)] = x[i];
            }
#pragma unroll
            for (int s = CH; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, s));
            if (top > m) {                                           // the same in all lanes
                const float f = exp2_fast(m - top);
                m = top;
                l *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] *= f;
            }
            const float base = m == NEG_INF ? 0.f : m;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const float p = exp2_fast(x[i] - base);
                l += p;
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = Elem<T>::wide(w[e]);
                    acc[2 * e] = fmaf(p, f.x, acc[2 * e]);
                    acc[2 * e + 1] = fmaf(p, f.y, acc[2 * e + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int s = CH; s < 32; s <<= 1) {
        l += __shfl_xor_sync(FULL, l, s);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += __shfl_xor_sync(FULL, acc[e], s);
    }
    // the lanes of the first two row places write four dimensions each
    if (sub < 2)
        write_row<T, D>(P, (int64_t)b * P.q_heads + g, c * 8 + sub * 4,
                        sub ? make_float4(acc[4], acc[5], acc[6], acc[7]) : make_float4(acc[0], acc[1], acc[2], acc[3]), m, l);
}

// -- the join of a pair's parts ------------------------------------------------

constexpr int JOIN_THREADS = 256;

// by a CTA: row r of the pair that run i begins and others go on with, if any
template <typename T, int D>
__device__ __forceinline__ void join_row(const Walk& P, int i, int r) {
    constexpr int W = JOIN_THREADS / 32, E = D / 32;
    __shared__ float s_o[W][D], s_l[W];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int4 cut = P.cuts[i];
    if (r >= cut.y) return;
    const int64_t row = (int64_t)cut.x + r;
    const int n = cut.z, part0 = cut.w;

    const float prior = P.prior_lse ? P.prior_lse[row] * LOG2E : NEG_INF;
    float m = prior;
    for (int s = lane; s < n; s += 32) m = fmaxf(m, P.part_ml[(int64_t)(s ? 2 * (i + s) : part0) * ROWS + r].x);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL, m, x));
    float l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
    for (int s = warp; s < n; s += W) {
        const int64_t part = (int64_t)(s ? 2 * (i + s) : part0) * ROWS + r;
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

template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(const __grid_constant__ Walk P) {
    // every CTA waits, also those without work: what comes after this kernel may then
    // rely on the one before it
    dependency_wait();
    join_row<T, D>(P, blockIdx.x, blockIdx.y);
}

// -- the slots' weights ----------------------------------------------------------

struct Shares {
    float* weights;           // [seqs][kv_heads][width]
    int64_t width;
    int accumulate;
    int chunks;               // CTAs of a row of weights
    int64_t ctas;             // of all rows
};

// Slots of a CTA.  Its heads' sums cost it as much as some thousand slots do, and long
// stretches leave SMs idle; by thread, at 131071 slots of 4 key heads, the whole call
// takes 77.0 us with one, 66.4 with 2, 62.1 with 4, 61.6 with 8 and 64.0 with 16.
constexpr int SHARE_SLOTS = 8 * JOIN_THREADS;
constexpr int SHARE_HEADS = 64;                 // whose sums a CTA finds at a time

// The first CTAs write the slots' weights, the rest join the cut pairs' rows, side by
// side: a slot's share needs its heads' sums, which a cut pair's parts give as well
// as the joined row does.  One kernel after the other took 63.9 us where this takes
// 61.6 (fp16, 32 heads on 4, 131071 slots); both wait for memory rather than fill it.
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_THREADS) finish_kernel(const __grid_constant__ Walk P,
                                                              const __grid_constant__ Shares S) {
    if ((int64_t)blockIdx.x >= S.ctas) {
        const int x = (int)(blockIdx.x - S.ctas);
        dependency_wait();
        join_row<T, D>(P, x / P.tile_heads, x % P.tile_heads);
        return;
    }
    __shared__ float s_off[SHARE_HEADS];
    constexpr int PER = SHARE_SLOTS / JOIN_THREADS, W = JOIN_THREADS / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunk = (int)(blockIdx.x % S.chunks), bg = (int)(blockIdx.x / S.chunks);
    const int b = bg / P.c.kv_heads, g = bg - b * P.c.kv_heads;
    const int far = P.window > 0 ? max(0, P.c.lengths[b] - P.window) : 0;
    const int L = P.c.length(b);
    // where the pairs of this key head lie among the runs: lengths are not what the
    // kernel before this one writes, so all this is found beside it
    const int tiles = P.c.kv_heads * P.head_tiles, units = units_of(P, b);
    int base = 0, all = 1;
    if (P.runs > 1) {
        Units U;
        U.count(P);
        all = U.total * tiles;
        const int src = b / U.per;
        int before = U.before;
        if (lane == src)
            for (int k = src * U.per; k < b; ++k) before += units_of(P, k);
        base = __shfl_sync(FULL, before, src) * tiles;
    }
    const Runs runs(all, max(1, P.runs));
    dependency_wait();

    const int64_t s0 = (int64_t)chunk * SHARE_SLOTS + threadIdx.x, row0 = (int64_t)b * P.q_heads + (int64_t)g * P.group;
    float acc[PER];
    bool seen[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int64_t j = s0 + k * JOIN_THREADS;
        acc[k] = 0.f;
        seen[k] = j < L && (j >= far || j < P.sinks);
    }
    for (int h0 = 0; h0 < P.group; h0 += SHARE_HEADS) {
        const int h1 = min(P.group, h0 + SHARE_HEADS);
        __syncthreads();
        for (int h = h0 + warp; h < h1; h += W) {
            const int ht = h / P.tile_heads, r = h - ht * P.tile_heads;
            const int first = base + (g * P.head_tiles + ht) * units;
            const int i = P.runs > 1 ? runs.owner(first) : 0;
            const int n = P.runs > 1 ? runs.owner(first + units - 1) - i + 1 : 1;
            float lse2;
            if (n == 1) {
                lse2 = P.lse2[row0 + h];          // the walk had the whole pair
            } else {
                const int part0 = 2 * i + (runs.begin(i) == first ? 0 : 1);
                const float prior = P.prior_lse ? P.prior_lse[row0 + h] * LOG2E : NEG_INF;
                auto part = [&](int s) { return P.part_ml[(int64_t)(s ? 2 * (i + s) : part0) * ROWS + r]; };
                float top = prior, l = 0.f;
                for (int s = lane; s < n; s += 32) top = fmaxf(top, part(s).x);
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, s));
                for (int s = lane; s < n; s += 32) {
                    const float2 y = part(s);
                    if (y.y != 0.f) l += y.y * exp2_fast(y.x - top);
                }
                if (lane == 0 && prior != NEG_INF) l += exp2_fast(prior - top);
#pragma unroll
                for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(FULL, l, s);
                lse2 = l == 0.f ? NEG_INF : top + log2f(l);
            }
            if (lane == 0) s_off[h - h0] = lse2 == NEG_INF ? 0.f : lse2;   // nothing seen: every logit is -inf
        }
        __syncthreads();
#pragma unroll 2
        for (int h = h0; h < h1; ++h) {
            const float off = s_off[h - h0];
            const float* x = P.logits + (row0 + h) * P.c.capacity();
            float y[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) y[k] = seen[k] ? x[s0 + k * JOIN_THREADS] : NEG_INF;
#pragma unroll
            for (int k = 0; k < PER; ++k) acc[k] += exp2_fast(y[k] - off);
        }
    }
    float* w = S.weights + (int64_t)bg * S.width;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int64_t j = s0 + k * JOIN_THREADS;
        if (j < S.width) w[j] = S.accumulate ? w[j] + acc[k] : acc[k];
    }
}

// -- host side --------------------------------------------------------------

// Whether a warp takes a whole pair.  Where pairs are many and short (search results) a
// run of a CTA would be many of them, each joined by its warps; where they are few or
// long, a warp a pair leaves SMs idle, more so with one query row, whose kernel loads
// little at a time.  Lengths uniform up to the table's slots, fp16, head_dim 128, us by
// runs / by whole pairs:
//   one row    512 slots: 592 pairs 26 / 94, 4096 140 / 118;  128 slots: 1184 23 / 22, 4096 82 / 34
//              2048 slots: 18944 pairs 1661 / 1790
//   four rows  512 slots: 148 pairs 11 / 23, 1184 39 / 34;  2048 slots: 592 52 / 100, 18944 1310 / 1243
// The two meet where pairs are about twice the slots (2 to 16 rows, head_dim 64 and 128,
// 64 to 4096 slots), with one row about eight times and beyond 1024 slots nowhere.
inline bool whole_pairs(const Cache& c, int group, int64_t pairs) {
    const int64_t sms = abi::num_sms(), slots = c.capacity();
    if (group == 1) return slots <= 1024 && pairs >= 4 * sms && pairs >= 8 * slots;
    return pairs >= sms && pairs >= 2 * slots;
}

template <typename T, int D, int NT>
int launch_walk(const Walk& w, int64_t pairs, cudaStream_t st) {
    static std::atomic<uint64_t> done[2];
    if (!w.runs && w.group == 1) {
        row_kernel<T, D><<<(unsigned)((pairs + ROW_WARPS - 1) / ROW_WARPS), ROW_WARPS * 32, 0, st>>>(w, pairs);
        return abi::cuda_check("attention launch");
    }
    if (!w.runs) {
        constexpr int ring = PAIR_STAGES * 2 * KEYS * D * 2, rows = 8 * NT * (D + 4) * 4, smem = ring > rows ? ring : rows;
        const cudaError_t e = allow_smem((const void*)pair_kernel<T, D, NT>, smem, done[0]);
        if (e != cudaSuccess) return abi::cuda_fail(e, "cudaFuncSetAttribute(attention)");
        pair_kernel<T, D, NT><<<(unsigned)pairs, 32, smem, st>>>(w);
        return abi::cuda_check("attention launch");
    }
    constexpr int ring = WARPS * STAGES * 2 * KEYS * D * 2, joined = WARPS * 8 * NT * (D + 4) * 4;
    constexpr int smem = ring > joined ? ring : joined;
    const cudaError_t e = allow_smem((const void*)walk_kernel<T, D, NT>, smem, done[1]);
    if (e != cudaSuccess) return abi::cuda_fail(e, "cudaFuncSetAttribute(attention)");
    walk_kernel<T, D, NT><<<(unsigned)w.runs, WARPS * 32, smem, st>>>(w);
    return abi::cuda_check("attention launch");
}

template <typename T, int D>
int launch_decode(const Walk& w, int64_t pairs, const Shares& shares, cudaStream_t st) {
    const int rc = w.tile_heads > 8 ? launch_walk<T, D, 2>(w, pairs, st) : launch_walk<T, D, 1>(w, pairs, st);
    if (rc) return rc;
    const int cuts = w.runs > 1 ? w.runs - 1 : 0;
    cudaError_t e = cudaSuccess;
    if (shares.weights)
        e = launch_after(finish_kernel<T, D>, dim3((unsigned)(shares.ctas + (int64_t)cuts * w.tile_heads)), dim3(JOIN_THREADS), 0,
                         st, w, shares);
    else if (cuts)
        e = launch_after(join_kernel<T, D>, dim3((unsigned)cuts, (unsigned)w.tile_heads), dim3(JOIN_THREADS), 0, st, w);
    if (e != cudaSuccess) return abi::cuda_fail(e, "attention join launch");
    return abi::cuda_check("attention join launch");
}

struct Space {
    int runs;
    uint64_t out, ml, cuts, lse2, logits, total;   // byte offsets
};
inline int tiles_of(int group) { return (group + ROWS - 1) / ROWS; }
inline Space decode_space(const Cache& c, int d, int q_heads, bool weights) {
    Space s;
    const int64_t pairs = (int64_t)c.seqs * c.kv_heads * tiles_of(q_heads / c.kv_heads);
    s.runs = whole_pairs(c, q_heads / c.kv_heads, pairs) ? 0 : cta_per_sm(d) * abi::num_sms();
    // no more runs than there can be units
    const int64_t most = pairs * ((c.capacity() + UNIT - 1) / UNIT + 1);
    if (s.runs > most) s.runs = (int)most;
    const uint64_t rows = (uint64_t)c.seqs * q_heads;
    s.out = 0;
    s.ml = (uint64_t)s.runs * 2 * ROWS * d * 4;
    s.cuts = s.ml + (uint64_t)s.runs * 2 * ROWS * 8;
    s.lse2 = s.cuts + (uint64_t)s.runs * 16;
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
    // rows go out and prior rows come in four elements at a time; what the workspace holds, 16 bytes
    if (reinterpret_cast<uintptr_t>(out) % 8 || reinterpret_cast<uintptr_t>(prior_out) % 8)
        return abi::fail(SWB_ERR_ARG, "out and the prior rows must start on 8-byte boundaries");
    if (sp.total && reinterpret_cast<uintptr_t>(workspace) % 16)
        return abi::fail(SWB_ERR_ARG, "the workspace must start on a 16-byte boundary");
    rc = earlier_wait();
    if (rc) return rc;
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
    w.cuts = reinterpret_cast<int4*>(ws + sp.cuts);
    if (weights_width == 0) weights = nullptr;      // of no slots: nothing to write
    w.lse2 = weights ? reinterpret_cast<float*>(ws + sp.lse2) : nullptr;
    w.logits = weights ? reinterpret_cast<float*>(ws + sp.logits) : nullptr;
    const int64_t pairs = (int64_t)c.seqs * c.kv_heads * w.head_tiles;
    const int64_t rows = (int64_t)c.seqs * q_heads;
    const int64_t chunks = (weights_width + SHARE_SLOTS - 1) / SHARE_SLOTS;
    const int64_t shares = weights ? chunks * c.seqs * c.kv_heads : 0;
    // units, output rows and cuts are counted in 32 bits
    if (pairs * ((c.capacity() + UNIT - 1) / UNIT + 1) >= ((int64_t)1 << 31) || rows >= ((int64_t)1 << 31) || shares >= ((int64_t)1 << 30))
        return abi::fail(SWB_ERR_ARG, "too many sequences in one call");
    Shares sh = {};
    sh.weights = weights;
    sh.width = weights_width;
    sh.accumulate = accumulate;
    sh.chunks = (int)chunks;
    sh.ctas = shares;
    if (cache->dtype == SWB_F16)
        return d == 64 ? launch_decode<__half, 64>(w, pairs, sh, st) : launch_decode<__half, 128>(w, pairs, sh, st);
    return d == 64 ? launch_decode<__nv_bfloat16, 64>(w, pairs, sh, st)
                   : launch_decode<__nv_bfloat16, 128>(w, pairs, sh, st);
}
