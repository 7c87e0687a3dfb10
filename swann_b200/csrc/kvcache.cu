// kvcache.cu -- what writes and trims a paged key-value cache.
//
// swb_rope_append: a new token's query and key heads normed (x / sqrt(mean x^2 +
// eps) * w) and rotated by its position, keys and values written to their slot.
// One pass: every element is read once and written once, in 32 bits between, so
// the kernel is bound by those bytes (and, for a few tokens, by its launch).  A
// lane has two 16-byte chunks of a head, rotation partners; the lanes of a head
// sum its squares by shuffles.  9721 tokens of 48 heads of 128: 54 us, 4.5 TB/s.
//
// swb_kv_evict: per key head, the `budget` slots with the largest accumulated
// weight stay (first and newest positions before all), and rows that lie beyond
// the budget move to the places that became free below it.  A slot's key is its
// weight's bits in an order that compares as the numbers do; three counting passes
// (11, 11 and 10 bits) find the budget-th largest key, and a pass in slot order
// splits the slots into those that stay, the free and the ones to move.  Counts
// and order are whole numbers: the result does not depend on timing.  A CTA a key
// head; each of its warps has a contiguous piece of the slots, so ranks need
// ballots and one sum over warps.  The moved rows' bytes bound it when many move;
// one row moves in a step of one token, and then it is the chain of passes.  8
// sequences of up to 16384 slots cut to 2048, 8 heads: 37 us (23 to select, the rows
// 13); 8 heads of 4097 slots cut to 4096: 14 us.

#include "attn.cuh"

namespace swb {
namespace attn {

// -- norms, rotation, append ------------------------------------------------------

struct Append {
    Cache c;
    const void* q;
    const void* k;
    const void* v;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;   // token and head strides, elements
    const int32_t* starts;
    int64_t tokens;
    int q_heads;
    const void* q_weight;
    const void* k_weight;
    float eps;
    const float* cos;
    const float* sin;
    int64_t table_rows;
    int half;                    // rotated dimensions / 2
    int interleaved;
    const int32_t* positions;    // [tokens]; null: a token's slot
    void* out;                   // [tokens, q_heads, D]
    int32_t* slot_positions;     // [seqs][kv_heads][width]; null: not kept
    int64_t width;
};

constexpr int APPEND_THREADS = 128;
constexpr int APPEND_HEADS = 3;      // heads of a thread, their loads in flight together
constexpr int APPEND_CTAS = 7;       // an SM: 54 us at 72 registers, 59 at 5 CTAs, 67 unbounded

template <typename T>
__device__ __forceinline__ void wide8(const uint4& r, float (&x)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = Elem<T>::wide(w[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
    }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
    return make_uint4(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]), Elem<T>::pack(x[4], x[5]),
                      Elem<T>::pack(x[6], x[7]));
}

// A CTA a token, so that its place and its angles are read once.  A thread has the
// same two 16-byte chunks of each of its heads: of the dimensions that are rotated
// by halves those that are turned into one another, so nothing is exchanged but the
// sum of squares.  (A chunk a thread, the partner's by shuffles: 75 us for 9721
// tokens of 48 heads of 128.)
template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS, APPEND_CTAS) append_kernel(const __grid_constant__ Append P) {
    constexpr int LPH = D / 16, HP = APPEND_THREADS / LPH, U = APPEND_HEADS;
    const int heads = P.q_heads + 2 * P.c.kv_heads, keys = P.q_heads, values = P.q_heads + P.c.kv_heads;
    const int64_t tok = blockIdx.x;
    const int idx = threadIdx.x % LPH, hc = P.half / 8;
    // chunks idx and idx + hc are rotated into one another; the others go two by two
    const bool halves = idx < hc && !P.interleaved;
    const int c0 = halves ? idx : 2 * idx, c1 = halves ? idx + hc : 2 * idx + 1;
    const bool turned = idx < hc;

    int b = 0, slot = 0, pos = 0;
    int64_t row = 0;
    float co[8], si[8];
    for (int hb = threadIdx.x / LPH; hb - (int)threadIdx.x / LPH < heads; hb += HP * U) {
        uint4 raw[U][2];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = hb + i * HP;
            const T* src = h < keys ? static_cast<const T*>(P.q) + tok * P.q_ts + h * P.q_hs
                         : h < values ? static_cast<const T*>(P.k) + tok * P.k_ts + (h - keys) * P.k_hs
                                      : static_cast<const T*>(P.v) + tok * P.v_ts + (h - values) * P.v_hs;
            raw[i][0] = raw[i][1] = make_uint4(0u, 0u, 0u, 0u);
            if (h < heads) {
                raw[i][0] = *reinterpret_cast<const uint4*>(src + c0 * 8);
                raw[i][1] = *reinterpret_cast<const uint4*>(src + c1 * 8);
            }
        }
        if (hb < HP) {
            // the token's sequence: the last one that starts at or before it, if it has not ended
            // there; a token of none has no slot
            int hi = P.c.seqs;
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (P.starts[mid] <= tok) b = mid;
                else hi = mid;
            }
            slot = -1;
            bool ours = false;
            if (P.c.seqs > 0) {
                const int to = P.starts[b + 1];
                ours = P.starts[b] <= tok && tok < to;
                if (ours) slot = max(P.c.lengths[b], 0) - (to - (int)tok);
            }
            pos = P.positions ? P.positions[tok] : slot;
            row = slot >= 0 && slot < P.c.capacity() ? P.c.row(b, slot) : -1;
            if (turned) {
                if (pos >= 0 && pos < P.table_rows) {
                    const float4* pc = reinterpret_cast<const float4*>(P.cos + (int64_t)pos * P.half + idx * 8);
                    const float4* ps = reinterpret_cast<const float4*>(P.sin + (int64_t)pos * P.half + idx * 8);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        *reinterpret_cast<float4*>(co + 4 * e) = pc[e];
                        *reinterpret_cast<float4*>(si + 4 * e) = ps[e];
                    }
                } else {                                    // a position outside the tables gives NaN, none no turn
                    const bool none = !ours && !P.positions;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        co[e] = none ? 1.f : __int_as_float(0x7fffffff);
                        si[e] = none ? 0.f : __int_as_float(0x7fffffff);
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int h = hb + i * HP;
            const bool is_q = h < keys, is_v = h >= values;
            const T* weight = static_cast<const T*>(is_v ? nullptr : is_q ? P.q_weight : P.k_weight);
            const bool turn = turned && !is_v;
            float x[8], y[8];
            wide8<T>(raw[i][0], x);
            wide8<T>(raw[i][1], y);
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e] + y[e] * y[e];
#pragma unroll
            for (int s = LPH / 2; s > 0; s >>= 1) ss += __shfl_xor_sync(FULL, ss, s);
            if (weight) {
                const float inv = rsqrtf(ss * (1.f / D) + P.eps);
                float w0[8], w1[8];
                wide8<T>(*reinterpret_cast<const uint4*>(weight + c0 * 8), w0);
                wide8<T>(*reinterpret_cast<const uint4*>(weight + c1 * 8), w1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] *= inv * w0[e];
                    y[e] *= inv * w1[e];
                }
            }
            if (turn) {
                if (P.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float a0 = x[2 * e], b0 = x[2 * e + 1], a1 = y[2 * e], b1 = y[2 * e + 1];
                        x[2 * e] = a0 * co[e] - b0 * si[e];
                        x[2 * e + 1] = b0 * co[e] + a0 * si[e];
                        y[2 * e] = a1 * co[e + 4] - b1 * si[e + 4];
                        y[2 * e + 1] = b1 * co[e + 4] + a1 * si[e + 4];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float a0 = x[e], b0 = y[e];
                        x[e] = a0 * co[e] - b0 * si[e];
                        y[e] = b0 * co[e] + a0 * si[e];
                    }
                }
            }
            if (h >= heads) continue;
            if (weight || turn) {
                raw[i][0] = pack8<T>(x);
                raw[i][1] = pack8<T>(y);
            }
            T* dst;
            if (is_q) {
                dst = static_cast<T*>(P.out) + (tok * P.q_heads + h) * D;
            } else {
                if (row < 0) continue;
                const int kh = is_v ? h - values : h - keys;
                dst = static_cast<T*>(const_cast<void*>(is_v ? P.c.v : P.c.k)) + row + kh * P.c.head_stride;
                if (P.slot_positions && !is_v && idx == 0 && slot < P.width)
                    P.slot_positions[((int64_t)b * P.c.kv_heads + kh) * P.width + slot] = pos;
            }
            *reinterpret_cast<uint4*>(dst + c0 * 8) = raw[i][0];
            *reinterpret_cast<uint4*>(dst + c1 * 8) = raw[i][1];
        }
    }
}

// -- eviction -----------------------------------------------------------------

struct Evict {
    Cache c;
    int budget, sinks, recent;
    const int32_t* seen;          // [seqs] positions given out so far
    const float* weights;         // [seqs][kv_heads][width]
    const int32_t* positions;
    int64_t width;
    int32_t* new_lengths;
    float* new_weights;
    int32_t* new_positions;
    int32_t* moves;               // [seqs * kv_heads][2][budget]: from, to
    int32_t* counts;              // [seqs * kv_heads]
    int row_chunks;               // 16-byte chunks of a row

    // slots of sequence b that there are: of the table and of a row of weights
    __device__ __forceinline__ int held(int b) const {
        return (int)max((int64_t)0, min((int64_t)c.lengths[b], min(c.capacity(), width)));
    }
};

constexpr int SELECT_THREADS = 1024;
constexpr int SELECT_WARPS = SELECT_THREADS / 32;
constexpr int BINS = 2048;
constexpr int COPIES = 8;        // of the bins: weights share exponents, so neighbouring lanes would meet in one
constexpr int COPY = BINS + 4;   // counts from a copy to the next: the same bin of each lies in banks of its own

// a slot's key: larger stays.  First and newest positions above every weight,
// then the weights as numbers, NaN below all of them.
__device__ __forceinline__ uint32_t keep_key(float w, int pos, int sinks, int64_t fresh) {
    if ((pos >= 0 && pos < sinks) || pos >= fresh) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);     // -0 as 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// sum of x over the warps before this one (x the same in a warp's lanes), and
// over all; called by the whole CTA
__device__ __forceinline__ int warps_before(int x, int* s_warp, int& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) s_warp[warp] = x;
    __syncthreads();
    const int y = s_warp[lane];
    int sum = y;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const int z = __shfl_up_sync(FULL, sum, s);
        if (lane >= s) sum += z;
    }
    total = __shfl_sync(FULL, sum, 31);
    return __shfl_sync(FULL, sum - y, warp);
}
static_assert(SELECT_WARPS == 32, "one lane a warp");

// KEEP: 32-slot steps of a warp whose keys stay in registers; beyond that they are
// read again in each pass
template <int KEEP>
__global__ void __launch_bounds__(SELECT_THREADS) select_kernel(const __grid_constant__ Evict P) {
    extern __shared__ int4 s_bins[];                       // [COPIES][COPY] counts
    int* s_hist = reinterpret_cast<int*>(s_bins);
    __shared__ int s_warp[SELECT_WARPS], s_pick[2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t head = blockIdx.x;                       // sequence * kv_heads + key head
    const int b = (int)(head / P.c.kv_heads);
    const int n = P.held(b);
    const int m = P.budget;
    const float* w = P.weights + head * P.width;
    const int32_t* pos = P.positions + head * P.width;
    float* nw = P.new_weights + head * P.width;
    int32_t* np = P.new_positions + head * P.width;
    const int64_t fresh = (int64_t)P.seen[b] - P.recent;
    if (threadIdx.x == 0 && head % P.c.kv_heads == 0) P.new_lengths[b] = min(n, m);
    if (n <= m) {
        for (int j = threadIdx.x; j < n; j += SELECT_THREADS) {
            nw[j] = w[j];
            np[j] = pos[j];
        }
        if (threadIdx.x == 0) P.counts[head] = 0;
        return;
    }
    // this warp's slots: 32 at a time from j0 on
    const int steps = (n + SELECT_THREADS - 1) / SELECT_THREADS, j0 = warp * steps * 32 + lane;
    const int mine = max(0, min(steps, (n - j0 + 31) / 32));      // of this lane
    auto key_at = [&](int i) -> uint32_t { return keep_key(w[j0 + i * 32], pos[j0 + i * 32], P.sinks, fresh); };
    uint32_t held[KEEP];
    constexpr int BATCH = KEEP < 8 ? KEEP : 8;             // slots whose loads are in flight together
#pragma unroll
    for (int i0 = 0; i0 < KEEP; i0 += BATCH) {
        float wv[BATCH];
        int pv[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const bool in = i0 + i < mine;
            wv[i] = in ? w[j0 + (i0 + i) * 32] : 0.f;
            pv[i] = in ? pos[j0 + (i0 + i) * 32] : -1;
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) held[i0 + i] = keep_key(wv[i], pv[i], P.sinks, fresh);
    }
    // f(slot, key) for this lane's slots; every lane takes part in every step, with
    // whether it has a slot there
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
            if (i < steps) f(j0 + i * 32, held[i], i < mine);
        for (int i = KEEP; i < steps; ++i) f(j0 + i * 32, i < mine ? key_at(i) : 0u, i < mine);
    };

    // the m-th largest key, some bits at a time from the top; `need` of the keys
    // that share the bits found so far are among the m largest
    uint32_t prefix = 0, mask = 0;
    int need = m;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digit = pass == 2 ? 1023u : 2047u;
        for (int i = threadIdx.x; i < COPY * COPIES / 4; i += SELECT_THREADS) s_bins[i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        each([&](int, uint32_t key, bool there) {
            if (there && (key & mask) == prefix) atomicAdd(&s_hist[(lane & (COPIES - 1)) * COPY + ((key >> shift) & digit)], 1);
        });
        __syncthreads();
        // bins from the largest down, two a thread: the one that holds the need-th
        int count[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < COPIES; ++k) {
            const int2 x = *reinterpret_cast<const int2*>(s_hist + k * COPY + BINS - 2 - 2 * threadIdx.x);
            count[0] += x.y;
            count[1] += x.x;
        }
        int sum = count[0] + count[1];
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int z = __shfl_up_sync(FULL, sum, s);
            if (lane >= s) sum += z;
        }
        int total;
        const int before = warps_before(__shfl_sync(FULL, sum, 31), s_warp, total) + sum - count[0] - count[1];
        if (before < need && need <= before + count[0] + count[1]) {
            const bool top = need <= before + count[0];
            s_pick[0] = BINS - 1 - 2 * threadIdx.x - (top ? 0 : 1);
            s_pick[1] = need - before - (top ? 0 : count[0]);
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        mask |= digit << shift;
        need = s_pick[1];
    }

    // equal keys stay in the lowest slots: up to the slot of the need-th of them
    int total, ties = 0;
    each([&](int, uint32_t key, bool there) { ties += there && key == prefix; });
    const int before = warps_before((int)__reduce_add_sync(FULL, ties), s_warp, total);
    if (threadIdx.x == 0) s_pick[0] = 0x7fffffff;
    __syncthreads();
    if (total > need) {
        int seen = before;
        each([&](int j, uint32_t key, bool there) {
            const unsigned t = __ballot_sync(FULL, there && key == prefix);
            if (there && key == prefix && seen + __popc(t & lanemask_lt()) == need - 1) s_pick[0] = j;
            seen += __popc(t);
        });
    }
    __syncthreads();
    const int last = s_pick[0];
    auto keeps = [&](int j, uint32_t key, bool there) { return there && (key > prefix || (key == prefix && j <= last)); };
    // ranks of the free places and of the rows to move, in slot order
    int free = 0, late = 0, moved;
    each([&](int j, uint32_t key, bool there) {
        const bool keep = keeps(j, key, there);
        free += there && j < m && !keep;
        late += j >= m && keep;
    });
    free = warps_before((int)__reduce_add_sync(FULL, free), s_warp, total);
    late = warps_before((int)__reduce_add_sync(FULL, late), s_warp, moved);
    int32_t* from = P.moves + head * 2 * m;
    int32_t* to = from + m;
    each([&](int j, uint32_t key, bool there) {
        const bool keep = keeps(j, key, there);
        const unsigned f = __ballot_sync(FULL, there && j < m && !keep), l = __ballot_sync(FULL, j >= m && keep);
        if (there && j < m && !keep) to[free + __popc(f & lanemask_lt())] = j;
        if (j >= m && keep) from[late + __popc(l & lanemask_lt())] = j;
        free += __popc(f);
        late += __popc(l);
    });
    // what stays in place, by all threads side by side
    for (int j = threadIdx.x; j < m; j += SELECT_THREADS) {
        const float wj = w[j];
        const int pj = pos[j];
        if (keeps(j, keep_key(wj, pj, P.sinks, fresh), true)) {
            nw[j] = wj;
            np[j] = pj;
        }
    }
    if (threadIdx.x == 0) P.counts[head] = moved;
}

constexpr int MOVE_THREADS = 256;
constexpr int MOVE_ROWS = 32;      // rows of a CTA
constexpr int MOVE_SLOTS = 4096;   // slots beyond the budget of a CTA

// the rows that move, with their weights and positions, and the slots that now hold nothing
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(const __grid_constant__ Evict P) {
    const int64_t head = blockIdx.x;
    const int b = (int)(head / P.c.kv_heads), g = (int)(head % P.c.kv_heads);
    const float* w = P.weights + head * P.width;
    const int32_t* pos = P.positions + head * P.width;
    float* nw = P.new_weights + head * P.width;
    int32_t* np = P.new_positions + head * P.width;
    {
        const int64_t j0 = min(P.held(b), P.budget) + (int64_t)blockIdx.y * MOVE_SLOTS, j1 = min(P.width, j0 + MOVE_SLOTS);
        for (int64_t j = j0 + threadIdx.x; j < j1; j += MOVE_THREADS) {
            nw[j] = 0.f;
            np[j] = -1;
        }
    }
    dependency_wait();
    const int n = P.counts[head];
    const int32_t* from = P.moves + head * 2 * P.budget;
    const int32_t* to = from + P.budget;
    const int i0 = blockIdx.y * MOVE_ROWS, i1 = min(n, i0 + MOVE_ROWS);
    if (i0 + (int)threadIdx.x < i1) {
        const int a = from[i0 + threadIdx.x], z = to[i0 + threadIdx.x];
        nw[z] = w[a];
        np[z] = pos[a];
    }
    for (int x = threadIdx.x; x < (i1 - i0) * P.row_chunks; x += MOVE_THREADS) {
        const int i = i0 + x / P.row_chunks, c = x % P.row_chunks;
        const int64_t a = P.c.row(b, from[i]), z = P.c.row(b, to[i]);
        if (a < 0 || z < 0) continue;
        const int64_t h = (int64_t)g * P.c.head_stride + c * 8;
        const uint16_t* k = static_cast<const uint16_t*>(P.c.k);
        const uint16_t* v = static_cast<const uint16_t*>(P.c.v);
        const uint4 kr = *reinterpret_cast<const uint4*>(k + a + h), vr = *reinterpret_cast<const uint4*>(v + a + h);
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(k) + z + h) = kr;
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(v) + z + h) = vr;
    }
}

}  // namespace attn
}  // namespace swb

using namespace swb;
using namespace swb::attn;

template <typename T, int D>
static int launch_append(const Append& a, cudaStream_t st) {
    if (a.tokens >= ((int64_t)1 << 31)) return abi::fail(SWB_ERR_ARG, "too many tokens in one call");
    append_kernel<T, D><<<(unsigned)a.tokens, APPEND_THREADS, 0, st>>>(a);
    return abi::cuda_check("append launch");
}

extern "C" int swb_rope_append(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                               int64_t v_head_stride, int q_heads, const int32_t* starts, int64_t tokens,
                               const void* q_weight, const void* k_weight, float eps, const float* cos,
                               const float* sin, int64_t table_rows, int rot_dim, int interleaved,
                               const int32_t* positions, const swb_kv_cache* cache, void* out,
                               int32_t* slot_positions, int64_t slot_width, void* stream) {
    Append a = {};
    int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if (tokens <= 0) return SWB_OK;
    if (!q || !k || !v || !starts || !out) return abi::fail(SWB_ERR_ARG, "null buffer");
    if (q_heads < 1 || q_heads % a.c.kv_heads)
        return abi::fail(SWB_ERR_ARG, "query heads must be a multiple of the cache's key heads");
    if (rot_dim < 0 || rot_dim % 16 || rot_dim > cache->head_dim)
        return abi::fail(SWB_ERR_ARG, "the rotated dimensions must be a multiple of 16, at most head_dim");
    if (rot_dim && (!cos || !sin)) return abi::fail(SWB_ERR_ARG, "null rotation tables");
    if (reinterpret_cast<uintptr_t>(cos) % 16 || reinterpret_cast<uintptr_t>(sin) % 16)
        return abi::fail(SWB_ERR_ARG, "the rotation tables must start on 16-byte boundaries");
    const void* at[6] = {q, k, v, out, q_weight, k_weight};
    const int64_t strides[6] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    for (int i = 0; i < 6; ++i)
        if (reinterpret_cast<uintptr_t>(at[i]) % 16 || strides[i] % 8)
            return abi::fail(SWB_ERR_ARG, "rows must start on 16-byte boundaries");
    rc = earlier_wait();
    if (rc) return rc;
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_ts = q_token_stride;
    a.q_hs = q_head_stride;
    a.k_ts = k_token_stride;
    a.k_hs = k_head_stride;
    a.v_ts = v_token_stride;
    a.v_hs = v_head_stride;
    a.starts = starts;
    a.tokens = tokens;
    a.q_heads = q_heads;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.cos = cos;
    a.sin = sin;
    a.table_rows = table_rows;
    a.half = rot_dim / 2;
    a.interleaved = interleaved;
    a.positions = positions;
    a.out = out;
    a.slot_positions = slot_positions;
    a.width = slot_width;
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dtype == SWB_F16)
        return cache->head_dim == 64 ? launch_append<__half, 64>(a, st) : launch_append<__half, 128>(a, st);
    return cache->head_dim == 64 ? launch_append<__nv_bfloat16, 64>(a, st) : launch_append<__nv_bfloat16, 128>(a, st);
}

extern "C" uint64_t swb_kv_evict_workspace(int seqs, int kv_heads, int budget) {
    if (seqs < 0 || kv_heads < 1 || budget < 1) return 0;
    return (uint64_t)seqs * kv_heads * (2 * (uint64_t)budget + 1) * 4;
}

extern "C" int swb_kv_evict(const swb_kv_cache* cache, const int32_t* seen, const float* weights,
                            const int32_t* positions, int64_t width, int budget, int sinks, int recent,
                            int32_t* new_lengths, float* new_weights, int32_t* new_positions, void* workspace,
                            uint64_t ws_bytes, void* stream) {
    Evict e = {};
    int rc = check_cache(cache, &e.c);
    if (rc) return rc;
    if (budget < 1 || sinks < 0 || recent < 0) return abi::fail(SWB_ERR_ARG, "budget, sinks or recent out of range");
    if ((int64_t)sinks + recent > budget) return abi::fail(SWB_ERR_ARG, "sinks and recent do not fit the budget");
    if (width < e.c.capacity()) return abi::fail(SWB_ERR_ARG, "weights are narrower than the page table's slots");
    if (e.c.seqs == 0) return SWB_OK;
    if (!seen || !weights || !positions || !new_lengths || !new_weights || !new_positions)
        return abi::fail(SWB_ERR_ARG, "null buffer");
    if (new_weights == weights || new_positions == positions || new_lengths == cache->lengths)
        return abi::fail(SWB_ERR_ARG, "the new weights, positions and lengths must be buffers of their own");
    if (!workspace || ws_bytes < swb_kv_evict_workspace(e.c.seqs, e.c.kv_heads, budget))
        return abi::fail(SWB_ERR_ARG, "workspace too small");
    const int64_t heads = (int64_t)e.c.seqs * e.c.kv_heads;
    if (heads >= ((int64_t)1 << 31)) return abi::fail(SWB_ERR_ARG, "too many sequences in one call");
    // at most min(budget, slots beyond it) rows of a head move, and slots beyond the
    // budget or the shortest length hold nothing
    const int64_t beyond = e.c.capacity() - budget;
    const int64_t most = beyond < budget ? (beyond > 0 ? beyond : 0) : budget;
    const int64_t rows = (most + MOVE_ROWS - 1) / MOVE_ROWS, slots = (width + MOVE_SLOTS - 1) / MOVE_SLOTS;
    const int64_t by = rows > slots ? rows : slots;
    if (by > 65535) return abi::fail(SWB_ERR_ARG, "budget or weights too wide");
    rc = earlier_wait();
    if (rc) return rc;
    e.budget = budget;
    e.sinks = sinks;
    e.recent = recent;
    e.seen = seen;
    e.weights = weights;
    e.positions = positions;
    e.width = width;
    e.new_lengths = new_lengths;
    e.new_weights = new_weights;
    e.new_positions = new_positions;
    e.moves = static_cast<int32_t*>(workspace);
    e.counts = e.moves + heads * 2 * budget;
    e.row_chunks = cache->head_dim / 8;
    cudaStream_t st = (cudaStream_t)stream;
    constexpr int smem = COPY * COPIES * 4;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    // up to 8192 slots half of the registers do: 8 heads of 4160 slots 15 us, 19 with room for
    // 16384; at 16384 slots they would be read again in each pass, 34 us against 26
    const bool few = e.c.capacity() <= 8 * SELECT_THREADS;
    const void* kernel = few ? (const void*)select_kernel<8> : (const void*)select_kernel<16>;
    static std::atomic<uint64_t> done[2];
    cudaError_t err = allow_smem(kernel, smem, done[few]);
    if (err != cudaSuccess) return abi::cuda_fail(err, "cudaFuncSetAttribute(evict)");
    if (few) select_kernel<8><<<(unsigned)heads, SELECT_THREADS, smem, st>>>(e);
    else select_kernel<16><<<(unsigned)heads, SELECT_THREADS, smem, st>>>(e);
    rc = abi::cuda_check("evict launch");
    if (rc) return rc;
    if (by == 0) return SWB_OK;
    err = launch_after(move_kernel, dim3((unsigned)heads, (unsigned)by), dim3(MOVE_THREADS), 0, st, e);
    if (err != cudaSuccess) return abi::cuda_fail(err, "evict move launch");
    return abi::cuda_check("evict move launch");
}
