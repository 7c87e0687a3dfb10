// kvcache.cu -- what writes and trims a paged key-value cache.
//
// swb_rope_append: a new token's query and key heads normed (x / sqrt(mean x^2 +
// eps) * w) and rotated by its position, keys and values written to their slot.
// One pass: every element is read once and written once, in 32 bits between, so
// the kernel is bound by those bytes (and, for a few tokens, by its launch).  A
// 16-byte chunk of a head is a lane's; the lanes of a head sum its squares by
// shuffles, and a lane gets its rotation partner's chunk from the lane that holds
// it.
//
// swb_kv_evict: per key head, the `budget` slots with the largest accumulated
// weight stay (first and newest positions before all), and rows that lie beyond
// the budget move to the places that became free below it.  A slot's key is its
// weight's bits in an order that compares as the numbers do; four counting passes
// over 8 bits each find the budget-th largest key, and one pass in slot order
// splits the slots into those that stay, the free and the ones to move.  Counts
// and order are whole numbers: the result does not depend on timing.

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

constexpr int APPEND_THREADS = 256;

template <typename T, int D>
__global__ void __launch_bounds__(APPEND_THREADS) append_kernel(const __grid_constant__ Append P) {
    constexpr int LPH = D / 8;
    const int heads = P.q_heads + 2 * P.c.kv_heads;
    const int64_t at = (int64_t)blockIdx.x * APPEND_THREADS + threadIdx.x;
    const int64_t item = at / LPH;
    const int c = (int)(at % LPH);
    const int64_t tok = item / heads;
    const int h = (int)(item % heads);
    const bool live = tok < P.tokens;      // whole heads: the shuffles below stay inside one

    // the token's sequence: the last one that starts at or before it
    int b = 0;
    if (live) {
        int hi = P.c.seqs;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (P.starts[mid] <= tok) b = mid;
            else hi = mid;
        }
    }
    const int64_t slot = live ? (int64_t)P.c.lengths[b] - (P.starts[b + 1] - tok) : -1;
    const int64_t pos = live ? (P.positions ? (int64_t)P.positions[tok] : slot) : 0;

    const bool is_q = h < P.q_heads, is_v = h >= P.q_heads + P.c.kv_heads;
    const int kh = is_v ? h - P.q_heads - P.c.kv_heads : h - P.q_heads;
    const T* src = is_q ? static_cast<const T*>(P.q) + tok * P.q_ts + h * P.q_hs
                 : is_v ? static_cast<const T*>(P.v) + tok * P.v_ts + kh * P.v_hs
                        : static_cast<const T*>(P.k) + tok * P.k_ts + kh * P.k_hs;
    uint4 raw = live ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
    float x[8];
    {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Elem<T>::wide(w[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
    const void* weight = is_v ? nullptr : is_q ? P.q_weight : P.k_weight;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
    for (int s = LPH / 2; s > 0; s >>= 1) ss += __shfl_xor_sync(FULL, ss, s);
    if (weight) {
        const float inv = rsqrtf(ss * (1.f / D) + P.eps);
        const uint4 wr = *reinterpret_cast<const uint4*>(static_cast<const T*>(weight) + c * 8);
        const uint32_t w[4] = {wr.x, wr.y, wr.z, wr.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = Elem<T>::wide(w[i]);
            x[2 * i] *= inv * f.x;
            x[2 * i + 1] *= inv * f.y;
        }
    }
    const bool turned = !is_v && c * 8 < 2 * P.half;
    const bool known = pos >= 0 && pos < P.table_rows;     // a position outside the tables gives NaN
    const float NaN = __int_as_float(0x7fffffff);
    if (P.interleaved) {
        if (turned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float co = known ? P.cos[pos * P.half + c * 4 + i] : NaN;
                const float si = known ? P.sin[pos * P.half + c * 4 + i] : NaN;
                const float a = x[2 * i], e = x[2 * i + 1];
                x[2 * i] = a * co - e * si;
                x[2 * i + 1] = e * co + a * si;
            }
        }
    } else {
        const int hc = P.half / 8;
        const bool lower = c < hc;
        const int partner = turned ? (lower ? c + hc : c - hc) : c;
        const int base = (threadIdx.x & 31) / LPH * LPH;
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __shfl_sync(FULL, x[i], base + partner);
        if (turned) {
            const int64_t row = pos * P.half + (lower ? c : c - hc) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float co = known ? P.cos[row + i] : NaN;
                const float si = known ? P.sin[row + i] : NaN;
                x[i] = lower ? x[i] * co - y[i] * si : x[i] * co + y[i] * si;
            }
        }
    }
    if (!live) return;
    if (weight || turned)
        raw = make_uint4(Elem<T>::pack(x[0], x[1]), Elem<T>::pack(x[2], x[3]), Elem<T>::pack(x[4], x[5]),
                         Elem<T>::pack(x[6], x[7]));
    if (is_q) {
        *reinterpret_cast<uint4*>(static_cast<T*>(P.out) + (tok * P.q_heads + h) * D + c * 8) = raw;
        return;
    }
    if (slot < 0 || slot >= P.c.capacity()) return;
    const int64_t row = P.c.row(b, (int)slot);
    if (row < 0) return;
    T* pool = static_cast<T*>(const_cast<void*>(is_v ? P.c.v : P.c.k));
    *reinterpret_cast<uint4*>(pool + row + kh * P.c.head_stride + c * 8) = raw;
    if (P.slot_positions && !is_v && c == 0 && slot < P.width)
        P.slot_positions[((int64_t)b * P.c.kv_heads + kh) * P.width + slot] = (int32_t)pos;
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
};

constexpr int SELECT_THREADS = 512;

// a slot's key: larger stays.  First and newest positions above every weight,
// then the weights as numbers, NaN below all of them.
__device__ __forceinline__ uint32_t keep_key(float w, int pos, int sinks, int64_t fresh) {
    if ((pos >= 0 && pos < sinks) || pos >= fresh) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.f);     // -0 as 0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive sum of a 0/1 flag over the block, and the total
__device__ __forceinline__ int block_rank(bool flag, int* s_warp, int& total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned m = __ballot_sync(FULL, flag);
    if (lane == 0) s_warp[warp] = __popc(m);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < SELECT_THREADS / 32; ++w) {
        before += w < warp ? s_warp[w] : 0;
        all += s_warp[w];
    }
    __syncthreads();
    total = all;
    return before + __popc(m & lanemask_lt());
}

__global__ void __launch_bounds__(SELECT_THREADS) select_kernel(const __grid_constant__ Evict P) {
    __shared__ int s_hist[256], s_warp[SELECT_THREADS / 32], s_pick[2];
    const int64_t head = blockIdx.x;                       // sequence * kv_heads + key head
    const int b = (int)(head / P.c.kv_heads);
    const int n = (int)max((int64_t)0, min((int64_t)P.c.lengths[b], min(P.c.capacity(), P.width)));
    const int m = P.budget;
    const float* w = P.weights + head * P.width;
    const int32_t* pos = P.positions + head * P.width;
    float* nw = P.new_weights + head * P.width;
    int32_t* np = P.new_positions + head * P.width;
    const int64_t fresh = (int64_t)P.seen[b] - P.recent;
    if (threadIdx.x == 0 && head % P.c.kv_heads == 0) P.new_lengths[b] = min(n, m);
    for (int64_t j = min(n, m) + threadIdx.x; j < P.width; j += SELECT_THREADS) {
        nw[j] = 0.f;
        np[j] = -1;
    }
    if (n <= m) {
        for (int j = threadIdx.x; j < n; j += SELECT_THREADS) {
            nw[j] = w[j];
            np[j] = pos[j];
        }
        if (threadIdx.x == 0) P.counts[head] = 0;
        return;
    }
    // the m-th largest key, 8 bits at a time from the top; `need` of the keys
    // that share the bits found so far are among the m largest
    uint32_t prefix = 0, mask = 0;
    int need = m;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += SELECT_THREADS) s_hist[i] = 0;
        __syncthreads();
        for (int j = threadIdx.x; j < n; j += SELECT_THREADS) {
            const uint32_t key = keep_key(w[j], pos[j], P.sinks, fresh);
            if ((key & mask) == prefix) atomicAdd(&s_hist[(key >> shift) & 255], 1);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int left = need, bin = 255;
            while (bin > 0 && s_hist[bin] < left) left -= s_hist[bin--];
            s_pick[0] = bin;
            s_pick[1] = left;
        }
        __syncthreads();
        prefix |= (uint32_t)s_pick[0] << shift;
        mask |= 255u << shift;
        need = s_pick[1];
        __syncthreads();
    }
    // in slot order: equal keys to the lowest slots, free places and rows to move
    int ties = 0, free = 0, late = 0;
    int32_t* from = P.moves + head * 2 * m;
    int32_t* to = from + m;
    for (int j0 = 0; j0 < n; j0 += SELECT_THREADS) {
        const int j = j0 + threadIdx.x;
        float wj = 0.f;
        int pj = 0;
        uint32_t key = 0;
        if (j < n) {
            wj = w[j];
            pj = pos[j];
            key = keep_key(wj, pj, P.sinks, fresh);
        }
        int total;
        const bool tie = j < n && key == prefix;
        const int tr = block_rank(tie, s_warp, total) + ties;
        ties += total;
        const bool keep = j < n && (key > prefix || (tie && tr < need));
        if (keep && j < m) {
            nw[j] = wj;
            np[j] = pj;
        }
        const int fr = block_rank(j < m && !keep, s_warp, total) + free;
        free += total;
        if (j < m && !keep) to[fr] = j;
        const int lr = block_rank(j >= m && keep, s_warp, total) + late;
        late += total;
        if (j >= m && keep) from[lr] = j;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < late; i += SELECT_THREADS) {
        nw[to[i]] = w[from[i]];
        np[to[i]] = pos[from[i]];
    }
    if (threadIdx.x == 0) P.counts[head] = late;
}

constexpr int MOVE_THREADS = 256;
constexpr int MOVE_ROWS = 32;      // rows of a block

__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(const __grid_constant__ Evict P) {
    dependency_wait();
    const int64_t head = blockIdx.x;
    const int b = (int)(head / P.c.kv_heads), g = (int)(head % P.c.kv_heads);
    const int n = P.counts[head];
    const int32_t* from = P.moves + head * 2 * P.budget;
    const int32_t* to = from + P.budget;
    const int i0 = blockIdx.y * MOVE_ROWS, i1 = min(n, i0 + MOVE_ROWS);
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
    const int64_t lanes = a.tokens * (a.q_heads + 2 * a.c.kv_heads) * (D / 8);
    const int64_t blocks = (lanes + APPEND_THREADS - 1) / APPEND_THREADS;
    if (blocks >= ((int64_t)1 << 31)) return abi::fail(SWB_ERR_ARG, "too many tokens in one call");
    append_kernel<T, D><<<(unsigned)blocks, APPEND_THREADS, 0, st>>>(a);
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
    const int rc = check_cache(cache, &a.c);
    if (rc) return rc;
    if (tokens <= 0 || a.c.seqs == 0) return SWB_OK;
    if (!q || !k || !v || !starts || !out) return abi::fail(SWB_ERR_ARG, "null buffer");
    if (q_heads < 1 || q_heads % a.c.kv_heads)
        return abi::fail(SWB_ERR_ARG, "query heads must be a multiple of the cache's key heads");
    if (rot_dim < 0 || rot_dim % 16 || rot_dim > cache->head_dim)
        return abi::fail(SWB_ERR_ARG, "the rotated dimensions must be a multiple of 16, at most head_dim");
    if (rot_dim && (!cos || !sin)) return abi::fail(SWB_ERR_ARG, "null rotation tables");
    const void* at[6] = {q, k, v, out, q_weight, k_weight};
    const int64_t strides[6] = {q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride, v_head_stride};
    for (int i = 0; i < 6; ++i)
        if (reinterpret_cast<uintptr_t>(at[i]) % 16 || strides[i] % 8)
            return abi::fail(SWB_ERR_ARG, "rows must start on 16-byte boundaries");
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
    const int rc = check_cache(cache, &e.c);
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
    select_kernel<<<(unsigned)heads, SELECT_THREADS, 0, st>>>(e);
    const int rc2 = abi::cuda_check("evict launch");
    if (rc2) return rc2;
    // at most min(budget, slots beyond it) rows of a head move
    const int64_t beyond = e.c.capacity() - budget;
    const int64_t most = beyond < budget ? beyond : budget;
    if (most <= 0) return SWB_OK;
    const int64_t by = (most + MOVE_ROWS - 1) / MOVE_ROWS;
    if (by > 65535) return abi::fail(SWB_ERR_ARG, "budget too large");
    const cudaError_t err = launch_after(move_kernel, dim3((unsigned)heads, (unsigned)by), dim3(MOVE_THREADS), 0, st, e);
    if (err != cudaSuccess) return abi::cuda_fail(err, "evict move launch");
    return abi::cuda_check("evict move launch");
}
