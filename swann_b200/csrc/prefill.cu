// prefill.cu -- attention of many new tokens over a paged cache, on the
// 5th-generation tensor cores.
//
// The definition is attention.cu's, for tokens at the last slots of their
// sequences.  Two products a block of keys, 4 d flops a visible pair, decide the
// time; the exponentials come next (one a pair against 16 a cycle and SM), so the
// layout below keeps the tensor pipe on one tile while another's softmax runs.
//
// A CTA owns two tiles of 128 query rows that share a key head: row r of a tile is
// token r / heads, head r % heads, so the heads of a group read each key once.  It
// walks steps of 64 keys that any of its rows sees:
//   warps 9..11   producers: K and V into a ring of 128-byte swizzled tiles, a
//                 step's a warp.  Where all 64 rows are seen by some query and lie
//                 in pages of at least 8 rows, TMA brings them, a box a page; else
//                 cp.async, one row address a lane, rows that no page holds or no
//                 query sees filled with zeros, so what is in memory there reaches
//                 no product.  (cp.async alone kept the tensor pipe waiting: 332 us
//                 against 254 for 2049 tokens over 8193 slots, 32 heads of 128);
//   warp 8        issues tcgen05.mma: S = Q K^T (both K-major) into one of the
//                 tile's two buffers of 64 TMEM columns, O += P V with P read from
//                 TMEM and V as it lies (MN-major).  What it does besides is kept
//                 short (a wait a stage and a tile, a commit each): the tensor pipe's
//                 queue is a few products deep;
//   warps 0..3 and 4..7  softmax of tile 0 and 1: a thread is a row.  It writes the
//                 weights, rounded to the cache's 16 bits, over the logits' columns
//                 and keeps the row's sum in 32 bits, before that rounding.
// With two buffers the next step's logits are there when a softmax ends: with one
// of 128 keys, which TMEM has room for instead, each tile's softmax and products
// took turns, and neither pipe was busy for more than half of the time.
//
// The running maximum that the exponentials are taken against is only raised when
// a row's maximum has passed it by 2^8 (weights stay below 2^8 and sums in range);
// only then is O rescaled in TMEM, which the first blocks of a row need and later
// ones hardly ever do.  In fp16 the weights and their sum are 2^7 times that, up to
// 2^15 (no instruction more: the exponents' offset is another one), so that what a
// long flat tail has is not lost beside one strong key: a weight that vanishes is
// below 2^-32 of the one at the maximum in use.
//
// MMAs of one thread run in order, so the logits of step i + 1 may be issued right
// after the product that reads step i - 1's weights, which lie in the same columns.
// CTAs stay and take job after job, the longest first; queries, keys and logits of
// the next one are under way while the last rows of this one are written.  All waits
// are bounded; if one runs out the CTA's rows are NaN and the status word is set, once
// copies and products in flight are done (or have had milliseconds to).
//
// Measured: 2049 tokens over 8193 slots, 32 heads of 128 over 8: 239 us, 1007 TFLOP/s
// (60% of a cuBLAS bf16 product's rate).  A step of the two tiles takes about 1700
// cycles, 1320 of them in the tensor pipe: Q K^T with 64 keys a product is bound by
// reading Q from shared memory (50 cycles a product of 32 cycles' work), and a
// row's chain of wait, maximum, exponentials and hand-over is about as long.  8192
// tokens by window 1024: 170 us, where 18 steps a job leave its ends a third of the time.

#include <cuda.h>
#include <cudaTypedefs.h>

#include "attn.cuh"
#include "tcgen05.cuh"

namespace swb {
namespace attn {
namespace pre {

constexpr int TILE = 128;                   // rows of a query tile
constexpr int STEP = 64;                    // keys
constexpr int THREADS = 384;
constexpr int MMA_WARP = 8, PRODUCER0 = 9, PRODUCERS = 3;   // warps
constexpr int SOFTMAX = 4;                  // warps of a tile
constexpr int SEEN = 32;                    // steps whose rows are on record
constexpr int LAG = 2;                      // parts of a warp in flight behind the one being issued
constexpr int FOLD = 16;                    // steps whose weights are summed by themselves
constexpr float RAISE = 8.f;                // log2 of how far a maximum may pass the one in use

struct Prefill {
    Cache c;
    const void* q;
    int64_t q_token_stride, q_head_stride;
    const int32_t* starts;
    int64_t tokens;
    int q_heads, group, head_tiles, tile_heads, tile_tokens;
    float scale2;               // |scale| * log2(e), above 0
    int flip;                   // scale below 0: the queries' signs are turned instead
    int window, sinks;
    int tma;                    // the maps hold: rows of a box, 0 where there are none
    int items;                  // at most so many
    void* out;
    float* lse;
    int32_t* status;
};

template <int D>
struct Layout {
    static constexpr int QB = TILE * D * 2;                     // a query tile
    static constexpr int KB = STEP * D * 2;                     // a step's K or V
    static constexpr int STAGEB = 2 * KB;
    static constexpr int SLOTS = D == 128 ? 4 : 8;
    static constexpr int Q = 0;                                 // two tiles
    static constexpr int RING = 2 * QB;
    static constexpr int BARS = RING + SLOTS * STAGEB;          // full, empty, q, q let go, s[2][2], p[2][2], o[2][2], end
    static constexpr int SEENB = BARS + (2 * SLOTS + 15) * 8;   // uint32 [SEEN][2], on an 8-byte boundary
    static constexpr int OUT = (SEENB + SEEN * 2 * 4 + 15) / 16 * 16;   // a warp's 32 rows of 64 dimensions, on their way out
    static constexpr int TOTAL = OUT + 2 * SOFTMAX * 32 * 128;
};

// chunk c (16 bytes) of row r of a tile made of panels of 64 dimensions
template <int ROWS>
__device__ __forceinline__ uint32_t place(int r, int c) {
    return (uint32_t)((c >> 3) * (ROWS * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Operand descriptors: the high word is the same for all (version, 128-byte
// swizzle, 1024 bytes from 8 rows to the next), the low word is the address / 16 and,
// for V (which lies with its dimensions contiguous: 64 of them x 8 keys in 1024
// bytes), the bytes from a panel to the next / 16.
constexpr uint32_t DESC_HI = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_k(uint32_t a) { return (a >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_v(uint32_t a) { return (a >> 4) | ((uint32_t)(STEP * 128 / 16) << 16); }

// A stage of the ring holds what is multiplied next to each other: stage q has K of
// step q and V of step q - 2, one after the other.

template <typename T>
struct Format;
template <>
struct Format<__half> {
    static constexpr uint32_t F = 0;
};
template <>
struct Format<__nv_bfloat16> {
    static constexpr uint32_t F = 1;
};
template <typename T>
__host__ __device__ constexpr uint32_t instr(int n, bool b_mn_major) {
    return (1u << 4) | (Format<T>::F << 7) | (Format<T>::F << 10) | (uint32_t(b_mn_major) << 16) |
           (uint32_t(n >> 3) << 17) | (uint32_t(TILE >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 x, {%1, %4};\n\tmov.b64 y, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(DESC_HI), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(DESC_HI), "r"(acc)
        : "memory");
}
// one lane of a converged warp, in a form that the compiler knows to be one
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// 32 columns of this thread's TMEM lane; the values are there after tmem_arrived
__device__ __forceinline__ void tmem_get32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_arrived(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
// 16 columns, arrived
__device__ __forceinline__ void tmem_get16(uint32_t a, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_put16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(a)
        : "memory");
}
// rows of one page and head into a panel (box: 64 dimensions x some rows)
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page,
                                        uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tmem_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// one arrival for a warp, after all of its lanes
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// two fp32 values an instruction, each rounded on its own
__device__ __forceinline__ unsigned long long pair(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// mbar_wait with nothing on the way of a phase that is complete: the clock is only
// read after many tries
__device__ __forceinline__ bool await(uint64_t* bar, uint32_t parity, long long limit = 1ll << 32) {
    long long t0 = 0;
    for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
        if ((n & 255u) == 0) {
            const long long t = clock64();
            if (t0 == 0) t0 = t;
            else if (t - t0 > limit) return false;
        }
    }
    return true;
}

// the low x bits of a word
__device__ __forceinline__ uint32_t low_bits(int x) { return x >= 32 ? 0xffffffffu : x <= 0 ? 0u : (1u << x) - 1u; }

// What the CTA's roles agree on.  Keys have places u, steps of 64 of them: place
// u is slot base + u, base a multiple of 64 so that places keep the slots'
// alignment to pages.  With a window the first slot seen is lo and base lies at
// least as many places below it as there are first tokens to see: those take the
// places u < first, and the places between hold nothing.
struct Job {
    int b, g, head0, heads;
    int64_t token0;             // of the batch: first token of tile 0
    int pos0;                   // its slot
    int live;                   // tokens of the CTA that exist
    int first, lo, base, n, steps;
    __device__ __forceinline__ int slot(int u) const { return u < first ? u : base + u; }
    __device__ __forceinline__ bool holds(int u) const { return u < n && (u < first || base + u >= lo); }
};

// how far x lies past y, 0 if it does not; x and y differ by up to 2^32: a window may be
// any 32-bit number, and tokens lie before slot 0 where lengths do not count them all
__device__ __forceinline__ int past(int64_t x, int64_t y) { return (int)max((int64_t)0, x - y); }

// item `item` of all; false past the last
__device__ __forceinline__ bool find_job(const Prefill& P, int item, Job& J) {
    if (item >= P.items) return false;
    const int lane = threadIdx.x & 31;
    int left = item / P.head_tiles;
    const int ht = item - left * P.head_tiles;
    J.g = left % P.c.kv_heads;
    left /= P.c.kv_heads;
    const int step = 2 * P.tile_tokens;
    // the sequences' tiles end to end, 32 sequences at a time
    int b = -1, tiles = 0, s0 = 0, ntok = 0, length = 0;
    for (int b0 = 0; b0 < P.c.seqs; b0 += 32) {
        const int mine = b0 + lane;
        int t = 0, from = 0, n = 0, held = 0;
        if (mine < P.c.seqs) {
            from = (int)clamp_start(P.starts, mine, P.tokens);
            n = (int)clamp_start(P.starts, mine + 1, P.tokens) - from;
            held = max(0, P.c.lengths[mine]);
            t = n > 0 ? (n + step - 1) / step : 0;
        }
        int sum = t;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int y = __shfl_up_sync(FULL, sum, s);
            if (lane >= s) sum += y;
        }
        const unsigned hit = __ballot_sync(FULL, left < sum);
        if (hit) {
            const int src = __ffs(hit) - 1;
            b = b0 + src;
            tiles = __shfl_sync(FULL, t, src);
            left -= __shfl_sync(FULL, sum, src) - tiles;
            s0 = __shfl_sync(FULL, from, src);
            ntok = __shfl_sync(FULL, n, src);
            length = __shfl_sync(FULL, held, src);
            break;
        }
        left -= __shfl_sync(FULL, sum, 31);
    }
    if (b < 0) return false;
    const int tile = tiles - 1 - left;               // the longest rows first
    J.b = b;
    J.heads = min(P.tile_heads, P.group - ht * P.tile_heads);
    J.head0 = J.g * P.group + ht * P.tile_heads;
    J.token0 = s0 + tile * step;
    J.live = min(step, ntok - tile * step);
    J.pos0 = length - ntok + tile * step;
    const int end = (int)max((int64_t)0, min((int64_t)J.pos0 + J.live, P.c.capacity()));
    J.lo = P.window > 0 ? min(past((int64_t)J.pos0 + 1, P.window), end) : 0;
    J.first = min(P.sinks, J.lo);
    J.base = (J.lo - J.first) / STEP * STEP;
    J.n = end - J.base;
    J.steps = (J.n + STEP - 1) / STEP;
    return true;
}

// the steps a..z-1 that tile t's rows see
struct Span {
    int tokens, pos, a, z;
    int f0, f1;                 // steps f0..f1-1: every row sees every place that holds something
};
__device__ __forceinline__ Span span_of(const Prefill& P, const Job& J, int t) {
    Span s;
    s.tokens = max(0, min(P.tile_tokens, J.live - t * P.tile_tokens));
    s.pos = J.pos0 + t * P.tile_tokens;
    s.a = s.z = s.f0 = s.f1 = 0;
    if (s.tokens == 0) return s;
    const int ub = min(J.n, s.pos + s.tokens - J.base);               // end of what its last token sees
    s.z = (max(0, ub) + STEP - 1) / STEP;
    // what its first token sees begins here, but for first tokens
    if (P.window > 0 && P.sinks == 0) s.a = min(s.z, past((int64_t)s.pos + 1 - J.base, P.window) / STEP);
    // from where its last token's window has begun, to what its first token sees
    s.f0 = P.window > 0 ? (past((int64_t)s.pos + s.tokens - J.base, P.window) + STEP - 1) / STEP : 0;
    s.f1 = max(0, s.pos + 1 - J.base) / STEP;
    return s;
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1) prefill_kernel(const __grid_constant__ Prefill P,
                                                             const __grid_constant__ CUtensorMap tmk,
                                                             const __grid_constant__ CUtensorMap tmv) {
    using Ly = Layout<D>;
    constexpr int SLOTS = Ly::SLOTS;
    constexpr int CH = D / 8;
    extern __shared__ __align__(1024) char sm[];
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + Ly::BARS);
    uint64_t* empty = full + SLOTS;
    uint64_t* qbar = empty + SLOTS;
    uint64_t* sbar = qbar + 2;           // [tile][buffer]
    uint64_t* pbar = sbar + 4;
    uint64_t* obar = pbar + 4;
    uint64_t* endbar = obar + 4;         // all products
    volatile uint32_t* s_seen = reinterpret_cast<volatile uint32_t*>(sm + Ly::SEENB);
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_store;
    volatile int* s_abort = &s_abort_store;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        *s_abort = (smem_u32(sm) & 1023u) ? 2 : 0;
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(&full[s], 2);               // K and V
            mbar_init(&empty[s], 1);
        }
        mbar_init(&qbar[0], PRODUCERS);
        mbar_init(&qbar[1], 1);
        for (int t = 0; t < 2; ++t) {
            for (int k = 0; k < 2; ++k) {
                mbar_init(&sbar[2 * t + k], 2);       // the product's commit and the issuing thread
                mbar_init(&pbar[2 * t + k], SOFTMAX);
                mbar_init(&obar[2 * t + k], 1);   // the product of the last step but one, and of the last
            }
        }
        mbar_init(endbar, 1);
        fence_mbar_init();
    }
    if (warp == MMA_WARP) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const uint32_t base = smem_u32(sm);

    // Every role walks the same jobs.  Barriers are not begun anew with one: stages,
    // steps and jobs are counted on.
    int stage0 = 0, jobs = 0;             // stages and jobs with keys before this job
    if (warp >= PRODUCER0) {
        // ---------------- producers
        const int w = warp - PRODUCER0;
        const T* q = static_cast<const T*>(P.q);
        // 32 rows, one row address a lane, -1 for a row of zeros
        auto copy = [&](auto at, const T* src, int64_t off) {
#pragma unroll
            for (int it = 0; it < CH; ++it) {
                const int rr = (it * 32 + lane) / CH, c = (it * 32 + lane) % CH;
                const int64_t o = __shfl_sync(FULL, (long long)off, rr);
                cp_async16_or_zero(at(rr, c), src + (o >= 0 ? o + c * 8 : 0), o >= 0);
            }
        };
        constexpr int QPIECES = TILE / 32;
        uint32_t boxed = 0, turn = 0;       // ring slots that boxes went to, and the parity of their last turn
        Job J;
        for (int item = blockIdx.x; !*s_abort && find_job(P, item, J); item += gridDim.x) {
        if (J.steps == 0) continue;
        const Span sp[2] = {span_of(P, J, 0), span_of(P, J, 1)};
        if (!__all_sync(FULL, await(&qbar[1], (jobs & 1) ^ 1))) {
            *s_abort = 1;
            break;
        }
        for (int i = w; i < 2 * QPIECES; i += PRODUCERS) {
            const int t = i / QPIECES, piece = i % QPIECES;
            const int r = piece * 32 + lane, tok = r / J.heads;
            const int64_t off = tok < sp[t].tokens ? (J.token0 + t * P.tile_tokens + tok) * P.q_token_stride +
                                                         (int64_t)(J.head0 + r % J.heads) * P.q_head_stride
                                                   : -1;
            copy([&](int rr, int c) { return base + Ly::Q + t * Ly::QB + place<TILE>(piece * 32 + rr, c); }, q, off);
        }
        cp_async_commit();
        cp_async_wait<0>();
        if (P.flip) {
            // each thread turns the chunks that it copied itself
            for (int i = w; i < 2 * QPIECES; i += PRODUCERS)
#pragma unroll
                for (int it = 0; it < CH; ++it) {
                    const int rr = (it * 32 + lane) / CH, c = (it * 32 + lane) % CH;
                    uint4* p = reinterpret_cast<uint4*>(sm + Ly::Q + (i / QPIECES) * Ly::QB + place<TILE>(i % QPIECES * 32 + rr, c));
                    uint4 x = *p;
                    x.x ^= 0x80008000u;
                    x.y ^= 0x80008000u;
                    x.z ^= 0x80008000u;
                    x.w ^= 0x80008000u;
                    *p = x;
                }
        }
        fence_async_smem();
        arrive_warp(&qbar[0]);

        const T* kp = static_cast<const T*>(P.c.k) + (int64_t)J.g * P.c.head_stride;
        const T* vp = static_cast<const T*>(P.c.v) + (int64_t)J.g * P.c.head_stride;
        // parts in order: K and V of stage 0, of stage 1, ..; this warp has every third
        const int total = 2 * (J.steps + 2);
        // the step of part i, -1 where its stage has none
        auto step_of = [&](int i) {
            const int s = (i & 1) ? (i >> 1) - 2 : (i >> 1);
            return s < J.steps ? s : -1;
        };
        // the pages of this lane's rows of part i (lane and lane + 32), -1 where there is none
        auto find = [&](int i) -> int2 {
            const int s = step_of(i), u = s * STEP + lane;
            const bool in = i < total && s >= 0;
            return make_int2(in && J.holds(u) ? P.c.page(J.b, J.slot(u)) : -1,
                             in && J.holds(u + 32) ? P.c.page(J.b, J.slot(u + 32)) : -1);
        };
        const int in_page = (1 << P.c.shift) - 1;
        int waits[LAG], behind = 0;         // ring slots whose copies by cp.async are in flight
        auto hand_over = [&]() {
            cp_async_wait<0>();
            fence_async_smem();
#pragma unroll
            for (int k = 0; k < LAG; ++k)
                if (k < behind) arrive_warp(&full[waits[k]]);
            behind = 0;
        };
        int2 page = find(w);
        for (int i = w; i < total && !*s_abort; i += PRODUCERS) {
            const int stage = stage0 + (i >> 1), slot = stage % SLOTS, step = step_of(i);
            const bool is_v = i & 1;
            const int2 mine = page;
            page = find(i + PRODUCERS);
            const unsigned seen0 = __ballot_sync(FULL, mine.x >= 0), seen1 = __ballot_sync(FULL, mine.y >= 0);
            if (!is_v && lane == 0) {
                s_seen[(stage % SEEN) * 2] = seen0;
                s_seen[(stage % SEEN) * 2 + 1] = seen1;
            }
            const uint32_t phase = ((stage / SLOTS) & 1) ^ 1;
            if (!__all_sync(FULL, mbar_try_wait(&empty[slot], phase))) {
                hand_over();                // no room yet: first what is in flight
                if (!__all_sync(FULL, await(&empty[slot], phase))) {
                    *s_abort = 1;
                    break;
                }
            }
            if (step < 0) {
                arrive_warp(&full[slot]);
                continue;
            }
            const uint32_t dst = base + Ly::RING + slot * Ly::STAGEB + (is_v ? Ly::KB : 0);
            const int u = step * STEP + lane;
            if (P.tma && (seen0 & seen1) == FULL && step * STEP >= J.first) {
                if (lane == 0) mbar_expect_tx(&full[slot], Ly::KB);
                __syncwarp();
                boxed |= 1u << slot;
                turn = (turn & ~(1u << slot)) | ((uint32_t)((stage / SLOTS) & 1) << slot);
                // a lane a box: rows from the lane's own on, a panel of 64 dimensions
                const CUtensorMap* map = is_v ? &tmv : &tmk;
                if ((lane & (P.tma - 1)) == 0) {
                    const int at = (J.base + u) & in_page, at1 = (J.base + u + 32) & in_page;
#pragma unroll
                    for (int h = 0; h < D / 64; ++h) {
                        tma_box(dst + h * (STEP * 128) + lane * 128, map, h * 64, at, J.g, mine.x, &full[slot]);
                        tma_box(dst + h * (STEP * 128) + (lane + 32) * 128, map, h * 64, at1, J.g, mine.y, &full[slot]);
                    }
                }
                continue;
            }
            const T* src = is_v ? vp : kp;
            auto row = [&](int pg, int place_) -> int64_t {
                return pg >= 0 ? pg * P.c.page_stride + (int64_t)(J.slot(place_) & in_page) * P.c.row_stride : -1;
            };
            copy([&](int rr, int c) { return dst + place<STEP>(rr, c); }, src, row(mine.x, u));
            copy([&](int rr, int c) { return dst + place<STEP>(32 + rr, c); }, src, row(mine.y, u + 32));
            cp_async_commit();
            if (behind == LAG) {
                cp_async_wait<LAG>();
                fence_async_smem();
                arrive_warp(&full[waits[0]]);
#pragma unroll
                for (int k = 1; k < LAG; ++k) waits[k - 1] = waits[k];
                --behind;
            }
#pragma unroll
            for (int k = 0; k < LAG; ++k)
                if (k == behind) waits[k] = slot;
            ++behind;
            if (P.tma) hand_over();         // a boundary's rows: their step waits for them
            __syncwarp();
        }
        hand_over();
        stage0 += J.steps + 2;
        ++jobs;
        }
        // boxes that nobody waits for any more must not outlive the CTA
        if (*s_abort)
            for (int k = 0; k < SLOTS; ++k)
                if ((boxed >> k) & 1u) await(&full[k], (turn >> k) & 1u, 1ll << 24);
        __syncwarp();
        // tokens of no sequence, before the first or after the last, see nothing
        const int64_t s0 = clamp_start(P.starts, 0, P.tokens), s1 = max(s0, clamp_start(P.starts, P.c.seqs, P.tokens));
        for (int64_t i = (int64_t)blockIdx.x * PRODUCERS + w; i < s0 + P.tokens - s1; i += (int64_t)gridDim.x * PRODUCERS) {
            const int64_t row = (i < s0 ? i : s1 + i - s0) * P.q_heads;
            for (int64_t c = lane; c < (int64_t)P.q_heads * CH; c += 32)
                *reinterpret_cast<uint4*>(static_cast<T*>(P.out) + row * D + c * 8) = make_uint4(0u, 0u, 0u, 0u);
            for (int h = lane; h < P.q_heads; h += 32) P.lse[row + h] = NEG_INF;
        }
    } else if (warp == MMA_WARP) {
        // ---------------- MMA issuer
        const uint32_t tm = __shfl_sync(FULL, tmem, 0);
        int done[2] = {0, 0};             // a tile's steps before this job
        Job J;
        for (int item = blockIdx.x; !*s_abort && find_job(P, item, J); item += gridDim.x) {
        if (J.steps == 0) continue;
        const Span sp[2] = {span_of(P, J, 0), span_of(P, J, 1)};
        if (elect_one()) {
            constexpr uint32_t IS = instr<T>(STEP, false), IO = instr<T>(D, true);
            const uint32_t q0 = desc_k(base + Ly::Q), k0 = desc_k(base + Ly::RING), v0 = desc_v(base + Ly::RING + Ly::KB);
            bool ok = await(&qbar[0], jobs & 1);
            // stage q: each tile's product with step q - 2's weights, then its logits of step q
            for (int q = 0; ok && q < J.steps + 2; ++q) {
                const int slot = (stage0 + q) % SLOTS;
                ok = await(&full[slot], ((stage0 + q) / SLOTS) & 1);
                if (!ok) break;
                const uint32_t kd = k0 + slot * (Ly::STAGEB / 16), vd = v0 + slot * (Ly::STAGEB / 16);
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    // of the tile's own steps, in this job and in all; n + 2 has the same buffer
                    const int n = q - 2 - sp[t].a, all = done[t] + n, buf = all & 1;
                    const uint32_t st = tm + t * TILE + buf * STEP, ot = tm + 2 * TILE + t * D;
                    const bool more = n + 2 >= 0 && q < sp[t].z;
                    if (n >= 0 && q - 2 < sp[t].z) {
                        ok = await(&pbar[2 * t + buf], (all >> 1) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        mma_ts(ot, st, vd, IO, n > 0 ? 1u : 0u);
#pragma unroll
                        for (int k = 1; k < STEP / 16; ++k) mma_ts(ot, st + k * 8, vd + k * 128, IO, 1u);
                        // done when the logits' commit says so, or at the last two steps its own
                        if (!more) umma_commit(&obar[2 * t + (q - 2 == sp[t].z - 1)]);
                    }
                    if (more) {
                        tc_fence_after();
                        const uint32_t qd = q0 + t * (Ly::QB / 16);
                        mma_ss(st, qd, kd, IS, 0u);
#pragma unroll
                        for (int k = 1; k < D / 16; ++k)
                            mma_ss(st, qd + (k >> 2) * (TILE * 8) + (k & 3) * 2, kd + (k >> 2) * (STEP * 8) + (k & 3) * 2, IS, 1u);
                        umma_commit(&sbar[2 * t + buf]);
                        mbar_arrive(&sbar[2 * t + buf]);
                    }
                }
                if (!ok) break;
                umma_commit(&empty[slot]);
                if (q == J.steps - 1) umma_commit(&qbar[1]);
            }
            if (!ok) *s_abort = 1;
        }
        __syncwarp();
        stage0 += J.steps + 2;
        ++jobs;
        done[0] += sp[0].z - sp[0].a;
        done[1] += sp[1].z - sp[1].a;
        }
        // nor must products, which read its shared memory, nor their commits
        if (elect_one()) {
            umma_commit(endbar);
            if (!await(endbar, 0)) *s_abort = 1;
        }
        __syncwarp();
    } else {
        // ---------------- softmax: a thread is a row
        const int t = warp / SOFTMAX, r = threadIdx.x & (TILE - 1);
        // (after a wait that gave up these go on, to NaN)
        int done = 0, ends = 0, pairs = 0;    // the tile's steps, its jobs with a step, and with two, before this job
        Job J, next;
        bool more = find_job(P, blockIdx.x, J);
        for (int item = blockIdx.x; more; J = next) {
        const Span S = span_of(P, J, t);
        const int tok = r / J.heads;
        const bool live = tok < S.tokens;
        const int pos = S.pos + min(tok, S.tokens - 1);     // rows of no token see what the last one does
        const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ot = tmem + quarter + 2 * TILE + t * D;
        // of the places that hold something the row sees u < us and ua <= u, below ub
        const int ub = pos + 1 - J.base, us = max(J.first, P.sinks - J.base);
        const int ua = P.window > 0 ? past((int64_t)pos + 1 - J.base, P.window) : 0;
        constexpr float LIFT = Elem<T>::TOP > RAISE ? Elem<T>::TOP - RAISE : 0.f;   // log2 of what weights are multiplied by
        float m = NEG_INF;
        // the sum of the weights: of the last few steps, and of those before.  One running sum
        // would lose, one by one, the thousands of weights below 2^-24 of it that a long flat
        // tail has; what FOLD steps lose is below 2^-16 of it.
        float2 l[2] = {{0.f, 0.f}, {0.f, 0.f}};
        float before = 0.f;
        bool ok = !*s_abort;
        for (int j = S.a; j < S.z; ++j) {
            const int i = j - S.a, all = done + i, u0 = j * STEP, buf = all & 1;
            const uint32_t st = tmem + quarter + t * TILE + buf * STEP;
            ok = ok && await(&sbar[2 * t + buf], (all >> 1) & 1);
            if (!__all_sync(FULL, ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            // the row's logits, and the largest of them
            uint32_t x[2][32];
            tmem_get32(st, x[0]);
            tmem_get32(st + 32, x[1]);
            const uint2 seen = *reinterpret_cast<const uint2*>(const_cast<const uint32_t*>(s_seen) + ((stage0 + j) % SEEN) * 2);
            const bool masked = j < S.f0 || j >= S.f1 || (seen.x & seen.y) != 0xffffffffu;
            tmem_arrived(x[0]);
            tmem_arrived(x[1]);
            if (masked) {
                const uint32_t sw[2] = {seen.x, seen.y};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int u = u0 + c * 32;
                    const uint32_t vis = low_bits(ub - u) & (low_bits(us - u) | ~low_bits(ua - u)) & sw[c];
#pragma unroll
                    for (int e = 0; e < 32; ++e) x[c][e] = (vis >> e) & 1u ? x[c][e] : __float_as_uint(NEG_INF);
                }
            }
            float a[4] = {NEG_INF, NEG_INF, NEG_INF, NEG_INF};
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    a[2 * c + (e & 1)] = max3(a[2 * c + (e & 1)], __uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1]));
            const float top = max3(max3(a[0], a[1], a[2]), a[3], a[3]) * P.scale2;
            const bool raise = top > m + RAISE || (m == NEG_INF && top != NEG_INF);
            if (__any_sync(FULL, raise)) {
                const float f = raise && m != NEG_INF ? exp2_fast(m - top) : 1.f;
                if (raise) m = top;
                l[0] = make_float2(l[0].x * f, l[0].y * f);
                l[1] = make_float2(l[1].x * f, l[1].y * f);
                before *= f;
                if (i > 0) {
                    // the product of step i - 1 is done when the next logits are there, or at the
                    // last step when its own commit says so
                    ok = j + 1 < S.z ? await(&sbar[2 * t + (buf ^ 1)], ((all + 1) >> 1) & 1)
                                     : await(&obar[2 * t], pairs & 1);
                    if (!__all_sync(FULL, ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t z[16];
                        tmem_get16(ot + c * 16, z);
#pragma unroll
                        for (int e = 0; e < 16; ++e) z[e] = __float_as_uint(__uint_as_float(z[e]) * f);
                        tmem_put16(ot + c * 16, z);
                    }
                    tmem_stored();
                }
            }
            const float off = m == NEG_INF ? 0.f : LIFT - m;
            // weights over the logits' columns
            const unsigned long long s2 = pair(P.scale2, P.scale2), o2 = pair(off, off);
            unsigned long long l2[2] = {pair(l[0].x, l[0].y), pair(l[1].x, l[1].y)};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float2 y = halves(fma2(pair(__uint_as_float(x[c][2 * e]), __uint_as_float(x[c][2 * e + 1])), s2, o2));
                    const float w0 = exp2_fast(y.x), w1 = exp2_fast(y.y);
                    l2[e & 1] = add2(l2[e & 1], pair(w0, w1));
                    p[e] = Elem<T>::pack(w0, w1);
                }
                tmem_put16(st + c * 16, p);
            }
            l[0] = halves(l2[0]);
            l[1] = halves(l2[1]);
            tmem_stored();
            tc_fence_before();
            arrive_warp(&pbar[2 * t + buf]);
            if ((i & (FOLD - 1)) == FOLD - 1) {
                before += (l[0].x + l[0].y) + (l[1].x + l[1].y);
                l[0] = l[1] = make_float2(0.f, 0.f);
            }
        }
        // ---- the rows
        const int steps = S.z - S.a;
        item += gridDim.x;
        more = find_job(P, item, next);       // while the last product runs
        if (steps > 0) ok = ok && !*s_abort && await(&obar[2 * t + 1], ends & 1);
        ok = __all_sync(FULL, ok);
        if (!ok) *s_abort = 1;
        tc_fence_after();
        const float sum = before + ((l[0].x + l[0].y) + (l[1].x + l[1].y));
        const float inv = ok ? (sum == 0.f ? 0.f : 1.f / sum) : __int_as_float(0x7fffffff);
        const int64_t row = (J.token0 + t * P.tile_tokens + tok) * P.q_heads + J.head0 + r % J.heads;
        // through shared memory, so that a store writes whole 128-byte lines: 64 dimensions of
        // 32 rows at a time, chunks placed so that neither side meets in a bank
        char* box = sm + Ly::OUT + warp * (32 * 128);
#pragma unroll 1
        for (int h = 0; h < D / 64; ++h) {
            uint32_t z[2][32];
            if (steps > 0) {
                tmem_get32(ot + h * 64, z[0]);
                tmem_get32(ot + h * 64 + 32, z[1]);
                tmem_arrived(z[0]);
                tmem_arrived(z[1]);
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e) z[0][e] = z[1][e] = 0u;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                uint32_t p[4];
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    p[y] = Elem<T>::pack(__uint_as_float(z[c >> 2][(c & 3) * 8 + 2 * y]) * inv,
                                         __uint_as_float(z[c >> 2][(c & 3) * 8 + 2 * y + 1]) * inv);
                *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(p[0], p[1], p[2], p[3]);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int rr = i * 4 + (lane >> 3), c = lane & 7;
                const int64_t to = __shfl_sync(FULL, (long long)(live ? row : -1), rr);
                const uint4 y = *reinterpret_cast<const uint4*>(box + rr * 128 + ((c ^ (rr & 7)) << 4));
                if (to >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(P.out) + to * D + h * 64 + c * 8) = y;
            }
            __syncwarp();
        }
        if (live) P.lse[row] = !ok ? inv : sum == 0.f ? NEG_INF : (m - LIFT + log2f(sum)) * LN2;
        if (J.steps) stage0 += J.steps + 2;
        done += steps;
        ends += steps > 0;
        pairs += steps > 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*s_abort && threadIdx.x == 0 && P.status)
        *static_cast<volatile int32_t*>(P.status) = *s_abort == 2 ? SWB_ERR_SMEM : ERR_TIMEOUT;
    if (warp == MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// A pool as a map of boxes of 64 dimensions x `rows` rows of a page and head.
// Returns whether there is one: strides that a map cannot express are left to
// cp.async.
inline bool pool_map(CUtensorMap* m, const void* pool, const Cache& c, int d, bool bf16, int rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    if (!fn) {
        cudaDriverEntryPointQueryResult q;
        void* p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            return false;
        fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
    if (c.row_stride <= 0 || c.head_stride <= 0 || c.page_stride <= 0) return false;
    cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)1 << c.shift, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
    cuuint64_t strides[3] = {(cuuint64_t)c.row_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
    cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, step[4] = {1, 1, 1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(pool), dims,
              strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
int launch(Prefill p, int64_t items, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem((const void*)prefill_kernel<T, D>, Layout<D>::TOTAL, done);
    if (e != cudaSuccess) return abi::cuda_fail(e, "cudaFuncSetAttribute(prefill)");
    // 8 rows are a swizzle period, 32 a piece
    CUtensorMap mk = {}, mv = {};
    const int page = 1 << p.c.shift, rows = page < 32 ? page : 32;
    constexpr bool bf16 = Format<T>::F == 1;
    if (rows >= 8 && p.c.pages && pool_map(&mk, p.c.k, p.c, D, bf16, rows) && pool_map(&mv, p.c.v, p.c, D, bf16, rows))
        p.tma = rows;
    p.items = (int)items;
    const int64_t sms = abi::num_sms();
    prefill_kernel<T, D><<<(unsigned)(items < sms ? items : sms), THREADS, Layout<D>::TOTAL, st>>>(p, mk, mv);
    return abi::cuda_check("prefill launch");
}

}  // namespace pre
}  // namespace attn
}  // namespace swb

using namespace swb;
using namespace swb::attn;

extern "C" int32_t* swb_attn_status(void) { return wait_word().load(std::memory_order_acquire); }

extern "C" int swb_attn_prefill(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads,
                                const int32_t* starts, int64_t tokens, const swb_kv_cache* cache, float scale,
                                int window, int sinks, void* out, float* lse, int32_t* status, void* stream) {
    pre::Prefill p = {};
    int rc = check_cache(cache, &p.c);
    if (rc) return rc;
    if (tokens <= 0) return SWB_OK;
    rc = check_query(q, q_token_stride, q_head_stride, q_heads, p.c);
    if (rc) return rc;
    if (!starts || !out || !lse) return abi::fail(SWB_ERR_ARG, "null buffer");
    if (reinterpret_cast<uintptr_t>(out) % 16) return abi::fail(SWB_ERR_ARG, "out must start on a 16-byte boundary");
    if (window < 0 || sinks < 0) return abi::fail(SWB_ERR_ARG, "window and sinks must not be negative");
    p.q = q;
    p.q_token_stride = q_token_stride;
    p.q_head_stride = q_head_stride;
    p.starts = starts;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.group = q_heads / p.c.kv_heads;
    p.tile_heads = p.group < pre::TILE ? p.group : pre::TILE;
    p.head_tiles = (p.group + p.tile_heads - 1) / p.tile_heads;
    p.tile_tokens = pre::TILE / p.tile_heads;
    p.flip = scale < 0.f;
    // a scale of 0 is the smallest number instead: logits of 0, and -inf stays what it is
    p.scale2 = fmaxf((scale < 0.f ? -scale : scale) * LOG2E, 1.2e-38f);
    p.window = window;
    p.sinks = sinks;
    p.out = out;
    p.lse = lse;
    rc = earlier_wait();
    if (rc) return rc;
    p.status = status ? status : make_wait_word();
    // every sequence may end in a tile that is not full
    const int64_t step = 2 * p.tile_tokens;
    const int64_t items = ((tokens + step - 1) / step + p.c.seqs) * p.c.kv_heads * p.head_tiles;
    if (items >= ((int64_t)1 << 30) || tokens >= ((int64_t)1 << 31) - 256) return abi::fail(SWB_ERR_ARG, "too many tokens in one call");
    cudaStream_t st = (cudaStream_t)stream;
    if (cache->dtype == SWB_F16)
        return cache->head_dim == 64 ? pre::launch<__half, 64>(p, items, st) : pre::launch<__half, 128>(p, items, st);
    return cache->head_dim == 64 ? pre::launch<__nv_bfloat16, 64>(p, items, st)
                                 : pre::launch<__nv_bfloat16, 128>(p, items, st);
}
