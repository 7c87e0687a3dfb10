// attn.cuh -- what the attention operators share: the 16-bit element types,
// the paged key-value cache as the kernels see it, and the warp-level matrix
// instructions of the kernels that are bound by memory.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "../../include/swann_b200.h"
#include "abi_util.h"
#include "common.cuh"

namespace swb {
namespace attn {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NEG_INF = -__builtin_huge_valf();

// -- element types ------------------------------------------------------------

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
    // A softmax weight that is rounded to this type is taken 2^x times larger, x so that the
    // largest comes to 2^TOP: fp16's steps end at 2^-24, and a weight of 2^-25 of the largest
    // would be 0 in the product with V but count in the sum.
    static constexpr float TOP = 15.f;
    static __device__ __forceinline__ float2 wide(uint32_t u) {
        return __half22float2(*reinterpret_cast<const __half2*>(&u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <>
struct Elem<__nv_bfloat16> {
    static constexpr float TOP = 0.f;      // has the exponents of fp32
    static __device__ __forceinline__ float2 wide(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

// four 8x8 matrices of 16-bit elements; lane l gives the address of row l % 8 of matrix l / 8
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// 2^x; -inf gives 0
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes global -> shared, or 16 zero bytes where `real` is false (nothing is read then)
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}

// -- the cache ------------------------------------------------------------------

struct Cache {
    const void* k;
    const void* v;
    int64_t page_stride, head_stride, row_stride;   // elements
    const int32_t* table;
    int64_t table_stride;
    const int32_t* lengths;
    int pages, max_pages, shift, seqs, kv_heads;

    // slots that the table has room for
    __host__ __device__ __forceinline__ int64_t capacity() const { return (int64_t)max_pages << shift; }
    // slots that sequence b holds: never more than its table has room for
    __device__ __forceinline__ int length(int b) const {
        const int64_t n = lengths[b];
        return (int)max((int64_t)0, min(n, capacity()));
    }
    // the page of a slot; -1 where the table names none of the pool's
    __device__ __forceinline__ int page(int b, int slot) const {
        const int p = table[(int64_t)b * table_stride + (slot >> shift)];
        return (unsigned)p < (unsigned)pages ? p : -1;
    }
    // element offset of a slot's row in a pool, for head 0; -1 without a page
    __device__ __forceinline__ int64_t row(int b, int slot) const {
        const int p = page(b, slot);
        if (p < 0) return -1;
        return p * page_stride + (int64_t)(slot & ((1 << shift) - 1)) * row_stride;
    }
};

// a sequence's first token in a ragged batch, never outside the batch
__device__ __forceinline__ int64_t clamp_start(const int32_t* starts, int b, int64_t tokens) {
    return max((int64_t)0, min((int64_t)starts[b], tokens));
}

// -- host side --------------------------------------------------------------

inline int log2_exact(int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return (1 << s) == x ? s : -1;
}

// checks a caller's cache and turns it into the kernels' form
inline int check_cache(const swb_kv_cache* c, Cache* out) {
    if (!c) return abi::fail(SWB_ERR_ARG, "null cache");
    if (c->seqs < 0 || c->kv_heads < 1 || c->max_pages < 0 || c->pages < 0)
        return abi::fail(SWB_ERR_ARG, "cache: sizes out of range");
    if (c->dtype != SWB_F16 && c->dtype != SWB_BF16) return abi::fail(SWB_ERR_ARG, "cache: fp16 or bf16");
    if (c->head_dim != 64 && c->head_dim != 128) return abi::fail(SWB_ERR_ARG, "cache: head_dim must be 64 or 128");
    const int shift = c->page_size >= 1 && c->page_size <= (1 << 20) ? log2_exact(c->page_size) : -1;
    if (shift < 0) return abi::fail(SWB_ERR_ARG, "cache: page_size must be a power of two up to 2^20");
    if (((int64_t)c->max_pages << shift) >= ((int64_t)1 << 31))
        return abi::fail(SWB_ERR_ARG, "cache: at most 2^31 - 1 slots a sequence");
    if (c->seqs && (!c->lengths || (c->max_pages && !c->table))) return abi::fail(SWB_ERR_ARG, "cache: null table");
    if (c->pages && (!c->k || !c->v)) return abi::fail(SWB_ERR_ARG, "cache: null pool");
    if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16 || c->page_stride % 8 ||
        c->head_stride % 8 || c->row_stride % 8)
        return abi::fail(SWB_ERR_ARG, "cache: rows must start on 16-byte boundaries");
    // without pages nothing is read, but 16-byte copies of nothing want an address all the
    // same, on their boundary: lengths need not lie on one, the 16 bytes they begin in do
    const void* none = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(c->lengths) & ~(uintptr_t)15);
    out->k = c->pages ? c->k : none;
    out->v = c->pages ? c->v : none;
    out->page_stride = c->page_stride;
    out->head_stride = c->pages ? c->head_stride : 0;
    out->row_stride = c->row_stride;
    out->table = c->table;
    out->table_stride = c->table_stride;
    out->lengths = c->lengths;
    out->pages = c->pages;
    out->max_pages = c->max_pages;
    out->shift = shift;
    out->seqs = c->seqs;
    out->kv_heads = c->kv_heads;
    return SWB_OK;
}

inline int check_query(const void* q, int64_t ts, int64_t hs, int q_heads, const Cache& c) {
    if (!q) return abi::fail(SWB_ERR_ARG, "null queries");
    if (q_heads < 1 || q_heads % c.kv_heads)
        return abi::fail(SWB_ERR_ARG, "query heads must be a multiple of the cache's key heads");
    if (reinterpret_cast<uintptr_t>(q) % 16 || ts % 8 || hs % 8)
        return abi::fail(SWB_ERR_ARG, "query rows must start on 16-byte boundaries");
    return SWB_OK;
}

// Lets `kernel` have `bytes` of dynamic shared memory; asked of the driver once a
// device (`done`: one bit each, a static of the caller's).
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    const int dev = abi::current_device();
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Where a prefill whose caller gives no status word says that a wait gave up: a word of
// host memory that the device writes, one for the process, made by its first prefill.
// Every call looks at it (nothing waits for that) and reports what it finds once, as
// the errors of earlier launches are reported.
inline std::atomic<int32_t*>& wait_word() {
    static std::atomic<int32_t*> word{nullptr};
    return word;
}
inline int32_t* make_wait_word() {
    int32_t* w = wait_word().load(std::memory_order_acquire);
    if (w) return w;
    // a stream may be capturing: this touches none
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) return nullptr;
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped);
    if (e != cudaSuccess) cudaGetLastError();
    else *static_cast<volatile int32_t*>(p) = 0;
    int32_t* mine = e == cudaSuccess ? static_cast<int32_t*>(p) : nullptr;
    if (mine && !wait_word().compare_exchange_strong(w, mine, std::memory_order_acq_rel)) {
        cudaFreeHost(mine);
        mine = w;
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
    return mine;
}
inline int earlier_wait() {
    volatile int32_t* w = wait_word().load(std::memory_order_acquire);
    const int code = w ? *w : 0;
    if (!code) return SWB_OK;
    *w = 0;
    return abi::fail(code, "an earlier prefill failed: a device-side wait gave up, and rows of its are NaN");
}

// Launches a kernel that may begin while the one before it in the stream ends:
// the kernel itself waits (dependency_wait) before it reads what that wrote.
template <typename... P, typename... A>
inline cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void dependency_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace attn
}  // namespace swb
