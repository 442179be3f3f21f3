// What the kernels of the decoding step share: division by a page size that is only known at launch, the word that
// records an index out of range, 16-byte asynchronous copies and the m16n8k16 matrix instruction.
#pragma once

#include <atomic>

#include "sm100.cuh"

namespace enc {

// Index arrays are device data, so the host cannot check them before the launch.  A kernel that meets a value out of
// range skips the access and raises this word; enc_synchronize reports it.  One word per source file that includes this
// header and per device, in the library image: reaching it needs no allocation, so a captured launch can raise it too.
static __device__ unsigned int g_bad_index;

// Host side of the word above: reads and clears the current device's (synchronous).
static inline unsigned int take_bad_index_word() {
    unsigned int host = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&host, g_bad_index, sizeof(host)) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (host) cudaMemcpyToSymbol(g_bad_index, &zero, sizeof(zero));
    return host;
}

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 by one multiplication (Granlund & Montgomery, "Division by invariant
// integers using multiplication", PLDI 1994): with s = ceil(log2 d) and mul = ceil(2^(31+s) / d) < 2^32,
// floor(n * mul / 2^(31+s)) = floor(n / d).
struct FastDiv {
    uint32_t d, mul, shift;
    explicit FastDiv(uint32_t div = 1) : d(div) {
        uint32_t s = 0;
        while (s < 31 && (1ull << s) < div) ++s;
        shift = s;
        mul = (uint32_t)(((1ull << (31 + s)) + div - 1) / div);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> (31 + shift)); }
};

// Shape checks of a cache that every entry point makes; 0 or a status.
static inline int check_cache(const enc_paged_cache &c, const char *me) {
    if (c.num_pages < 0 || c.num_seqs < 0 || c.table_width < 0 || c.page_size < 1 || c.kv_heads < 1 || c.head_dim < 1)
        return fail(ENC_ERR_BAD_ARG, "%s: bad cache shape (%lld pages of %lld tokens, %lld heads of %lld, table %lld x %lld)", me,
                    (long long)c.num_pages, (long long)c.page_size, (long long)c.kv_heads, (long long)c.head_dim,
                    (long long)c.num_seqs, (long long)c.table_width);
    if (c.page_size > 0x7fffffffLL || c.num_pages > 0x7fffffffLL || c.num_seqs > 0x7fffffffLL || c.table_width > 0x7fffffffLL ||
        c.kv_heads > 0xffff || c.head_dim > 0xffff)
        return fail(ENC_ERR_UNSUPPORTED, "%s: a cache dimension beyond 2^31-1 (65535 for heads and head_dim)", me);
    return 0;
}
// Tokens that a row of the block table can address (positions are 32-bit).
static inline int64_t paged_capacity(const enc_paged_cache &c) {
    const int64_t n = c.table_width * c.page_size;  // both below 2^31
    return n < 0x7fffff00LL ? n : 0x7fffff00LL;  // (room for the last tile in 32 bits)
}

// Opting in to more than 48 KB of shared memory, once per kernel and device instead of at every launch.
struct OncePerDevice {
    std::atomic<uint64_t> done{0};
    template <typename K> int opt_in(K kernel, int bytes, const char *me) {
        int dev = 0;
        cudaGetDevice(&dev);
        const uint64_t bit = 1ull << (dev & 63);
        if (done.load(std::memory_order_acquire) & bit) return ENC_OK;
        const int most = device_props().max_smem_optin;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most > 0 && bytes > most ? most : bytes);
        if (e != cudaSuccess) return fail(ENC_ERR_LAUNCH, "%s: cannot opt in to %d bytes of shared memory: %s", me, bytes, cudaGetErrorString(e));
        done.fetch_or(bit, std::memory_order_release);
        return ENC_OK;
    }
};

#ifdef __CUDACC__
using sm100::smem_u32;

// 16 bytes global -> shared; with bytes == 0 nothing is read and 16 zero bytes are written.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 matrix of 16-bit elements held across the warp (row lane / 4, columns 2 (lane % 4) + {0, 1}), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// c[16x8] += a[16x16] b[16x8], float32 accumulation
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
#endif

}  // namespace enc
