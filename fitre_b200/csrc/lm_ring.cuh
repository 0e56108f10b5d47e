// A ring of buffers in shared memory that bulk copies fill with rows of global memory (rows on 16-byte
// boundaries, whole multiples of 16 bytes).  One thread fills, all threads of the block read; a
// block-wide barrier between the last read of a stage and its refill is the caller's, as is that every value
// read has been used before it: a load whose value has been used cannot be overtaken by the refill, which is
// written through the asynchronous proxy.
#pragma once

#include "tma_util.cuh"

namespace fitre {
namespace {

constexpr int kRingMax = 8;

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

struct RowRing {
    unsigned char *base;
    unsigned long long *bars;
    int stages, bytes, at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ RowRing(unsigned char *b, unsigned long long *m, int s, int n)
        : base(b), bars(m), stages(s), bytes(n) {}
    __device__ __forceinline__ void init() {
        if (threadIdx.x == 0) {
            for (int i = 0; i < stages; ++i) mbar_init(smem_u32(bars + i), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    __device__ __forceinline__ void fill(int i, const void *src) {
        const uint32_t bar = smem_u32(bars + i);
        mbar_expect_tx(bar, bytes);
        bulk_load(smem_u32(base + (size_t)i * bytes), src, bytes, bar);
    }
    // `n` rows of a pair of matrices, `each` bytes a row and `step` rows apart: a's and b's rows in turn
    template <class T>
    __device__ __forceinline__ void fill_pairs(int i, const T *a, long lda, const T *b, long ldb, long row, long step, int n,
                                               int each) {
        const uint32_t bar = smem_u32(bars + i), dst = smem_u32(base + (size_t)i * bytes);
        mbar_expect_tx(bar, 2 * n * each);
        for (int k = 0; k < n; ++k) {
            bulk_load(dst + 2 * k * each, a + (row + k * step) * lda, each, bar);
            bulk_load(dst + (2 * k + 1) * each, b + (row + k * step) * ldb, each, bar);
        }
    }
    // false: the bounded wait ran out
    __device__ __forceinline__ bool wait() const { return mbar_wait(smem_u32(bars + at), phase); }
    __device__ __forceinline__ const unsigned char *data() const { return base + (size_t)at * bytes; }
    __device__ __forceinline__ void advance() {
        if (++at == stages) {
            at = 0;
            phase ^= 1;
        }
    }
};

}  // namespace
}  // namespace fitre
