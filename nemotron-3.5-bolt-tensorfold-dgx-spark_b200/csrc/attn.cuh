// Shared pieces of the paged attention kernels: their arguments, the score's scaling, the cache's tensor maps.
#pragma once
#include <atomic>
#include <climits>
#include <cmath>

#include <cuda.h>   // CUtensorMap and its enums: types alone, the encoder is looked up at run time

#include "kv.cuh"

namespace b200q {

struct AttnArgs {
    const __nv_bfloat16* q;
    __nv_bfloat16* out;
    int64_t ldq, ldo;
    KvSeqs s;
    int rows, max_rows;        // rows of q; the most rows of a sequence
    int hkv, group;            // kv heads, query heads a kv head
    int pages, page_log2;
    float c;                   // a score times c is the exponent in powers of two (log2 e * scale; softcap: log2 e * cap)
    float cap_in;              // softcap: scale / cap, 0: none
    int window;                // keys a row sees at most (INT_MAX / 2: no window)
    void* ws;
};

// The exponent of a raw score q . k: with a cap, cap * tanh(scale q.k / cap) = cap * (1 - 2 / (exp(2 y) + 1)).  The
// subtraction leaves 2^-24 of the cap, far below bf16; tanh.approx (2^-11) would move a score of 50 by 0.02.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float capped(float x, float cap_in) {
    return 1.f - __fdividef(2.f, ex2(x * cap_in * 2.885390081777927f) + 1.f);
}

__device__ __forceinline__ void tma_prefetch(const CUtensorMap* m) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(m) : "memory");
}
// rows `row` .. of page `page`, kv head `head`: box of 64 values x (the map's rows) x d / 64, each 64-value column block
// [rows][128 B] in the 128-byte swizzle
__device__ __forceinline__ void tma_kv(uint32_t dst, const CUtensorMap* m, int row, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4, %5}], [%6];"
        ::"r"(dst), "l"(m), "r"(0), "r"(row), "r"(head), "r"(page), "r"(bar) : "memory");
}

// the tensor map of one side of the cache: dims (64, page, d / 64, heads, pages), box (64, box_rows, box_blocks, 1, 1)
bool kv_tensor_map(CUtensorMap* m, const void* pages, int64_t stride, const b200q_paged& kv, int box_rows, int box_blocks);

// a kernel's dynamic shared memory allowed once a device
struct SmemOptIn {
    std::atomic<uint64_t> done{0};
    cudaError_t allow(const void* kernel, size_t bytes) {
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess || (dev < 64 && (done.load() >> dev & 1))) return e;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e == cudaSuccess && dev < 64) done |= (uint64_t)1 << dev;
        return e;
    }
};

// the checks both forms share
inline bool attn_ok(const b200q_paged* kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                    int window, const void* out, int64_t ldo, const void* workspace) {
    return kv_ok(kv) && q && out && workspace && aligned(q, 16) && aligned(out, 16) && aligned(workspace, 16) && ldq % 8 == 0 &&
           ldo % 8 == 0 && rows >= 0 && hq > 0 && hq <= 4096 && hq % kv->hkv == 0 && ldq >= (int64_t)hq * kv->d &&
           ldo >= (int64_t)hq * kv->d && max_rows > 0 && (int64_t)max_rows * (hq / kv->hkv) < (1 << 30) && scale > 0.f &&
           scale < INFINITY && softcap >= 0.f && softcap < INFINITY && window >= 0;
}
inline AttnArgs attn_args(const b200q_paged& kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                          int window, void* out, int64_t ldo, void* ws) {
    AttnArgs a = {};
    a.q = (const __nv_bfloat16*)q; a.ldq = ldq; a.rows = rows; a.out = (__nv_bfloat16*)out; a.ldo = ldo; a.s = kv_seqs(kv);
    a.max_rows = max_rows; a.hkv = kv.hkv; a.group = hq / kv.hkv; a.pages = kv.pages; a.page_log2 = log2_of(kv.page);
    a.c = 1.4426950408889634f * (softcap > 0.f ? softcap : scale);
    a.cap_in = softcap > 0.f ? scale / softcap : 0.f;
    a.window = window > 0 && window < INT_MAX / 2 ? window : INT_MAX / 2;
    a.ws = ws;
    return a;
}

}  // namespace b200q
