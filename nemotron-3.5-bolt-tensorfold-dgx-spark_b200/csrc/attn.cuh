// Shared pieces of the paged attention kernels: their arguments, the score's scaling, the cache's tensor maps.
#pragma once
#include <atomic>
#include <cfloat>
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
    uint32_t group_mul, group_shift;
    int pages, page_log2;
    float c;                   // a score times c is the exponent in powers of two (log2 e * scale; softcap: log2 e * cap)
    float cap_in;              // softcap: scale / cap, 0: none
    bool cap_exact;            // a cap above 512
    float cap_near;            // scores up to here in size are capped by cap_poly: s sum_k cap_poly[k] s^2k (attn_tc.cuh)
    float cap_poly[3];
    bool whole;                // decode form: no row block is cut, so none is joined
    int window;                // keys a row sees at most (INT_MAX / 2: no window)
    void* ws;
    const __nv_bfloat16 *kp, *vp;   // the cache as row_again (attn_line.cuh) reads it; the kernels' tiles come by tensor maps
    int64_t k_stride, v_stride;
    // row / group for rows below 2^31: with 2^s >= group > 2^(s-1) and mul = floor(2^32 (2^s - group) / group) + 1, the quotient
    // is (floor(row mul / 2^32) + row) >> s (Granlund and Montgomery)
    __device__ __forceinline__ int token(int row) const { return (int)((__umulhi((uint32_t)row, group_mul) + (uint32_t)row) >> group_shift); }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A raw score q . k with a cap, in caps: tanh(scale q.k / cap).  The exponent is the cap times it.  1 - 2 / (exp(2 y) + 1) leaves an
// error of 1.5 2^-22 at most, below 2^-12 in the exponent for caps up to 512; from there on tanhf, right to 2 steps of its value
// (it costs capped prompts a tenth more where scores come near the cap, so not for all; tanh.approx would leave 2^-11).
__device__ __forceinline__ float capped(float x, float cap_in, bool exact) {
    const float y = x * cap_in;
    return exact ? tanhf(y) : 1.f - __fdividef(2.f, ex2(y * 2.885390081777927f) + 1.f);
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
           scale < 2e38f && softcap >= 0.f && softcap < 1e38f &&   // the exponents' factor, log2 e times one of them, is finite
           (softcap == 0.f || (scale / softcap < INFINITY && scale / softcap >= FLT_MIN)) && window >= 0;
}
inline AttnArgs attn_args(const b200q_paged& kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                          int window, void* out, int64_t ldo, void* ws) {
    AttnArgs a = {};
    a.q = (const __nv_bfloat16*)q; a.ldq = ldq; a.rows = rows; a.out = (__nv_bfloat16*)out; a.ldo = ldo; a.s = kv_seqs(kv);
    a.max_rows = max_rows; a.hkv = kv.hkv; a.group = hq / kv.hkv;
    while ((1u << a.group_shift) < (uint32_t)a.group) a.group_shift++;
    a.group_mul = (uint32_t)((((uint64_t)((1u << a.group_shift) - a.group)) << 32) / a.group + 1);
    a.pages = kv.pages; a.page_log2 = log2_of(kv.page);
    a.c = 1.4426950408889634f * (softcap > 0.f ? softcap : scale);
    a.cap_in = softcap > 0.f ? scale / softcap : 0.f;
    a.cap_exact = softcap > 512.f;
    // tanh(u) for |u| <= 3/8: u times the polynomial of degree 2 in u^2 with the least relative error (4.3e-6, a Remez fit), in
    // terms of the score; its powers are ordinary numbers for scale / cap within 2^20 of 1.  Up to a capped score of 56 that is
    // below 2^-12 of a probability, 2^-4 of P's rounding to bf16; beyond, as beyond 3/8 of the cap, capped().
    static const double tanh_poly[3] = {0.999995707885, -0.332780666598, 0.122647585951};
    if (a.cap_in > 0x1p-20f && a.cap_in < 0x1p20f) {
        a.cap_near = fminf(0.375f / a.cap_in, 56.f / scale);
        double u = a.cap_in;
        for (int k = 0; k < 3; k++, u *= (double)a.cap_in * a.cap_in) a.cap_poly[k] = (float)(tanh_poly[k] * u);
    }
    a.window = window > 0 && window < INT_MAX / 2 ? window : INT_MAX / 2;
    a.ws = ws;
    a.kp = (const __nv_bfloat16*)kv.k_pages; a.vp = (const __nv_bfloat16*)kv.v_pages; a.k_stride = kv.k_stride; a.v_stride = kv.v_stride;
    return a;
}

// The tensor-core form (attn_prompt.cu), which the decode form calls for more rows than its own kernel takes: workspace bytes
// for up to `rows` rows a sequence and kv head, and the launch, returning a status.
size_t prompt_workspace(int d, int64_t rows);
int prompt_launch(const b200q_paged& kv, const AttnArgs& a, void* stream);

}  // namespace b200q
