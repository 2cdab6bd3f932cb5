// Appending a step's keys and values to a paged cache (the role of kv_store_k, bolt_kernels.cu:1735), with what stands
// between the q/k/v projection and the attention on the way: the RMS norm of each query and key head (optional), the
// rotation by position (optional) and the rounding to bf16.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        per head, fp32
//   (a, c) -> (a cos t - c sin t, c cos t + a sin t)          t = position * inv_freq[i], pairs (i, i + R/2) or (2i, 2i + 1)
//
// The angle is a product of a position and an fp32 frequency, formed and reduced by 2 pi in fp64 (exact but for the
// reduction's last bits: at position 2^18 an fp32 angle would be off by up to 2^-7), then one sincosf of the remainder.
// cos and sin depend on the token alone, so a CTA computes them once for all heads of its token, in shared memory.
//
// Bound by HBM: every input value is read once and every output written once (bf16).  A CTA takes one token; each of its
// warps keeps kUnroll loads of 32 lanes x 8 values in flight before the first is used (a head is d / 8 lanes, so a warp's
// load covers two heads of 128 or four of 64, and the partner of a rotated half is a shuffle away).
#include "kv.cuh"

namespace b200q {

__device__ int g_kv_error;   // bit 0: a position outside the page table, or a table entry outside the cache

int kv_error_read(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_kv_error, sizeof(int)) != cudaSuccess) return -1;
    if (clear) {
        const int z = 0;
        cudaMemcpyToSymbol(g_kv_error, &z, sizeof(int));
    }
    return v;
}

struct AppendArgs {
    const void *q, *k, *v;
    int64_t ldq, ldk, ldv;
    int rows, hq, hkv;
    __nv_bfloat16 *kp, *vp;
    int64_t k_stride, v_stride;
    int pages, page_log2;
    KvSeqs s;
    const float* inv_freq;
    int rope;                 // rotated dims of a head (0: none)
    const void *q_norm, *k_norm;
    int norm_dtype;
    float eps;
    __nv_bfloat16* qo;
    int64_t ldo;
};

constexpr int kAppendWarps = 8;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
    const float4 a = *(const float4*)p, b = *((const float4*)p + 1);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 a = *(const uint4*)p;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// the sequence that row t belongs to (batch if none), by the whole warp: the count of range ends at or before t
__device__ __forceinline__ int row_sequence(const KvSeqs& s, int t, int lane) {
    int b = 0;
    for (int j = lane; j - lane < s.batch; j += 32) b += __popc(__ballot_sync(~0u, j < s.batch && s.cu[j + 1] <= t));
    return b;
}

template <typename T, int D, bool INTERLEAVED, int U>
__global__ void __launch_bounds__(kAppendWarps * 32) kv_append_k(AppendArgs a) {
    pdl_wait();
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes;   // lanes of a head, heads of a warp's load
    __shared__ float2 cs[D / 2];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
    const int heads = a.hq + 2 * a.hkv;
    const int sub = lane / kLanes, e0 = (lane % kLanes) * 8;   // this lane's head of the load, first value in it

    const int b = row_sequence(a.s, t, lane);
    if (b >= a.s.batch || t < a.s.cu[0]) { pdl_trigger(); return; }   // padding rows
    const int pos = a.s.lens[b] - a.s.cu[b + 1] + t;
    if (pos < 0) { pdl_trigger(); return; }   // more rows than tokens: no place
    const int entry = pos >> a.page_log2;
    int page = -1;
    if (entry < a.s.width) page = a.s.table[b * a.s.ldt + entry];
    const bool stored = page >= 0 && page < a.pages;
    if (!stored && threadIdx.x == 0) atomicOr(&g_kv_error, 1);
    const int half = a.rope >> 1;
    for (int i = threadIdx.x; i < half; i += blockDim.x) {
        const double turn = (double)pos * (double)a.inv_freq[i];
        const float r = (float)fma(-6.283185307179586476925, rint(turn * 0.15915494309189533577), turn);
        float2 v;
        sincosf(r, &v.y, &v.x);
        cs[i] = v;
    }
    __syncthreads();

    const int step = (int)gridDim.y * kAppendWarps * kHeads;
    for (int h0 = ((int)blockIdx.y * kAppendWarps + warp) * kHeads; h0 < heads; h0 += step * U) {
        float x[U][8];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + u * step + sub;
            if (h >= heads) continue;
            const T* p = h < a.hq ? (const T*)a.q + t * a.ldq + h * D
                       : h < a.hq + a.hkv ? (const T*)a.k + t * a.ldk + (h - a.hq) * D
                                          : (const T*)a.v + t * a.ldv + (h - a.hq - a.hkv) * D;
            load8(p + e0, x[u]);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int h = h0 + u * step + sub;
            const bool live = h < heads, is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
            const void* w = is_q ? a.q_norm : a.k_norm;
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < 8; j++) ss = fmaf(x[u][j], x[u][j], ss);
#pragma unroll
            for (int m = kLanes / 2; m; m >>= 1) ss += __shfl_xor_sync(~0u, ss, m);
            if (live && !is_v && w) {
                const float r = rsqrtf(ss * (1.f / D) + a.eps);
                float wv[8];
                if (a.norm_dtype == B200Q_F32) load8((const float*)w + e0, wv);
                else load8((const __nv_bfloat16*)w + e0, wv);
#pragma unroll
                for (int j = 0; j < 8; j++) x[u][j] = x[u][j] * r * wv[j];
            }
            if (a.rope) {
                if (INTERLEAVED) {
                    if (live && !is_v && e0 < a.rope) {
#pragma unroll
                        for (int j = 0; j < 8; j += 2) {
                            const float2 v = cs[(e0 + j) >> 1];
                            const float p = x[u][j], c = x[u][j + 1];
                            x[u][j] = p * v.x - c * v.y;
                            x[u][j + 1] = c * v.x + p * v.y;
                        }
                    }
                } else {
                    // rope % 16 == 0: a lane's eight values lie in one half, their partners in one other lane
                    const bool turned = e0 < a.rope, low = e0 < half;
                    const int from = turned ? lane + (low ? half : -half) / 8 : lane;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float o = __shfl_sync(~0u, x[u][j], from);
                        if (live && !is_v && turned) {
                            const float2 v = cs[low ? e0 + j : e0 - half + j];
                            x[u][j] = x[u][j] * v.x + (low ? -o : o) * v.y;
                        }
                    }
                }
            }
            if (!live) continue;
            __nv_bfloat162 o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = __floats2bfloat162_rn(x[u][2 * j], x[u][2 * j + 1]);   // the cache's type
            if (is_q) *(uint4*)(a.qo + t * a.ldo + h * D + e0) = *(uint4*)o;
            else if (stored) {
                const int hk = is_v ? h - a.hq - a.hkv : h - a.hq;
                __nv_bfloat16* c = (is_v ? a.vp + page * a.v_stride : a.kp + page * a.k_stride);
                *(uint4*)(c + (((int64_t)hk << a.page_log2) + (pos & ((1 << a.page_log2) - 1))) * D + e0) = *(uint4*)o;
            }
        }
    }
    pdl_trigger();
}

template <typename T, int D>
static cudaError_t launch_append(const AppendArgs& a, int interleaved, cudaStream_t s) {
    constexpr int kHeads = 32 / (D / 8), U = 3;
    // few tokens: a token's heads over several CTAs, until each warp has one load or there are two CTAs an SM
    const int loads = (a.hq + 2 * a.hkv + kHeads - 1) / kHeads, most = (loads + kAppendWarps - 1) / kAppendWarps;
    int split = 1;
    while (split < most && (int64_t)a.rows * split < 2 * 148) split++;
    const dim3 grid((unsigned)a.rows, (unsigned)split);
    return interleaved ? launch(kv_append_k<T, D, true, U>, grid, dim3(kAppendWarps * 32), 0, s, a)
                       : launch(kv_append_k<T, D, false, U>, grid, dim3(kAppendWarps * 32), 0, s, a);
}

}  // namespace b200q

using namespace b200q;

extern "C" int b200q_kv_append(const b200q_paged* kv, const void* q, const void* k, const void* v, int x_dtype, int64_t ldq,
                               int64_t ldk, int64_t ldv, int rows, int hq, const float* inv_freq, int rope, int interleaved,
                               const void* q_norm, const void* k_norm, int norm_dtype, float eps, void* q_out, int64_t ldo,
                               void* stream) {
    if (!kv_ok(kv)) return B200Q_EINVAL;
    const int e = x_dtype == B200Q_F32 ? 4 : 2, d = kv->d;
    const int64_t wq = (int64_t)hq * d, wk = (int64_t)kv->hkv * d;
    if (rows < 0 || hq < 0 || hq > 4096 || (x_dtype != B200Q_F32 && x_dtype != B200Q_BF16) || !k || !v ||
        (hq > 0 && (!q || !q_out || ldq < wq || ldo < wq)) || !aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) ||
        !aligned(q_out, 16) || (ldq * e) % 16 || (ldk * e) % 16 || (ldv * e) % 16 || ldo % 8 || ldk < wk || ldv < wk ||
        rope < 0 || rope > d || rope % 16 || (rope && !inv_freq) || !aligned(inv_freq, 4) ||
        ((q_norm || k_norm) && ((norm_dtype != B200Q_F32 && norm_dtype != B200Q_BF16) || !(eps >= 0.f))) ||
        !aligned(q_norm, 16) || !aligned(k_norm, 16))
        return B200Q_EINVAL;
    if (rows == 0) return B200Q_OK;
    AppendArgs a = {};
    a.q = q; a.k = k; a.v = v; a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.rows = rows; a.hq = hq; a.hkv = kv->hkv;
    a.kp = (__nv_bfloat16*)kv->k_pages; a.vp = (__nv_bfloat16*)kv->v_pages; a.k_stride = kv->k_stride; a.v_stride = kv->v_stride;
    a.pages = kv->pages; a.page_log2 = log2_of(kv->page);
    a.s = kv_seqs(*kv);
    a.inv_freq = inv_freq; a.rope = rope; a.q_norm = q_norm; a.k_norm = k_norm; a.norm_dtype = norm_dtype; a.eps = eps;
    a.qo = (__nv_bfloat16*)q_out; a.ldo = ldo;
    const cudaStream_t s = (cudaStream_t)stream;
    const cudaError_t r = x_dtype == B200Q_F32
        ? (d == 128 ? launch_append<float, 128>(a, interleaved, s) : launch_append<float, 64>(a, interleaved, s))
        : (d == 128 ? launch_append<__nv_bfloat16, 128>(a, interleaved, s) : launch_append<__nv_bfloat16, 64>(a, interleaved, s));
    return status_from(r);
}
