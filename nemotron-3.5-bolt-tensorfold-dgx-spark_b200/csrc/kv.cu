// Appending a step's keys and values to a paged cache (libbolt: bolt_kernels.cu:1735), with what stands
// between the q/k/v projection and the attention on the way: the RMS norm of each query and key head (optional), the
// rotation by position (optional) and the rounding to bf16.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                        per head, fp32
//   (a, c) -> (a cos t - c sin t, c cos t + a sin t)          t = position * inv_freq[i], pairs (i, i + R/2) or (2i, 2i + 1)
//
// The angle is a product of a position and an fp32 frequency, formed and reduced by 2 pi in fp64 (exact but for the
// reduction's last bits: at position 2^18 an fp32 angle would be off by up to 2^-7), then one sincosf of the remainder.
// cos and sin depend on the token alone: a warp computes its row's once for all heads it takes.
//
// Bound by HBM: every input value is read once and every output written once (bf16).  A warp takes some of a row's
// heads, two of 128 or four of 64 a load; its first batch of loads leaves before the row's place in the cache is known
// (a chain of loads of cu, lens, table), and a pair to rotate lies in one lane, so rows cost few instructions besides.
// Measured: 8192 fp32 rows of 48 heads of 128 (norm, half rotated; 302 MB) 57.8 us = 5.2 TB/s, 80 % of the measured
// copy rate; 5560 bf16 rows of 72 heads of 64 (102 MB) 23.6 us = 4.3 TB/s; one row 2.7 us.
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
// Four values as they lie in memory, and kept so while in flight; loads a batch (what 64 registers hold, four CTAs an
// SM: three CTAs, or five with spills, were 10 to 60 % slower), loads a warp (its row's place and angles are found once)
template <typename T> struct Raw;
template <> struct Raw<float> {
    typedef float4 type;
    static constexpr int kUnroll = 3, kLoads = 12;
};
template <> struct Raw<__nv_bfloat16> {
    typedef uint2 type;
    static constexpr int kUnroll = 5, kLoads = 10;
};
__device__ __forceinline__ void widen(float4 v, float* x) { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
__device__ __forceinline__ void widen(uint2 v, float* x) {
    x[0] = __uint_as_float(v.x << 16);
    x[1] = __uint_as_float(v.x & 0xffff0000u);
    x[2] = __uint_as_float(v.y << 16);
    x[3] = __uint_as_float(v.y & 0xffff0000u);
}
template <typename T>
__device__ __forceinline__ typename Raw<T>::type raw4(const T* p) { return *(const typename Raw<T>::type*)p; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, const float* x) {
    __nv_bfloat162 o[2] = {__floats2bfloat162_rn(x[0], x[1]), __floats2bfloat162_rn(x[2], x[3])};   // the cache's type
    *(uint2*)p = *(uint2*)o;
}

// the sequence that row t belongs to (batch if none), by the whole warp: the count of range ends at or before t
__device__ __forceinline__ int row_sequence(const KvSeqs& s, int t, int lane) {
    int b = 0;
    for (int j = lane; j - lane < s.batch; j += 32) b += __popc(__ballot_sync(~0u, j < s.batch && s.cu[j + 1] <= t));
    return b;
}

template <typename T, int D, bool INTERLEAVED>
__global__ void __launch_bounds__(kAppendWarps * 32, 4) kv_append_k(AppendArgs a, int parts) {
    pdl_wait();
    constexpr int kLanes = D / 8, kHeads = 32 / kLanes, U = Raw<T>::kUnroll;   // lanes of a head, heads of a load
    __shared__ alignas(16) float2 angles[kAppendWarps][D / 2];   // read two at a time
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t task = (int64_t)blockIdx.x * kAppendWarps + warp;
    const int t = (int)(task / parts), part = (int)(task - (int64_t)t * parts);
    if (t >= a.rows) { pdl_trigger(); return; }
    // This lane's eight values of a head: in the rotated part four and their four partners, so that a pair never leaves
    // its lane, elsewhere (and where pairs stand side by side) eight in a row.
    const int sub = lane / kLanes, hl = lane % kLanes, half = a.rope >> 1;
    const bool turned = hl < a.rope / 8;
    const int ea = !INTERLEAVED && turned ? 4 * hl : 8 * hl, eb = !INTERLEAVED && turned ? half + 4 * hl : 8 * hl + 4;
    // loads: kHeads heads of q, of k or of v each
    const int lq = (a.hq + kHeads - 1) / kHeads, lk = (a.hkv + kHeads - 1) / kHeads, loads = lq + 2 * lk;
    auto head = [&](int l) { return (l < lq ? l : l < lq + lk ? l - lq : l - lq - lk) * kHeads + sub; };
    typename Raw<T>::type x[U][2];
    auto load = [&](int l0) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int l = l0 + u * parts, h = head(l);
            if (l >= loads || h >= (l < lq ? a.hq : a.hkv)) continue;
            const T* p = (l < lq ? (const T*)a.q + t * a.ldq : l < lq + lk ? (const T*)a.k + t * a.ldk : (const T*)a.v + t * a.ldv) + h * D;
            x[u][0] = raw4(p + ea);
            x[u][1] = raw4(p + eb);
        }
    };
    load(part);   // before the row's place is known: that is a chain of four more loads (cu, lens, table, angles)
    float freq[D / 64];
#pragma unroll
    for (int i = 0; i < D / 64; i++) freq[i] = lane + 32 * i < half ? a.inv_freq[lane + 32 * i] : 0.f;

    const int b = row_sequence(a.s, t, lane);
    if (b >= a.s.batch || t < a.s.cu[0]) { pdl_trigger(); return; }   // padding rows
    const int pos = a.s.lens[b] - a.s.cu[b + 1] + t;
    if (pos < 0) { pdl_trigger(); return; }   // more rows than tokens: no place
    const int entry = pos >> a.page_log2;
    const int page = entry < a.s.width ? a.s.table[b * a.s.ldt + entry] : -1;
    const bool stored = page >= 0 && page < a.pages;
    if (!stored && part == 0 && lane == 0) atomicOr(&g_kv_error, 1);
    const int64_t slot = (int64_t)(pos & ((1 << a.page_log2) - 1)) * D;
    float4 c0, c1;   // (cos, sin) of this lane's four angles
    if (half) {
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
            if (lane + 32 * i >= half) break;
            const double turn = (double)pos * (double)freq[i];
            const float r = (float)fma(-6.283185307179586476925, rint(turn * 0.15915494309189533577), turn);
            float2 v;
            sincosf(r, &v.y, &v.x);
            angles[warp][lane + 32 * i] = v;
        }
        __syncwarp();
        if (turned) {
            c0 = *(const float4*)&angles[warp][4 * hl];
            c1 = *(const float4*)&angles[warp][4 * hl + 2];
        }
    }

    for (int l0 = part; l0 < loads; l0 += parts * U) {
        if (l0 != part) load(l0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int l = l0 + u * parts;
            if (l >= loads) break;
            const int h = head(l);
            const bool is_q = l < lq, is_v = l >= lq + lk, live = h < (is_q ? a.hq : a.hkv);
            float y[8];
            widen(x[u][0], y);
            widen(x[u][1], y + 4);
            if (!is_v) {
                const void* w = is_q ? a.q_norm : a.k_norm;
                if (w) {
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; j++) ss = fmaf(y[j], y[j], ss);
#pragma unroll
                    for (int m = kLanes / 2; m; m >>= 1) ss += __shfl_xor_sync(~0u, ss, m);
                    const float r = rsqrtf(ss * (1.f / D) + a.eps);
                    float wv[8];
                    if (a.norm_dtype == B200Q_F32) { widen(raw4((const float*)w + ea), wv); widen(raw4((const float*)w + eb), wv + 4); }
                    else { widen(raw4((const __nv_bfloat16*)w + ea), wv); widen(raw4((const __nv_bfloat16*)w + eb), wv + 4); }
#pragma unroll
                    for (int j = 0; j < 8; j++) y[j] = y[j] * r * wv[j];
                }
                if (turned) {
                    const float c[4] = {c0.x, c0.z, c1.x, c1.z}, s[4] = {c0.y, c0.w, c1.y, c1.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int i0 = INTERLEAVED ? 2 * j : j, i1 = INTERLEAVED ? 2 * j + 1 : j + 4;
                        const float p = y[i0], q = y[i1];
                        y[i0] = p * c[j] - q * s[j];
                        y[i1] = q * c[j] + p * s[j];
                    }
                }
            }
            if (!live || (!is_q && !stored)) continue;
            __nv_bfloat16* o = is_q ? a.qo + t * a.ldo + h * D
                                    : (is_v ? a.vp + page * a.v_stride : a.kp + page * a.k_stride) + (((int64_t)h * D) << a.page_log2) + slot;
            store4(o + ea, y);
            store4(o + eb, y + 4);
        }
    }
    pdl_trigger();
}

template <typename T, int D>
static cudaError_t launch_append(const AppendArgs& a, int interleaved, cudaStream_t s) {
    constexpr int kHeads = 32 / (D / 8);
    // a row over so many warps that each has kLoads loads; with few rows more, until each has one
    const int loads = (a.hq + kHeads - 1) / kHeads + 2 * ((a.hkv + kHeads - 1) / kHeads);
    int64_t parts = (loads + Raw<T>::kLoads - 1) / Raw<T>::kLoads;
    const int64_t fill = (int64_t)device_sms() * 2 * kAppendWarps / a.rows;
    if (parts < fill) parts = fill < loads ? fill : loads;
    const dim3 grid((unsigned)(((int64_t)a.rows * parts + kAppendWarps - 1) / kAppendWarps));
    return interleaved ? launch(kv_append_k<T, D, true>, grid, dim3(kAppendWarps * 32), 0, s, a, (int)parts)
                       : launch(kv_append_k<T, D, false>, grid, dim3(kAppendWarps * 32), 0, s, a, (int)parts);
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
    // a row's heads go to several warps and batches of loads: q_out may lie on q where every value replaces itself, and nowhere
    // else on what is still to be read
    const bool in_place = q_out == q && x_dtype == B200Q_BF16 && (ldo == ldq || rows == 1);
    if (hq > 0 && ((!in_place && !rows_apart(q_out, ldo * 2, wq * 2, q, ldq * e, wq * e, rows)) ||
                   !rows_apart(q_out, ldo * 2, wq * 2, k, ldk * e, wk * e, rows) ||
                   !rows_apart(q_out, ldo * 2, wq * 2, v, ldv * e, wk * e, rows)))
        return B200Q_EINVAL;
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
