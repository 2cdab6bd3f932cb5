// Attention of prompt chunks over a paged key/value cache on the tcgen05 tensor cores (the role of attn_mma_part_k /
// attn_mma2_part_k and attn_mma_comb_k, bolt_mma.cu:1406-1724).
//
// A CTA computes 256 rows (row = token * group + query head of the group) of one (sequence, kv head), so the heads that
// share keys share their loads, as two tiles of 128 rows.  Per 128 keys and tile:
//   S = Q K^T        tcgen05.mma m128n128k16, Q and K from shared memory, S (fp32) in 128 TMEM columns
//   P = exp2(c S - m) one warpgroup a tile, one thread a row: row maximum and sum need no exchange
//   O += P V         P (bf16) written over S and read as the A operand from TMEM, V from shared memory as it lies in
//                    the cache ([key][d]: N-major), O (fp32) in d columns
// While one tile's warpgroup computes its exponentials, the tensor core works on the other tile.  One thread issues all
// MMAs; they execute in that order, so S of the next keys may overwrite P of the last once PV has been issued.
//
// m is not the running maximum but a reference at most 2^8 below it: the quotient is the same for any reference that
// neither overflows nor loses the largest terms, and O (in TMEM) is rescaled only when the maximum has outgrown the
// reference by 2^8, a few times a row instead of every 128 keys.  Probabilities are then at most 2^8, a row's sum at most
// 2^8 n.  P is rounded to bf16 (2^-8 relative at most) for the product with V; scores, sums and O stay in fp32.
//
// Bound by the tensor cores (4 d operations a visible pair) and, at d = 64, by the exponentials.
#include "attn.cuh"
#include "tcgen05.cuh"

namespace b200q {

__device__ int g_prompt_error;   // as g_attn_error in attn_decode.cu

int prompt_error_read(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_prompt_error, sizeof(int)) != cudaSuccess) return -1;
    if (clear) {
        const int z = 0;
        cudaMemcpyToSymbol(g_prompt_error, &z, sizeof(int));
    }
    return v;
}

namespace {

constexpr int kTile = 128;            // rows of a tile, keys of a step
constexpr int kRows = 2 * kTile;      // rows of a CTA
constexpr int kThreads = 384;         // two softmax warpgroups; MMA and TMA warps
constexpr int kMinSteps = 4;          // a share of a cut row block has at least so many steps of keys
constexpr int kMaxShares = 32;
constexpr int kPoly = 2;              // of 8 pairs of exponentials, those by polynomial

template <int D>
struct Lay {
    static constexpr int kBytes = kTile * D * 2;              // a tile of Q, K or V: [D / 64][128][128 B]
    static constexpr int kStages = D == 128 ? 2 : 4;          // of K and of V
    static constexpr int kBars = 4 * kStages + 11;
    static constexpr size_t kSlot = (size_t)kRows * (D + 2);  // floats of a partial: O [256][D], m [256], sum [256]
    static size_t smem(int batch) { return 1024 + (2 + 2 * kStages) * (size_t)kBytes + kBars * 8 + 16 + (size_t)(batch + 1) * 4; }
};

struct Desc {   // a cut row block: shares to join (0, 1: none), its rows
    int n, cu0, row0, nrows, h, pad[3];
};

constexpr uint32_t kIdescBf16 = (1u << 4) | (1u << 7) | (1u << 10) | (128u >> 4) << 24;   // fp32 += bf16 bf16, M = 128
constexpr uint32_t kIdescQK = kIdescBf16 | (128u >> 3) << 17;
template <int D>
constexpr uint32_t kIdescPV = kIdescBf16 | (1u << 16) | ((uint32_t)D >> 3) << 17;          // B is N-major

// B operand [key][d] (N-major), 128-byte swizzle: 64-value column blocks kTile * 128 bytes apart (leading offset), groups
// of 8 keys 1024 bytes apart (stride offset)
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((kTile * 128) >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
          "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
          "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t*)&v;
}
// one lane of a converged warp, as the compiler knows: MMA operands then stay in uniform registers
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
// two fp32 at a time
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if any is
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// 2^x for two x <= 8, without the special-function unit: x = n + f, |f| <= 1/2, and 2^f by the polynomial of degree 3
// with the least relative error there (7.5e-5 = 2^-13.7, a Remez fit; the result is rounded to bf16 next, 2^-8).  Below
// 2^-126 it stays there.  Adding 1.5 2^23 leaves n in the low bits of the sum, and n << 23 adds to the exponent.
__device__ __forceinline__ void ex2_poly(uint64_t x, float& lo, float& hi) {
    const uint64_t magic = pair(12582912.f, 12582912.f);
    float a, b;
    unpair(x, a, b);
    x = pair(fmaxf(a, -126.f), fmaxf(b, -126.f));
    const uint64_t t = add2(x, magic), n = add2(t, pair(-12582912.f, -12582912.f)), f = fma2(n, pair(-1.f, -1.f), x);
    uint64_t p = fma2(pair(0.05517166852951050f, 0.05517166852951050f), f, pair(0.24261112511157990f, 0.24261112511157990f));
    p = fma2(p, f, pair(0.69326096773147583f, 0.69326096773147583f));
    p = fma2(p, f, pair(0.99992805719375610f, 0.99992805719375610f));
    float n0, n1;
    unpair(t, n0, n1);
    unpair(p, a, b);
    lo = __uint_as_float(__float_as_uint(a) + (__float_as_uint(n0) << 23));
    hi = __uint_as_float(__float_as_uint(b) + (__float_as_uint(n1) << 23));
}
// rows row .. of one 64-value column block `chunk` of page `page`, kv head `head`
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* m, int row, int chunk, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(m), "r"(0), "r"(row), "r"(chunk), "r"(head), "r"(page), "r"(bar) : "memory");
}

struct PromptArgs {
    AttnArgs a;
    int blocks;      // row blocks of a kv head the grid holds
    int shares;      // CTAs a row block may be cut into along the keys
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
attn_prompt_k(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, PromptArgs pa) {
    using L = Lay<D>;
    constexpr int NS = L::kStages;
    const AttnArgs& a = pa.a;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int warp_sum[kThreads / 32];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), sq = (raw + 1023) & ~1023u;
    uint8_t* base = smem_raw + (sq - raw);
    const uint32_t sk = sq + 2 * L::kBytes, sv = sk + NS * L::kBytes, bars = sv + NS * L::kBytes;
    const uint32_t kfull = bars, kempty = kfull + NS * 8, vfull = kempty + NS * 8, vempty = vfull + NS * 8;
    const uint32_t qfull = vempty + NS * 8, sfull = qfull + 8, pready = sfull + 16, odone = pready + 32;   // odone [2], last
    const uint32_t tslot = bars + L::kBars * 8;
    int* pre = (int*)(base + (tslot + 16 - sq));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();

    // the row blocks of the sequences before each
    const int most = (int)(((int64_t)a.max_rows * a.group + kRows - 1) / kRows);
    int carry = 0;
    if (tid == 0) pre[0] = 0;
    for (int b0 = 0; b0 < a.s.batch; b0 += kThreads) {
        const int b = b0 + tid;
        int c = 0;
        if (b < a.s.batch) {
            const int cu0 = min(max(a.s.cu[b], 0), a.rows), r = min(max(a.s.cu[b + 1], cu0), a.rows) - cu0, len = a.s.lens[b];
            c = (int)min(((int64_t)r * a.group + kRows - 1) / kRows, (int64_t)most);
            if (blockIdx.x == 0) {
                if (r > a.max_rows) atomicOr(&g_prompt_error, 4);
                if (len < 0 || len > a.s.width << a.page_log2) atomicOr(&g_prompt_error, 2);
            }
        }
        int sum = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += v;
        }
        if (lane == 31) warp_sum[warp] = sum;
        __syncthreads();
        int below = carry;
        for (int w = 0; w < kThreads / 32; w++) {
            if (w < warp) below += warp_sum[w];
            carry += warp_sum[w];
        }
        if (b < a.s.batch) pre[b + 1] = below + sum;
        __syncthreads();
    }

    // this CTA's row block and share of its keys; the last row blocks, which see the most keys, come first
    const int share = blockIdx.x % pa.shares, place = blockIdx.x / pa.shares, h = place % a.hkv, at = place / a.hkv;
    Desc* desc = (Desc*)a.ws + place;
    const int block = carry - 1 - at;
    if (block < 0) {
        if (tid == 0 && share == 0 && pa.shares > 1) desc->n = 0;
        return;
    }
    int b = 0;
    for (int hi = a.s.batch - 1; b < hi;) {   // the last b with pre[b] <= block
        const int mid = (b + hi + 1) >> 1;
        if (pre[mid] <= block) b = mid; else hi = mid - 1;
    }
    const int cu0 = min(max(a.s.cu[b], 0), a.rows), r = min(max(a.s.cu[b + 1], cu0), a.rows) - cu0;
    const int len = min(max(a.s.lens[b], 0), a.s.width << a.page_log2);
    const int row0 = (block - pre[b]) * kRows, rows = min(kRows, r * a.group - row0), tiles = rows > kTile ? 2 : 1;
    // per tile: positions of its first and last row, the steps of 128 keys that hold what its rows see
    int p0[2], p1[2], ja[2], jb[2], lo = INT_MAX, hi = 0;
#pragma unroll
    for (int t = 0; t < 2; t++) {
        p0[t] = p1[t] = -1;
        ja[t] = jb[t] = 0;
        if (t < tiles) {
            p0[t] = len - r + (row0 + t * kTile) / a.group;
            p1[t] = len - r + (row0 + min(rows, (t + 1) * kTile) - 1) / a.group;
            const int l = max(0, p0[t] - a.window + 1), e = p1[t] + 1;
            if (e > l) {
                ja[t] = l / kTile;
                jb[t] = (e + kTile - 1) / kTile;
                lo = min(lo, l);
                hi = max(hi, e);
            }
        }
    }
    int j0 = INT_MAX, j1 = 0;
#pragma unroll
    for (int t = 0; t < 2; t++)
        if (jb[t] > ja[t]) { j0 = min(j0, ja[t]); j1 = max(j1, jb[t]); }
    if (j1 == 0) j0 = 0;
    const int steps = j1 - j0, cut = max(1, min(pa.shares, steps / kMinSteps));
    if (share == 0 && tid == 0 && pa.shares > 1) {
        desc->n = cut;
        desc->cu0 = cu0; desc->row0 = row0; desc->nrows = rows; desc->h = h;
    }
    if (share >= cut) return;
    j1 = j0 + (int)((int64_t)steps * (share + 1) / cut);
    j0 = j0 + (int)((int64_t)steps * share / cut);
#pragma unroll
    for (int t = 0; t < 2; t++) {
        ja[t] = max(ja[t], j0);
        jb[t] = max(min(jb[t], j1), ja[t]);
    }

    if (tid == 0) {
        for (int i = 0; i < 4 * NS; i++) tc_mbar_init(bars + i * 8, 1);
        tc_mbar_init(qfull, 256);
        for (int t = 0; t < 2; t++) {
            tc_mbar_init(sfull + t * 8, 1);
            tc_mbar_init(pready + t * 16, 128);
            tc_mbar_init(pready + t * 16 + 8, 128);
            tc_mbar_init(odone + t * 8, 1);
        }
        tc_mbar_init(odone + 16, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tslot), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)(base + (tslot - sq));

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 9) {
            // ------------------------------------------------------------ TMA: pieces of a page, at most 128 rows
            const int piece = min(1 << a.page_log2, kTile), pieces = kTile / piece;
            const int* tab = a.s.table + b * a.s.ldt;
            bool bad = false, dead = false;
            auto lookup = [&](int j) {   // lane i: piece i's page, -1 where no row sees it
                const int key = j * kTile + lane * piece;
                return j < j1 && lane < pieces && key < hi && key + piece > lo ? tab[key >> a.page_log2] : INT_MIN;
            };
            int next = lookup(j0), issued = 0;
            for (int j = j0; j < j1 && !dead; j++) {
                int page = next;
                next = lookup(j + 1);
                const bool live = page != INT_MIN;
                const uint32_t bytes = __popc(__ballot_sync(~0u, live)) * piece * D * 2;
                if (live && (page < 0 || page >= a.pages)) { bad = true; page = a.pages; }   // TMA fills zeros
                const int n = j - j0, st = n % NS, row = (j * kTile + lane * piece) & ((1 << a.page_log2) - 1);
#pragma unroll
                for (int side = 0; side < 2; side++) {
                    const uint32_t full = (side ? vfull : kfull) + st * 8;
                    if (!tc_mbar_wait((side ? vempty : kempty) + st * 8, (n / NS & 1) ^ 1)) dead = true;
                    dead = __any_sync(~0u, dead);
                    if (dead) break;
                    if (lane == 0) tc_mbar_arrive_tx(full, bytes);
                    __syncwarp();
                    if (live)
#pragma unroll
                        for (int c = 0; c < D / 64; c++)
                            tma_rows((side ? sv : sk) + st * L::kBytes + c * (kTile * 128) + lane * piece * 128, side ? &mv : &mk, row,
                                     c, h, page, full);
                    issued += 1;
                }
            }
            for (int i = max(0, issued - 2 * NS); i < issued; i++)   // landed before the block ends
                tc_mbar_wait((i & 1 ? vfull : kfull) + (i / 2 % NS) * 8, i / 2 / NS & 1);
            if (__any_sync(~0u, bad) && lane == 0) atomicOr(&g_prompt_error, 2);
            if (dead && lane == 0) atomicOr(&g_prompt_error, 1);
        } else if (warp == 8) {
            // ------------------------------------------------------------ MMA: lane 0 issues
            bool dead = !tc_mbar_wait(qfull, 0);
            int pr[2] = {0, 0};   // P tiles used so far
            auto scores = [&](int t, int st) {
                const uint64_t qd = umma_desc_sw128(sq + t * L::kBytes), kd = umma_desc_sw128(sk + st * L::kBytes);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < D / 16; k++) {
                        const uint32_t off = ((k / 4) * (kTile * 128) + (k % 4) * 32) >> 4;
                        umma_ss(tmem + t * kTile, qd + off, kd + off, kIdescQK, k > 0);
                    }
                    umma_commit(sfull + t * 8);
                }
                __syncwarp();
            };
            if (j0 < j1) {
                if (!dead && !tc_mbar_wait(kfull, 0)) dead = true;
                dead = __any_sync(~0u, dead);
                if (!dead) {
                    tc_fence_after();
                    for (int t = 0; t < 2; t++)
                        if (ja[t] == j0 && jb[t] > j0) scores(t, 0);
                    if (elect_one()) umma_commit(kempty);
                }
            }
            for (int j = j0; j < j1 && !dead; j++) {
                const int n = j - j0, st = n % NS, sn = (n + 1) % NS;
                if (!tc_mbar_wait(vfull + st * 8, n / NS & 1)) dead = true;
                dead = __any_sync(~0u, dead);
                if (dead) break;
                const int key0 = j * kTile;
                if (key0 < lo || key0 + kTile > hi) {
                    // values that no row sees may hold anything, and 0 * NaN is NaN: they become zero
                    for (int i = lane; i < kTile * D / 8; i += 32) {
                        const int key = key0 + i / 8 % kTile;
                        if (key < lo || key >= hi) sts128(sv + st * L::kBytes + i * 16, make_uint4(0, 0, 0, 0));
                    }
                    tc_fence_proxy_async();
                    __syncwarp();
                }
                for (int t = 0; t < 2; t++) {
                    if (j >= ja[t] && j < jb[t]) {
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            if (!tc_mbar_wait(pready + (t * 2 + half) * 8, pr[t] & 1)) dead = true;
                            dead = __any_sync(~0u, dead);
                            if (dead) break;
                            tc_fence_after();
                            const uint64_t vd = desc_v(sv + st * L::kBytes);
                            if (elect_one()) {
#pragma unroll
                                for (int k = half * 4; k < half * 4 + 4; k++)
                                    umma_ts(tmem + 256 + t * D, tmem + t * kTile + k * 8, vd + k * (2048 >> 4), kIdescPV<D>,
                                            pr[t] > 0 || k > 0);
                            }
                        }
                        if (dead) break;
                        if (elect_one()) umma_commit(odone + t * 8);
                        __syncwarp();
                        pr[t]++;
                    }
                    if (t == 1 && elect_one()) umma_commit(vempty + st * 8);
                    if (t == 0 && j + 1 < j1) {
                        if (!tc_mbar_wait(kfull + sn * 8, (n + 1) / NS & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) break;
                    }
                    if (j + 1 >= ja[t] && j + 1 < jb[t]) scores(t, sn);
                }
                if (dead) break;
                if (j + 1 < j1 && elect_one()) umma_commit(kempty + sn * 8);
                __syncwarp();
            }
            if (elect_one()) umma_commit(odone + 16);   // every MMA issued
            __syncwarp();
            tc_mbar_wait(odone + 16, 0);
            if (dead && lane == 0) atomicOr(&g_prompt_error, 1);
        }
    } else {
        // ---------------------------------------------------------------- softmax: warpgroup t, thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int t = warp >> 2, row = t * kTile + (warp & 3) * 32 + lane;   // of the block
        // Q into the swizzled tiles: a row's 16-byte pieces over the lanes of D / 8
        for (int i = (warp & 3) * (256 / D) + lane / (D / 8); i < kTile; i += 4 * (256 / D)) {
            const int ri = t * kTile + i, c = lane % (D / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (ri < rows) {
                const int rr = row0 + ri, tok = rr / a.group;
                v = *(const uint4*)(a.q + (cu0 + tok) * a.ldq + (int64_t)(h * a.group + rr - tok * a.group) * D + c * 8);
            }
            sts128(sw128(sq + t * L::kBytes + (c >> 3) * (kTile * 128), i, c & 7), v);
        }
        tc_fence_proxy_async();
        tc_mbar_arrive(qfull);

        const int n = jb[t] - ja[t];
        const uint32_t ts = tmem + t * kTile + ((uint32_t)(warp & 3) << 21), to = tmem + 256 + t * D + ((uint32_t)(warp & 3) << 21);
        const int pos = row < rows ? len - r + (row0 + row) / a.group : -1;
        const float c = a.c;
        float ref = -INFINITY, sum = 0.f;   // the reference, in powers of two
        bool dead = false;
        for (int i = 0; i < n; i++) {
            const int key0 = (ja[t] + i) * kTile;
            if (!tc_mbar_wait(sfull + t * 8, i & 1)) dead = true;
            if (__any_sync(~0u, dead)) { dead = true; break; }
            tc_fence_after();
            uint32_t s[4][32];
#pragma unroll
            for (int k = 0; k < 4; k++) tmem_ld32(ts + k * 32, s[k]);
            tmem_ld_wait();
            if (a.cap_in != 0.f)
#pragma unroll
                for (int k = 0; k < kTile; k++) s[k / 32][k % 32] = __float_as_uint(capped(__uint_as_float(s[k / 32][k % 32]), a.cap_in));
            bool exact = key0 + kTile - 1 > p0[t] || key0 <= p1[t] - a.window;   // some row does not see some key
            if (exact) {
                const int last = pos - key0, first = pos - a.window - key0;
#pragma unroll
                for (int k = 0; k < kTile; k++)
                    if (k > last || k <= first) s[k / 32][k % 32] = 0xff800000u;
            }
            float tops[4];
#pragma unroll
            for (int k = 0; k < 4; k++) tops[k] = max3(__uint_as_float(s[k][0]), __uint_as_float(s[k][1]), __uint_as_float(s[k][2]));
#pragma unroll
            for (int x = 3; x < 31; x += 2)
#pragma unroll
                for (int k = 0; k < 4; k++) tops[k] = max3(tops[k], __uint_as_float(s[k][x]), __uint_as_float(s[k][x + 1]));
#pragma unroll
            for (int k = 0; k < 4; k++) tops[k] = max3(tops[k], tops[k], __uint_as_float(s[k][31]));
            const float top = max3(max3(tops[0], tops[1], tops[2]), tops[3], tops[3]) * c;
            if (__any_sync(~0u, !(top <= ref + 8.f))) {
                // an infinite or NaN score makes its row NaN: by the reference, since ex2_poly does not carry NaN
                const float now = top <= ref + 8.f ? ref : top < INFINITY ? top : NAN, f = ex2(ref - (now == -INFINITY ? 0.f : now));
                ref = now;
                sum *= f;
                if (i > 0) {
                    if (!tc_mbar_wait(odone + t * 8, (i - 1) & 1)) dead = true;
                    if (__any_sync(~0u, dead)) { dead = true; break; }
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < D / 32; k++) {
                        uint32_t o[32];
                        tmem_ld32(to + k * 32, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 32; x++) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                        tmem_st32(to + k * 32, o);
                    }
                }
            }
            exact |= __any_sync(~0u, ref == -INFINITY);
            const float z = ref == -INFINITY ? 0.f : ref;
            const uint64_t c2 = pair(c, c), z2 = pair(-z, -z);
            uint64_t sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
            auto exps = [&](bool all) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t p[16];
#pragma unroll
                    for (int x = 0; x < 16; x++) {
                        const uint64_t e = fma2(pair(__uint_as_float(s[k][2 * x]), __uint_as_float(s[k][2 * x + 1])), c2, z2);
                        float e0, e1;
                        if (all || x * kPoly % 8 < 8 - kPoly) {
                            unpair(e, e0, e1);
                            e0 = ex2(e0);
                            e1 = ex2(e1);
                        } else ex2_poly(e, e0, e1);
                        sums[x & 1] = add2(sums[x & 1], pair(e0, e1));
                        p[x] = pack2(e0, e1);
                    }
                    tmem_st16(ts + k * 16, p);
                    if (k & 1) {   // half of P: its product may begin
                        tmem_st_wait();
                        tc_fence_before();
                        tc_mbar_arrive(pready + (t * 2 + k / 2) * 8);
                    }
                }
            };
            if (exact) exps(true); else exps(false);
            float s0, s1;
            unpair(add2(sums[0], sums[1]), s0, s1);
            sum += s0 + s1;
        }
        // ---------------------------------------------------------------- out
        if (n > 0 && !dead && !tc_mbar_wait(odone + t * 8, (n - 1) & 1)) dead = true;
        dead = __any_sync(~0u, dead);
        tc_fence_after();
        if (dead) {
            if (lane == 0) atomicOr(&g_prompt_error, 1);
        } else if (cut == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no key seen: zeros
#pragma unroll
            for (int k = 0; k < D / 32; k++) {
                uint32_t o[32];
                if (n > 0) { tmem_ld32(to + k * 32, o); tmem_ld_wait(); }
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (n > 0) {
                        v.x = pack2(__uint_as_float(o[x * 8]) * inv, __uint_as_float(o[x * 8 + 1]) * inv);
                        v.y = pack2(__uint_as_float(o[x * 8 + 2]) * inv, __uint_as_float(o[x * 8 + 3]) * inv);
                        v.z = pack2(__uint_as_float(o[x * 8 + 4]) * inv, __uint_as_float(o[x * 8 + 5]) * inv);
                        v.w = pack2(__uint_as_float(o[x * 8 + 6]) * inv, __uint_as_float(o[x * 8 + 7]) * inv);
                    }
                    const int ch = k * 4 + x;   // through Q's tile, whose MMAs are done, to whole rows in the stores
                    sts128(sw128(sq + t * L::kBytes + (ch >> 3) * (kTile * 128), row - t * kTile, ch & 7), v);
                }
            }
            __syncwarp();
            for (int i = (warp & 3) * 32 + lane / (D / 8); i < (warp & 3) * 32 + 32; i += 256 / D) {
                const int ri = t * kTile + i, ch = lane % (D / 8);
                if (ri < rows) {
                    const int rr = row0 + ri, tok = rr / a.group;
                    const uint32_t off = sw128(sq + t * L::kBytes + (ch >> 3) * (kTile * 128), i, ch & 7);
                    *(uint4*)(a.out + (cu0 + tok) * a.ldo + (int64_t)(h * a.group + rr - tok * a.group) * D + ch * 8) =
                        *(const uint4*)(base + (off - sq));
                }
            }
        } else {
            float* slot = (float*)((Desc*)a.ws + (size_t)pa.blocks * a.hkv) + (size_t)blockIdx.x * L::kSlot;
#pragma unroll
            for (int k = 0; k < D / 32; k++) {
                uint32_t o[32];
                if (n > 0) { tmem_ld32(to + k * 32, o); tmem_ld_wait(); }
#pragma unroll
                for (int x = 0; x < 8; x++)
                    *(uint4*)(slot + row * D + k * 32 + x * 4) =
                        n > 0 ? make_uint4(o[x * 4], o[x * 4 + 1], o[x * 4 + 2], o[x * 4 + 3]) : make_uint4(0, 0, 0, 0);
            }
            slot[kRows * D + row] = ref;
            slot[kRows * D + kRows + row] = sum;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// the row blocks cut along the keys: their shares' partials, in order; a warp a row
template <int D>
__global__ void __launch_bounds__(256) prompt_join_k(PromptArgs pa) {
    using L = Lay<D>;
    constexpr int V = D / 32;
    const AttnArgs& a = pa.a;
    pdl_wait();
    pdl_trigger();
    const Desc d = ((const Desc*)a.ws)[blockIdx.x];
    if (d.n <= 1) return;
    const float* slots = (const float*)((const Desc*)a.ws + (size_t)pa.blocks * a.hkv) + (size_t)blockIdx.x * pa.shares * L::kSlot;
    const int lane = threadIdx.x & 31;
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < d.nrows; r += gridDim.y * 8) {
        // lane i holds share i's (kMaxShares = 32)
        const float m = lane < d.n ? slots[lane * L::kSlot + kRows * D + r] : -INFINITY;
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float w = ex2(m - (top == -INFINITY ? 0.f : top));
        float sum = lane < d.n ? w * slots[lane * L::kSlot + kRows * D + kRows + r] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        float acc[V] = {};
#pragma unroll 4
        for (int i = 0; i < d.n; i++) {
            const float* p = slots + i * L::kSlot + r * D + lane * V;
            const float wi = __shfl_sync(~0u, w, i);
            float x[V];
            if (V == 4) *(float4*)x = *(const float4*)p; else *(float2*)x = *(const float2*)p;
#pragma unroll
            for (int j = 0; j < V; j++) acc[j] = fmaf(wi, x[j], acc[j]);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int rr = d.row0 + r, tok = rr / a.group;
        uint32_t* dst = (uint32_t*)(a.out + (d.cu0 + tok) * a.ldo + (int64_t)(d.h * a.group + rr - tok * a.group) * D + lane * V);
#pragma unroll
        for (int j = 0; j < V / 2; j++) dst[j] = pack2(acc[2 * j] * inv, acc[2 * j + 1] * inv);
    }
}

// row blocks of a kv head at most, whatever the sequences' rows on the device are; CTAs a row block is cut into
int64_t row_blocks(int group, int rows, int max_rows, int batch) {
    const int64_t by_rows = (int64_t)rows * group / kRows + batch, by_seq = batch * (((int64_t)max_rows * group + kRows - 1) / kRows);
    return by_rows < by_seq ? by_rows : by_seq;
}
int key_shares(int64_t ctas) {
    const int64_t n = device_sms() / (ctas > 0 ? ctas : 1);
    return n < 1 ? 1 : n > kMaxShares ? kMaxShares : (int)n;
}

template <int D>
cudaError_t launch_prompt(const CUtensorMap& mk, const CUtensorMap& mv, const PromptArgs& p, cudaStream_t s) {
    const size_t smem = Lay<D>::smem(p.a.s.batch);
    static SmemOptIn opted;
    cudaError_t e = opted.allow((const void*)attn_prompt_k<D>, Lay<D>::smem(4096));
    if (e != cudaSuccess) return e;
    e = launch(attn_prompt_k<D>, dim3((unsigned)(p.blocks * p.a.hkv * p.shares)), dim3(kThreads), smem, s, mk, mv, p);
    if (e != cudaSuccess || p.shares == 1) return e;
    return launch(prompt_join_k<D>, dim3((unsigned)(p.blocks * p.a.hkv), 8), dim3(256), 0, s, p);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_attn_prompt_workspace_bytes(int hq, int hkv, int d, int rows, int max_rows, int batch) {
    if (hq <= 0 || hkv <= 0 || hq % hkv || (d != 64 && d != 128) || rows < 0 || max_rows <= 0 || batch <= 0) return 0;
    const int64_t ctas = row_blocks(hq / hkv, rows, max_rows, batch) * hkv;
    const int n = key_shares(ctas);
    return n == 1 ? 16 : (size_t)ctas * (sizeof(Desc) + n * (size_t)kRows * (d + 2) * sizeof(float));
}

int b200q_attn_prompt(const b200q_paged* kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                      int window, void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (!attn_ok(kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace)) return B200Q_EINVAL;
    const int d = kv->d, hkv = kv->hkv;
    if (workspace_bytes < b200q_attn_prompt_workspace_bytes(hq, hkv, d, rows, max_rows, kv->batch)) return B200Q_ENOSPACE;
    if (rows == 0) return B200Q_OK;
    PromptArgs p = {};
    p.a = attn_args(*kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace);
    const int64_t blocks = row_blocks(p.a.group, rows, max_rows, kv->batch);
    if (blocks * hkv > (1 << 28)) return B200Q_EINVAL;
    p.blocks = (int)blocks;
    p.shares = key_shares(blocks * hkv);
    CUtensorMap mk, mv;
    const int piece = kv->page < kTile ? kv->page : kTile;
    if (!kv_tensor_map(&mk, kv->k_pages, kv->k_stride, *kv, piece, 1) || !kv_tensor_map(&mv, kv->v_pages, kv->v_stride, *kv, piece, 1))
        return status_from(cudaErrorInvalidValue);
    return status_from(d == 128 ? launch_prompt<128>(mk, mv, p, (cudaStream_t)stream) : launch_prompt<64>(mk, mv, p, (cudaStream_t)stream));
}

}  // extern "C"
