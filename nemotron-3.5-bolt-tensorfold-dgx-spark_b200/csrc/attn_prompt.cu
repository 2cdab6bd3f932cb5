// Attention of prompt chunks over a paged key/value cache on the tcgen05 tensor cores (the role of attn_mma_part_k /
// attn_mma2_part_k and attn_mma_comb_k, bolt_mma.cu:1406-1724), also for verify windows of many rows.
//
// Work is shared as attn_line.cuh says, in steps of 128 keys and row blocks of 128 rows a CTA.  A share is a pair of CTAs on
// an SM pair (row blocks of 256), whose tcgen05.mma.cta_group::2 take half of each K and V tile from either SM, so that a
// step's 256 rows load the keys once; or, where no sequence has more than 128 rows a kv head, one CTA.  Per step
//   S = Q K^T         Q and K from shared memory, S (fp32) in 128 TMEM columns, two buffers
//   P = exp2(c S - m) one warpgroup, one thread a row: the row's maximum and sum need no exchange
//   O += P V          P (bf16) from TMEM (two buffers), V from shared memory as it lies in the cache ([key][d]: N-major)
// The two softmax warpgroups take the steps in turn.  S of the step after next is formed as soon as its buffer has been read,
// so the tensor core never waits for the exponentials of the step at hand: the loop S -> softmax -> PV -> S, whose length
// bounds a kernel that keeps P in S's place (measured: 3280 cycles a step of 2 x 128 rows, 2400 of them MMAs), is not there.
// One thread issues all of a share's MMAs; they execute in that order.  TMEM: S 2 x 128, O d, P 2 x 64 columns.
//
// m is not the running maximum but a reference at most 2^8 below it: the quotient is the same for any reference that
// neither overflows nor loses the largest terms, and O (in TMEM) is rescaled only when the maximum has outgrown the
// reference by 2^8, a few times a row instead of every step.  Probabilities are then at most 2^8.  The reference goes from
// one warpgroup to the other through shared memory, step by step.  P is rounded to bf16 (2^-8 relative at most) for the
// product with V; scores, sums and O stay in fp32.
#include "attn_line.cuh"
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

using namespace line;

constexpr int kKeys = 128;            // keys of a step
constexpr int kTile = 128;            // rows of a CTA
constexpr int kThreads = 384;         // two softmax warpgroups; MMA, TMA and two Q warps
constexpr int kMinSteps = 4;          // a share is not smaller, unless there are CTAs for every row block
constexpr int kPoly = 2;              // of 8 pairs of exponentials, those by polynomial

template <int D, int CG>   // CG: CTAs of a share
struct Lay {
    static constexpr int kRows = kTile * CG;
    static constexpr int kQ = kTile * D * 2;                  // Q: [D / 64][128][128 B], two of them
    static constexpr int kKRows = kKeys / CG, kVCols = D / CG;   // this CTA's part of K (keys) and V (columns)
    static constexpr int kK = kKRows * D * 2;                 // K: [D / 64][kKRows][128 B]
    static constexpr int kVRow = kVCols * 2 > 128 ? 128 : kVCols * 2, kVBlocks = kVCols * 2 / kVRow;   // V: [kVBlocks][128][kVRow B]
    static constexpr int kV = kKeys * kVCols * 2;
    static constexpr int kStages = 128 * 1024 / (kK + kV);
    static constexpr int kBars = 4 * kStages + 14;
    static constexpr size_t kSmem = 1024 + 2 * kQ + kStages * (size_t)(kK + kV) + kBars * 8 + 16 + 5 * kTile * 4;
};

template <int CG>
constexpr uint32_t kIdescBf16 = (1u << 4) | (1u << 7) | (1u << 10) | (uint32_t)(CG * 128 >> 4) << 24;   // fp32 += bf16 bf16
template <int CG>
constexpr uint32_t kIdescQK = kIdescBf16<CG> | (128u >> 3) << 17;
template <int D, int CG>
constexpr uint32_t kIdescPV = kIdescBf16<CG> | (1u << 16) | ((uint32_t)D >> 3) << 17;   // B is N-major

// B operand [key][columns] (N-major): blocks of 64 columns (128-byte swizzle) or of 32 (64-byte swizzle), kKeys rows apart
// (leading offset); groups of 8 keys 8 rows apart (stride offset)
template <int ROW>
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((kKeys * ROW) >> 4) << 16;
    d |= (uint64_t)((8 * ROW) >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)(ROW == 128 ? 2 : 4) << 61;
    return d;
}
template <int CG>
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p; }"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0));
}
template <int CG>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
    else
        asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p; }"
                     ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0));
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {   // a shared address in the CTA of that rank
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// the MMAs issued so far, complete, arrive on `bar` in every CTA of the share
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CG == 1) umma_commit(bar);
    else
#pragma unroll
        for (uint32_t r = 0; r < 2; r++)
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(at_rank(bar, r)) : "memory");
}
// arrive on the leader's barrier
template <int CG>
__device__ __forceinline__ void arrive_lead(uint32_t bar, uint32_t rank) {
    if (CG == 1 || rank == 0) tc_mbar_arrive(bar);
    else asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(at_rank(bar, 0)) : "memory");
}
template <int CG>
__device__ __forceinline__ void share_sync() {   // all threads of the share
    if constexpr (CG == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
template <int CG>
__device__ __forceinline__ void tmem_take(uint32_t slot) {
    if constexpr (CG == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
}
template <int CG>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// one lane of a converged warp, as the compiler knows: MMA operands then stay in uniform registers (issued by "lane 0" an
// MMA took some 50 cycles more)
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the warpgroups' hand-over: 256 threads in all, those that arrive and those that wait
__device__ __forceinline__ void bar_arrive(int id) { asm volatile("barrier.cta.arrive.aligned %0, 256;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void bar_sync(int id) { asm volatile("barrier.cta.sync.aligned %0, 256;" ::"r"(id) : "memory"); }

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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
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
// tanh of two |u| <= 1: u times the polynomial of degree 5 in u^2 with the least relative error (6.2e-7, a Remez fit)
__device__ __forceinline__ uint64_t tanh2_small(uint64_t u) {
    const uint64_t v = mul2(u, u);
    uint64_t p = fma2(pair(-0.003067060374f, -0.003067060374f), v, pair(0.01674311422f, 0.01674311422f));
    p = fma2(p, v, pair(-0.05160567537f, -0.05160567537f));
    p = fma2(p, v, pair(0.1328143328f, 0.1328143328f));
    p = fma2(p, v, pair(-0.3332904279f, -0.3332904279f));
    p = fma2(p, v, pair(0.999999404f, 0.999999404f));
    return mul2(u, p);
}
// rows row .. of one column block `block` of page `page`, kv head `head`
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* m, int row, int block, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(m), "r"(0), "r"(row), "r"(block), "r"(head), "r"(page), "r"(bar) : "memory");
}

template <int D, int CG>
__global__ void __launch_bounds__(kThreads, 1)
attn_prompt_k(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, AttnArgs a) {
    using L = Lay<D, CG>;
    using At = Cursor<L::kRows, kKeys>;
    constexpr int NS = L::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), sq = (raw + 1023) & ~1023u;
    uint8_t* base = smem_raw + (sq - raw);
    const uint32_t sk = sq + 2 * L::kQ, sv = sk + NS * L::kK, bars = sv + NS * L::kV;
    // full: this CTA's copies, and in the leader the other CTA's word for its own; empty, sfull, pdone, drain: one commit
    const uint32_t kfull = bars, kempty = kfull + NS * 8, vfull = kempty + NS * 8, vempty = vfull + NS * 8;
    // in the leader, for its MMAs: qfull (Q warps), sfree (S read), pready (P written), ofree (O read)
    const uint32_t qfull = vempty + NS * 8, qempty = qfull + 16, sfull = qempty + 16, sfree = sfull + 16, pready = sfree + 16;
    const uint32_t pdone = pready + 16, ofree = pdone + 16, drain = ofree + 8;
    const uint32_t tslot = bars + L::kBars * 8;
    float* refs = (float*)(base + (tslot + 16 - sq));   // [128]: the reference of each row
    float* sums = refs + kTile;                          // [2][2][128]: piece parity, warpgroup
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint32_t rank = 0;
    if (CG == 2) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int share = blockIdx.x / CG, places = gridDim.x / CG;
    pdl_wait();
    pdl_trigger();

    const int nrb = (int)(((int64_t)a.max_rows * a.group + L::kRows - 1) / L::kRows);
    Scan<L::kRows, kKeys, kThreads> scan(*(typename Scan<L::kRows, kKeys, kThreads>::Shared*)base, nrb);   // in Q's place
    const long long total = scan.total(a, blockIdx.x == 0 ? &g_prompt_error : nullptr);
    const int shares = (int)min((long long)places, max((total + kMinSteps - 1) / kMinSteps, min(total, (long long)a.blocks)));
    Desc* desc = (Desc*)a.ws;
    if (share >= shares) {   // both CTAs of a pair
        if (tid == 0 && rank == 0) desc[share].n = 0;
        return;
    }
    const Shares split(total, shares);
    const long long begin = split.start(share), end = split.start(share + 1);
    At p = scan.seek(a, begin);
    // the piece of block p that is this share's: steps skip .. skip + n - 1
    auto skip_of = [&](const At& c) { return (int)(max(begin, c.begin) - c.begin); };
    auto steps_of = [&](const At& c) { return c.s.n ? (int)(min(end, c.end()) - c.begin) - skip_of(c) : 0; };

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            tc_mbar_init(kfull + i * 8, rank == 0 ? CG : 1);
            tc_mbar_init(vfull + i * 8, rank == 0 ? CG : 1);
            tc_mbar_init(kempty + i * 8, 1);
            tc_mbar_init(vempty + i * 8, 1);
        }
        for (int i = 0; i < 2; i++) {
            tc_mbar_init(qfull + i * 8, 2 * CG);
            tc_mbar_init(qempty + i * 8, 8);
            tc_mbar_init(sfull + i * 8, 1);
            tc_mbar_init(sfree + i * 8, 4 * CG);
            tc_mbar_init(pready + i * 8, 4 * CG);
            tc_mbar_init(pdone + i * 8, 1);
        }
        tc_mbar_init(ofree, 8 * CG);
        tc_mbar_init(drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    if (warp == 8) tmem_take<CG>(tslot);
    tc_fence_before();
    __syncthreads();
    share_sync<CG>();   // both CTAs' barriers exist
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)(base + (tslot - sq));
    constexpr uint32_t kO = 256, kP = 256 + D;   // TMEM columns; S at 0 and 128
    if (tid == 0 && rank == 0) desc[share].n = 0;   // unless the share ends inside a block, below

    bool dead = false;
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp >= 10) {
            // ------------------------------------------------------------ Q, a piece ahead: two warps, half of the rows each
            int k = 0;   // pieces with steps so far
            for (;;) {
                const int n = steps_of(p), buf = k & 1;
                if (n) {
                    if (k >= 2 && !dead && !tc_mbar_wait(qempty + buf * 8, (k >> 1) - 1 & 1)) dead = true;
                    const int row0 = p.rb * L::kRows + rank * kTile, rows = min(kTile, p.r * a.group - row0);
                    const uint32_t dst = sq + buf * L::kQ;
                    for (int i = (warp - 10) * (256 / D) + lane / (D / 8); i < kTile; i += 2 * (256 / D)) {
                        const int c = lane % (D / 8);
                        const uint32_t to = sw128(dst + (c >> 3) * (kTile * 128), i, c & 7);
                        if (i < rows) {
                            const int rr = row0 + i, tok = rr / a.group;
                            cp_async16(to, a.q + (p.cu0 + tok) * a.ldq + (int64_t)(p.h * a.group + rr - tok * a.group) * D + c * 8);
                        } else sts128(to, make_uint4(0, 0, 0, 0));
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    tc_fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) arrive_lead<CG>(qfull + buf * 8, rank);
                    k++;
                }
                if (p.end() >= end) break;
                p.advance(a, nrb);
            }
        } else if (warp == 9) {
            // ------------------------------------------------------------ K and V: pieces of a page, a lane each
            const int piece = min(1 << a.page_log2, 64), pieces = kKeys / piece;
            bool bad = false;
            int o = 0;   // steps so far
            for (; !dead;) {
                const int n = steps_of(p), u0 = p.s.u0 + skip_of(p);
                const int* tab = a.s.table + p.b * a.s.ldt;
                auto lookup = [&](int i) {   // lane l: piece l's page, INT_MIN where no row sees it
                    const int key = (u0 + i) * kKeys + lane * piece;
                    return i < n && lane < pieces && key < p.s.hi && key + piece > p.s.lo ? tab[key >> a.page_log2] : INT_MIN;
                };
                int next = lookup(0);
                for (int i = 0; i < n && !dead; i++, o++) {
                    int page = next;
                    next = lookup(i + 1);
                    const bool live = page != INT_MIN;
                    if (live && (page < 0 || page >= a.pages)) { bad = true; page = a.pages; }   // TMA fills zeros
                    const int st = o % NS, key = (u0 + i) * kKeys + lane * piece, row = key & ((1 << a.page_log2) - 1);
                    const uint32_t parity = (o / NS & 1) ^ 1;
                    // K: this CTA's keys
                    const int first = rank * L::kKRows / piece, own = L::kKRows / piece;
                    const bool klive = live && lane >= first && lane < first + own;
                    const unsigned kcount = __popc(__ballot_sync(~0u, klive)), vcount = __popc(__ballot_sync(~0u, live));
                    if (!tc_mbar_wait(kempty + st * 8, parity)) dead = true;
                    dead = __any_sync(~0u, dead);
                    if (dead) break;
                    if (lane == 0) tc_mbar_arrive_tx(kfull + st * 8, kcount * piece * D * 2);
                    __syncwarp();
                    if (klive)
#pragma unroll
                        for (int c = 0; c < D / 64; c++)
                            tma_rows(sk + st * L::kK + c * (L::kKRows * 128) + (lane - first) * piece * 128, &mk, row, c, p.h, page,
                                     kfull + st * 8);
                    // V: all keys, this CTA's columns
                    if (!tc_mbar_wait(vempty + st * 8, parity)) dead = true;
                    dead = __any_sync(~0u, dead);
                    if (dead) { o++; break; }
                    if (lane == 0) tc_mbar_arrive_tx(vfull + st * 8, vcount * piece * L::kVCols * 2);
                    __syncwarp();
                    if (live)
#pragma unroll
                        for (int c = 0; c < L::kVBlocks; c++)
                            tma_rows(sv + st * L::kV + c * (kKeys * L::kVRow) + lane * piece * L::kVRow, &mv, row,
                                     rank * L::kVBlocks + c, p.h, page, vfull + st * 8);
                }
                if (p.end() >= end) break;
                p.advance(a, nrb);
            }
            // every commit on this CTA's barriers has landed (and so every copy) before the block ends
            for (int i = max(0, o - NS) + lane; i < o; i += 32) {
                if (!tc_mbar_wait(kempty + (i % NS) * 8, i / NS & 1)) dead = true;
                if (!tc_mbar_wait(vempty + (i % NS) * 8, i / NS & 1)) dead = true;
            }
            dead = __any_sync(~0u, dead);
            if (__any_sync(~0u, bad) && lane == 0) atomicOr(&g_prompt_error, 2);
        } else {
            // ------------------------------------------------------------ MMA (leader), or the word for this CTA's copies
            // values that no row sees may hold anything, and 0 * NaN is NaN: they become zero
            auto clear_unseen = [&](int key0, int st, const Span& s) {
                if (key0 >= s.lo && key0 + kKeys <= s.hi) return;
                for (int i = lane; i < L::kV / 16; i += 32) {
                    const int key = key0 + i / (L::kVRow / 16) % kKeys;
                    if (key < s.lo || key >= s.hi) sts128(sv + st * L::kV + i * 16, make_uint4(0, 0, 0, 0));
                }
                tc_fence_proxy_async();
                __syncwarp();
            };
            if (rank == 0) {
                // S runs two steps ahead of PV, into the next piece too (its Q is there), but not past that: the Q after
                // next waits for this piece's end.  A cursor each.
                At q = p;
                int so = 0, si = 0, sn = steps_of(q), sp = 0;   // S: ordinal, step of its piece, its steps; pieces with steps before
                bool more = true;
                auto issue_s = [&](int upto, int piece) {   // the steps below `upto`, in pieces up to `piece`
                    while (so < upto && !dead) {
                        while (more && si >= sn) {   // to the next piece with steps
                            if (sn) sp++;
                            if (q.end() >= end) { more = false; break; }
                            q.advance(a, nrb);
                            si = 0;
                            sn = steps_of(q);
                        }
                        if (!more || sp > piece) return;
                        const int st = so % NS, x = so & 1, buf = sp & 1;
                        if (si == 0 && !tc_mbar_wait(qfull + buf * 8, sp >> 1 & 1)) dead = true;
                        if (!tc_mbar_wait(kfull + st * 8, so / NS & 1)) dead = true;
                        if (so >= 2 && !tc_mbar_wait(sfree + x * 8, (so >> 1) - 1 & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) return;
                        tc_fence_after();
                        const uint64_t qd = umma_desc_sw128(sq + buf * L::kQ), kd = umma_desc_sw128(sk + st * L::kK);
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < D / 16; k++)
                                umma_ss<CG>(tmem + x * 128, qd + (((k / 4) * (kTile * 128) + (k % 4) * 32) >> 4),
                                            kd + (((k / 4) * (L::kKRows * 128) + (k % 4) * 32) >> 4), kIdescQK<CG>, k > 0);
                            commit<CG>(sfull + x * 8);
                            commit<CG>(kempty + st * 8);
                        }
                        __syncwarp();
                        so++;
                        si++;
                    }
                };
                int o = 0, k = 0;
                for (; !dead;) {
                    const int n = steps_of(p), u0 = p.s.u0 + skip_of(p);
                    for (int i = 0; i < n && !dead; i++, o++) {
                        const int st = o % NS, x = o & 1;
                        issue_s(o + 3, k + 1);
                        if (!dead && !tc_mbar_wait(vfull + st * 8, o / NS & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) break;
                        clear_unseen((u0 + i) * kKeys, st, p.s);
                        if (i == 0 && k > 0 && !tc_mbar_wait(ofree, k - 1 & 1)) dead = true;
                        if (!tc_mbar_wait(pready + x * 8, o >> 1 & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) break;
                        tc_fence_after();
                        const uint64_t vd = desc_v<L::kVRow>(sv + st * L::kV);
                        if (elect_one()) {
#pragma unroll
                            for (int kk = 0; kk < kKeys / 16; kk++)
                                umma_ts<CG>(tmem + kO, tmem + kP + x * 64 + kk * 8, vd + kk * ((16 * L::kVRow) >> 4), kIdescPV<D, CG>,
                                            i > 0 || kk > 0);
                            commit<CG>(pdone + x * 8);
                            commit<CG>(vempty + st * 8);
                        }
                        __syncwarp();
                    }
                    if (n) k++;
                    if (p.end() >= end) break;
                    p.advance(a, nrb);
                }
                if (elect_one()) commit<CG>(drain);   // every MMA issued
                __syncwarp();
            } else {
                int o = 0;
                for (; !dead;) {
                    const int n = steps_of(p), u0 = p.s.u0 + skip_of(p);
                    for (int i = 0; i < n; i++, o++) {
                        const int st = o % NS;
                        if (!tc_mbar_wait(kfull + st * 8, o / NS & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) break;
                        if (lane == 0) arrive_lead<CG>(kfull + st * 8, rank);
                        if (!tc_mbar_wait(vfull + st * 8, o / NS & 1)) dead = true;
                        dead = __any_sync(~0u, dead);
                        if (dead) break;
                        clear_unseen((u0 + i) * kKeys, st, p.s);
                        if (lane == 0) arrive_lead<CG>(vfull + st * 8, rank);
                    }
                    if (p.end() >= end) break;
                    p.advance(a, nrb);
                }
            }
            if (!tc_mbar_wait(drain, 0)) dead = true;
            dead = __any_sync(~0u, dead);
        }
    } else {
        // ---------------------------------------------------------------- softmax: warpgroup x takes the steps of parity x
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int x = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;   // thread = row of the CTA
        const uint32_t lanes = (uint32_t)quarter << 21;
        const uint32_t ts = tmem + x * 128 + lanes, tp = tmem + kP + x * 64 + lanes, to = tmem + kO + lanes;
        const float c = a.c;
        const uint64_t c2 = pair(c, c);
        int o = 0, k = 0;
        for (;;) {
            const int skip = skip_of(p), n = steps_of(p), u0 = p.s.u0 + skip;
            const int row0 = p.rb * L::kRows + rank * kTile, rows = min(kTile, p.r * a.group - row0);   // of this CTA; may be <= 0
            const int p0 = p.len - p.r + row0 / a.group, p1 = p.len - p.r + (row0 + max(rows, 1) - 1) / a.group;
            const int pos = row < rows ? p.len - p.r + (row0 + row) / a.group : p1;   // rows that are none: like the last
            float ref = -INFINITY, sum = 0.f;   // the reference, in powers of two; the sum by it of this warpgroup's steps
            bool settled = false;               // every row of the warp has a reference
            const int o0 = o;
            o += n;
            for (int os = o0 + ((o0 ^ x) & 1); os < o; os += 2) {
                const int i = os - o0, key0 = (u0 + i) * kKeys;
                if (!dead && !tc_mbar_wait(sfull + x * 8, os >> 1 & 1)) dead = true;
                dead = __any_sync(~0u, dead);
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int j = 0; j < 4; j++) tmem_ld32(ts + j * 32, s[j]);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_lead<CG>(sfree + x * 8, rank);
                if (a.cap_in != 0.f) {
                    // |scale q.k / cap| <= 1 nearly always: no special function then
                    float far = 0.f;
#pragma unroll
                    for (int j = 0; j < kKeys; j += 2)
                        far = max3(far, fabsf(__uint_as_float(s[j / 32][j % 32])), fabsf(__uint_as_float(s[j / 32][j % 32 + 1])));
                    if (__any_sync(~0u, !(far * a.cap_in <= 1.f))) {
#pragma unroll
                        for (int j = 0; j < kKeys; j++) s[j / 32][j % 32] = __float_as_uint(capped(__uint_as_float(s[j / 32][j % 32]), a.cap_in));
                    } else {
                        const uint64_t in2 = pair(a.cap_in, a.cap_in);
#pragma unroll
                        for (int j = 0; j < kKeys; j += 2) {
                            float lo, hi;
                            unpair(tanh2_small(mul2(pair(__uint_as_float(s[j / 32][j % 32]), __uint_as_float(s[j / 32][j % 32 + 1])), in2)), lo, hi);
                            s[j / 32][j % 32] = __float_as_uint(lo);
                            s[j / 32][j % 32 + 1] = __float_as_uint(hi);
                        }
                    }
                }
                const bool part = key0 + kKeys - 1 > p0 || key0 <= p1 - a.window;   // some row does not see some key
                if (part) {
                    const int last = pos - key0, first = last - a.window;
#pragma unroll
                    for (int j = 0; j < kKeys; j++)
                        if (j > last || j <= first) s[j / 32][j % 32] = 0xff800000u;
                }
                float m[4];
#pragma unroll
                for (int j = 0; j < 4; j++) m[j] = max3(__uint_as_float(s[j][0]), __uint_as_float(s[j][1]), __uint_as_float(s[j][2]));
#pragma unroll
                for (int y = 3; y < 31; y += 2)
#pragma unroll
                    for (int j = 0; j < 4; j++) m[j] = max3(m[j], __uint_as_float(s[j][y]), __uint_as_float(s[j][y + 1]));
#pragma unroll
                for (int j = 0; j < 4; j++) m[j] = max3(m[j], m[j], __uint_as_float(s[j][31]));
                const float top = max3(max3(m[0], m[1], m[2]), m[3], m[3]) * c;
                if (i > 0) {   // the reference that the other warpgroup's step left
                    bar_sync(1 + x);
                    const float now = refs[row];
                    if (__any_sync(~0u, now != ref)) {
                        sum *= ex2(ref - (now == -INFINITY ? 0.f : now));
                        ref = now;
                        settled = !__any_sync(~0u, ref == -INFINITY);
                    }
                }
                const bool over = __any_sync(~0u, !(top <= ref + 8.f));
                float f = 1.f;
                if (over) {
                    // an infinite or NaN score makes its row NaN: by the reference, since ex2_poly does not carry NaN
                    const float now = top <= ref + 8.f ? ref : top < INFINITY ? top : NAN;
                    f = ex2(ref - (now == -INFINITY ? 0.f : now));
                    ref = now;
                    sum *= f;
                    settled = !__any_sync(~0u, ref == -INFINITY);
                }
                if (i + 1 < n) {
                    refs[row] = ref;
                    bar_arrive(1 + (x ^ 1));
                }
                if (over && i > 0) {
                    // O holds the steps before by the old reference; the next product waits for this step's P
                    if (!dead && !tc_mbar_wait(pdone + (x ^ 1) * 8, (os - 1) >> 1 & 1)) dead = true;
                    dead = __any_sync(~0u, dead);
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < D / 16; j++) {
                        uint32_t v[16];
                        tmem_ld16(to + j * 16, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int y = 0; y < 16; y++) v[y] = __float_as_uint(__uint_as_float(v[y]) * f);
                        tmem_st16(to + j * 16, v);
                    }
                }
                // P's buffer: the product two steps ago has read it
                if (os >= 2 && !dead && !tc_mbar_wait(pdone + x * 8, (os >> 1) - 1 & 1)) dead = true;
                dead = __any_sync(~0u, dead);
                tc_fence_after();
                const float z = ref == -INFINITY ? 0.f : ref;
                const uint64_t z2 = pair(-z, -z);
                uint64_t acc[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                auto exps = [&](bool all) {   // all: a key that is not seen counts nothing at all, so none by ex2_poly
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        uint32_t v[16];
#pragma unroll
                        for (int y = 0; y < 16; y++) {
                            const uint64_t e = fma2(pair(__uint_as_float(s[j][2 * y]), __uint_as_float(s[j][2 * y + 1])), c2, z2);
                            float e0, e1;
                            if (all || y * kPoly % 8 < 8 - kPoly) {
                                unpair(e, e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                            } else ex2_poly(e, e0, e1);
                            acc[y & 1] = add2(acc[y & 1], pair(e0, e1));
                            v[y] = pack_bf16(e0, e1);
                        }
                        tmem_st16(tp + j * 16, v);
                    }
                };
                if (part || !settled) exps(true); else exps(false);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_lead<CG>(pready + x * 8, rank);
                float s0, s1;
                unpair(add2(acc[0], acc[1]), s0, s1);
                sum += s0 + s1;
            }
            // ------------------------------------------------------------ out: each warpgroup half of the columns
            const bool whole = p.begin >= begin && p.end() <= end;
            if (n > 0) {
                // the sums of both warpgroups by the last step's reference; refs holds it once its warpgroup has written it
                if (((o - 1) & 1) == x) refs[row] = ref;
                float* mine = sums + ((k & 1) * 2) * kTile;
                bar_sync(3);
                const float last = refs[row], z = last == -INFINITY ? 0.f : last;
                mine[x * kTile + row] = sum * ex2(ref - z);
                bar_sync(3);
                sum = mine[row] + mine[kTile + row];
                ref = last;
                if (!dead && !tc_mbar_wait(pdone + ((o - 1) & 1) * 8, (o - 1) >> 1 & 1)) dead = true;
                dead = __any_sync(~0u, dead);
                tc_fence_after();
            }
            const uint32_t stage = sq + (k & 1) * L::kQ;   // Q's tile, whose MMAs are done
            float* slot = slots(a.ws) + ((size_t)share * 2 + (p.begin >= begin ? 1 : 0)) * kSlot<D, L::kRows>;
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no key seen: zeros
            const int col0 = x * (D / 2);
#pragma unroll
            for (int j = 0; j < D / 32; j++) {   // 16 columns at a time
                uint32_t v[16];
                if (n > 0) { tmem_ld16(to + col0 + j * 16, v); tmem_ld_wait(); }
                else
#pragma unroll
                    for (int y = 0; y < 16; y++) v[y] = 0;
                if (whole) {
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        uint4 w;
                        w.x = pack_bf16(__uint_as_float(v[y * 8]) * inv, __uint_as_float(v[y * 8 + 1]) * inv);
                        w.y = pack_bf16(__uint_as_float(v[y * 8 + 2]) * inv, __uint_as_float(v[y * 8 + 3]) * inv);
                        w.z = pack_bf16(__uint_as_float(v[y * 8 + 4]) * inv, __uint_as_float(v[y * 8 + 5]) * inv);
                        w.w = pack_bf16(__uint_as_float(v[y * 8 + 6]) * inv, __uint_as_float(v[y * 8 + 7]) * inv);
                        const int ch = col0 / 8 + j * 2 + y;
                        if (n > 0) sts128(sw128(stage + (ch >> 3) * (kTile * 128), row, ch & 7), w);
                        else if (row < rows) {
                            const int rr = row0 + row, tok = rr / a.group;
                            *(uint4*)(a.out + (p.cu0 + tok) * a.ldo + (int64_t)(p.h * a.group + rr - tok * a.group) * D + ch * 8) = w;
                        }
                    }
                } else if (row < rows) {
                    float* dst = slot + (size_t)(rank * kTile + row) * D + col0 + j * 16;
#pragma unroll
                    for (int y = 0; y < 4; y++) *(uint4*)(dst + y * 4) = make_uint4(v[y * 4], v[y * 4 + 1], v[y * 4 + 2], v[y * 4 + 3]);
                }
            }
            if (n > 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_lead<CG>(ofree, rank);
                if (whole) {   // whole lines out of Q's tile
                    constexpr int kLanes = D / 16;   // lanes of half a row
                    for (int i = quarter * 32 + lane / kLanes; i < quarter * 32 + 32; i += 32 / kLanes) {
                        const int ch = x * kLanes + lane % kLanes;
                        if (i < rows) {
                            const int rr = row0 + i, tok = rr / a.group;
                            const uint32_t off = sw128(stage + (ch >> 3) * (kTile * 128), i, ch & 7);
                            *(uint4*)(a.out + (p.cu0 + tok) * a.ldo + (int64_t)(p.h * a.group + rr - tok * a.group) * D + ch * 8) =
                                *(const uint4*)(base + (off - sq));
                        }
                    }
                    __syncwarp();
                }
                if (lane == 0) tc_mbar_arrive(qempty + (k & 1) * 8);
                k++;
            }
            if (!whole) {
                if (x == 0 && row < rows) {
                    slot[L::kRows * D + rank * kTile + row] = ref;
                    slot[L::kRows * D + L::kRows + rank * kTile + row] = sum;
                }
                if (tid == 0 && rank == 0 && p.begin >= begin) {
                    Desc& d = desc[share];
                    d.n = split.of(p.end() - 1) - share + 1;
                    d.cu0 = p.cu0; d.row0 = p.rb * L::kRows; d.nrows = min(L::kRows, p.r * a.group - p.rb * L::kRows); d.h = p.h;
                }
            }
            if (p.end() >= end) break;
            p.advance(a, nrb);
        }
    }
    if (dead && lane == 0) atomicOr(&g_prompt_error, 1);
    tc_fence_before();
    __syncthreads();
    share_sync<CG>();   // neither CTA leaves while the other may still arrive on its barriers
    if (warp == 8) {
        tc_fence_after();
        tmem_free<CG>(tmem);
    }
}

template <int D, int CG>
cudaError_t launch_prompt(const b200q_paged& kv, const AttnArgs& args, cudaStream_t s) {
    using L = Lay<D, CG>;
    auto kernel = attn_prompt_k<D, CG>;
    static SmemOptIn opted;
    cudaError_t e = opted.allow((const void*)kernel, L::kSmem);
    if (e != cudaSuccess) return e;
    CUtensorMap mk, mv;
    const int piece = kv.page < 64 ? kv.page : 64;
    if (!kv_tensor_map(&mk, kv.k_pages, kv.k_stride, kv, piece, 1, 64) ||
        !kv_tensor_map(&mv, kv.v_pages, kv.v_stride, kv, piece, 1, L::kVRow / 2))
        return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = CG;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CG == 1 ? 1 : 2;
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = s;
    int places = min(device_sms(), kMaxShares);
    if (CG == 2) {   // pairs that can be resident at once
        static std::atomic<int> resident[64];
        int dev = 0;
        if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
        dev = dev < 64 ? dev : 0;
        places = resident[dev].load();
        if (!places) {
            cfg.gridDim = dim3(2);
            cudaLaunchConfig_t probe = cfg;
            probe.attrs = at + 1;
            probe.numAttrs = 1;
            if ((e = cudaOccupancyMaxActiveClusters(&places, kernel, &probe)) != cudaSuccess) return e;
            places = places < 1 ? 1 : min(places, kMaxShares);
            resident[dev].store(places);
        }
    }
    AttnArgs a = args;
    // row blocks, at most: fewer shares than that would put one block after another though there are SMs
    const int64_t by_rows = (int64_t)a.rows * a.group / L::kRows + a.s.batch;
    const int64_t by_seq = a.s.batch * (((int64_t)a.max_rows * a.group + L::kRows - 1) / L::kRows);
    a.blocks = (int)min((by_rows < by_seq ? by_rows : by_seq) * a.hkv, (int64_t)INT_MAX);
    cfg.gridDim = dim3((unsigned)(places * CG));
    e = cudaLaunchKernelEx(&cfg, kernel, mk, mv, a);
    if (e != cudaSuccess) return e;
    return launch(join_k<D, L::kRows>, dim3((unsigned)places, L::kRows / 32), dim3(256), 0, s, a);
}

}  // namespace

// shared with the decode form, whose wide row blocks come here
size_t prompt_workspace(int d) {
    return kMaxShares * (sizeof(line::Desc) + 2 * (size_t)256 * (d + 2) * sizeof(float));
}
int prompt_launch(const b200q_paged& kv, const AttnArgs& a, void* stream) {
    const cudaStream_t s = (cudaStream_t)stream;
    const bool one = (int64_t)a.max_rows * a.group <= kTile;
    if (kv.d == 128) return status_from(one ? launch_prompt<128, 1>(kv, a, s) : launch_prompt<128, 2>(kv, a, s));
    return status_from(one ? launch_prompt<64, 1>(kv, a, s) : launch_prompt<64, 2>(kv, a, s));
}

}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_attn_prompt_workspace_bytes(int hq, int hkv, int d, int rows, int max_rows, int batch) {
    if (hq <= 0 || hkv <= 0 || hq % hkv || (d != 64 && d != 128) || rows < 0 || max_rows <= 0 || batch <= 0) return 0;
    return prompt_workspace(d);
}

int b200q_attn_prompt(const b200q_paged* kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                      int window, void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (!attn_ok(kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace)) return B200Q_EINVAL;
    if (workspace_bytes < prompt_workspace(kv->d)) return B200Q_ENOSPACE;
    if (rows == 0) return B200Q_OK;
    return prompt_launch(*kv, attn_args(*kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace), stream);
}

}  // extern "C"
