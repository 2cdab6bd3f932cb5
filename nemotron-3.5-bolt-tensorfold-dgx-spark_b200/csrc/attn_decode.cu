// Attention of a step's few rows over a paged key/value cache (libbolt: bolt_kernels.cu:1779-2009): per row
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(cap(scale q . k_j) - m)
// over the keys it sees, in one pass over the cache with the running maximum m and sum.
//
// Bound by HBM: every key and value a row sees is read once for all rows and query heads of its kv head.  32 heads of d 128
// over 8: 64 sequences of up to 6000 keys 157 us, 6.3 TB/s; one of 262144 keys 162 us, 6.6 TB/s; one of 1000 keys 10.3 us.
//
// Work is shared as attn_line.cuh says, in units of 16 keys (within one page, since pages hold 16 or more) and one row block
// of 8 NT rows a kv head, a CTA an SM.  More than 16 rows a kv head are the tensor core's (attn_prompt.cu).
//
// A CTA is one producer warp, which walks the share and fills a ring of units by TMA (128-byte swizzle), and eight
// consumer warps, which take the ring's units in turn.  Scores are formed transposed, S^T = K Q^T: 16 keys are the rows of
// an m16n8k16 and 8 query rows its columns, so a group of 4 or 8 query heads wastes half or none of it (16 x 8 the
// other way round would waste three quarters).  The probabilities' accumulator becomes the B operand of O^T += V^T P^T by one
// 8 x 8 transpose (movmatrix) each; P is rounded to bf16 there, V's type: 2^-8 at most on weights that are summed with
// independent signs, below the output's own rounding.  m, the sum and O stay in fp32.
#include "attn_line.cuh"
#include "ring.cuh"
#include "tcgen05.cuh"

namespace b200q {

__device__ int g_attn_error;   // bit 0: a wait ran out, bit 1: a page table or length out of range, bit 2: over max_rows

int attn_error_read(int clear) {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_error, sizeof(int)) != cudaSuccess) return -1;
    if (clear) {
        const int z = 0;
        cudaMemcpyToSymbol(g_attn_error, &z, sizeof(int));
    }
    return v;
}

bool kv_tensor_map(CUtensorMap* m, const void* pages, int64_t stride, const b200q_paged& kv, int box_rows, int box_blocks) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess ||
            r != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (Encode)f;
    }();
    if (!encode) return false;
    const cuuint64_t dims[5] = {64, (cuuint64_t)kv.page, (cuuint64_t)kv.d / 64, (cuuint64_t)kv.hkv, (cuuint64_t)kv.pages};
    const cuuint64_t strides[4] = {(cuuint64_t)kv.d * 2, 128, (cuuint64_t)kv.page * kv.d * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks, 1, 1}, one[5] = {1, 1, 1, 1, 1};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(pages), dims, strides, box, one,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

namespace {

constexpr int kWarps = 8;                    // consumer warps
constexpr int kUnit = 16;                    // keys a unit
constexpr int kMinUnits = 16;                // a share is not smaller: two units a warp (one sequence of 1100 keys 10.1 us; 32: 11.7, 8: 9.5)

template <int D, int NT>
struct Shape {
    static constexpr int kRows = 8 * NT;                     // rows of a row block
    static constexpr int kBytes = kUnit * D * 4;             // a unit: K [D / 64][16][128 B], then V
    // 128 KB: 64 sequences of up to 6000 keys 161.5 us, not 156.5
    static constexpr int kStages = 192 * 1024 / kBytes;
    // A warp meets its own stages only.  Otherwise one could wait for a stage's next fill before its last has landed, and a
    // wait for the parity after next returns at once.
    static_assert(kStages % kWarps == 0 && kStages >= 2 * kWarps, "ring");
    static constexpr int kRing = kStages * kBytes;
    static constexpr int kFrags = D / 16 * NT;               // accumulator fragments (16 x 8) of a warp
    static constexpr int kJoin = NT == 1 ? kFrags : 4;       // those that a pass of the join moves
    static constexpr int kQ = kRows * D * 2, kJ = kWarps * kJoin * 512, kMix = kQ > kJ ? kQ : kJ;   // Q, then the join: one place
    static constexpr size_t kSmem = 1024 + kRing + kMix + (size_t)kWarps * kRows * 8 + kStages * 16;
};

using namespace line;

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool consumers_any(bool mine) {
    uint32_t any;
    asm volatile("{ .reg .pred p, q; setp.ne.u32 p, %1, 0; barrier.cta.red.or.pred.aligned q, 1, 256, p; selp.u32 %0, 1, 0, q; }"
                 : "=r"(any) : "r"((uint32_t)mine) : "memory");
    return any != 0;
}

// MANY: steps with several rows a sequence, which see different keys (row_again); without that code a single token's step is up to
// 1 % faster (one sequence of 1000 keys 10.3 us, not 10.4)
template <int D, int NT, bool MANY>
__global__ void __launch_bounds__((kWarps + 1) * 32, 1)
attn_rows_k(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, AttnArgs a) {
    using S = Shape<D, NT>;
    constexpr int RB = S::kRows, NS = S::kStages, kRing = S::kRing, kJoin = S::kJoin;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), ring = (raw + 1023) & ~1023u;
    uint8_t* base = smem_raw + (ring - raw);
    uint2* qs = (uint2*)(base + kRing);                                   // Q fragments [D / 16][NT][32]
    float4* jo = (float4*)(base + kRing);                                 // join: [kWarps][kJoin][32], once Q is done with
    float* jm = (float*)(base + kRing + S::kMix);                         // join: m [kWarps][RB], then sums
    float* jl = jm + kWarps * RB;
    const uint32_t full = ring + kRing + S::kMix + kWarps * RB * 8, empty = full + NS * 8;
    constexpr int kAll = (kWarps + 1) * 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < NS; i++) { tc_mbar_init(full + i * 8, 1); tc_mbar_init(empty + i * 8, 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch(&mk);
        tma_prefetch(&mv);
    }
    pdl_wait();
    pdl_trigger();

    const int nrb = (a.max_rows * a.group + RB - 1) / RB;
    Scan<RB, kUnit, 0, kAll> scan(*(typename Scan<RB, kUnit, 0, kAll>::Shared*)base, nrb);   // in the ring, before its first fill
    const long long total = scan.total(a, blockIdx.x == 0 ? &g_attn_error : nullptr);
    const int shares = (int)min((long long)gridDim.x, (total + kMinUnits - 1) / kMinUnits);
    Desc* desc = (Desc*)a.ws;
    if ((int)blockIdx.x >= shares) {
        if (tid == 0) desc[blockIdx.x].n = 0;
        return;
    }
    const Shares split(total, shares);
    const long long begin = split.start(blockIdx.x), end = split.start(blockIdx.x + 1);
    Cursor<RB, kUnit, 0> p = scan.seek(a, begin);
    tc_fence_proxy_async();
    __syncthreads();
    int ordinal = 0;   // units of the share before the piece
    bool dead = false;

    if (warp == kWarps) {
        // ---------------------------------------------------------------- producer: eight units at a time, a lane each
        // (one lane for all took 170 ns a unit, the time of 8 KB at the full rate).  A unit's stage was last that of the
        // unit NS >= 16 before it, so no lane waits for what another lane of its eight has yet to issue.
        bool bad_page = false;
        int issued = 0, tried = 0;   // behind the lane's last unit; the last whose place it waited for
        for (long long at = begin; at < end;) {
            const int skip = p.from(begin), n = p.to(end) - skip, u0 = p.s.u0 + skip;
            const int* tab = a.s.table + p.b * a.s.ldt;
            int next = 0;
            if (lane < n) next = tab[((u0 + lane) * kUnit) >> a.page_log2];
            for (int i0 = 0; i0 < n; i0 += 32) {
                const int mine = next;
                if (i0 + 32 + lane < n) next = tab[((u0 + i0 + 32 + lane) * kUnit) >> a.page_log2];   // a round ahead
#pragma unroll
                for (int k = 0; k < 32; k += kWarps) {
                    const int i = i0 + k + lane;
                    int page = __shfl_sync(~0u, mine, k + (lane & 7));
                    const int o = ordinal + i, st = Ring<NS>::stage(o);
                    const bool live = lane < kWarps && i < n && !dead;
                    if (live) tried = o;
                    if (live && !tc_mbar_wait(empty + st * 8, Ring<NS>::parity(o) ^ 1)) dead = true;
                    __syncwarp();
                    if (live && !dead) {
                        if (page < 0 || page >= a.pages) { bad_page = true; page = a.pages; }   // past the end: TMA fills zeros
                        const uint32_t dst = ring + st * S::kBytes, bar = full + st * 8;
                        const int row = ((u0 + i) * kUnit) & ((1 << a.page_log2) - 1);
                        tc_mbar_arrive_tx(bar, S::kBytes);
                        tma_kv(dst, &mk, row, p.h, page, bar);
                        tma_kv(dst + S::kBytes / 2, &mv, row, p.h, page, bar);
                        issued = o + 1;
                    }
                    dead = __any_sync(~0u, dead);
                }
            }
            ordinal += n;
            at = p.end();
            if (at < end) p.advance(a, nrb);
        }
        if (dead && lane == 0) atomicOr(&g_attn_error, 1);
        if (__any_sync(~0u, bad_page) && lane == 0) atomicOr(&g_attn_error, 2);
        // The last copy of every stage has landed before the block ends, whatever became of its readers.  Where a wait ran out, some
        // of the last eight were issued and others not.
        using R = Ring<NS>;
        auto landed = [&](int o) { tc_mbar_wait(full + R::stage(o) * 8, R::parity(o)); };
        if (!dead) {
            issued = __reduce_max_sync(~0u, issued);
            for (int o = R::oldest(issued) + lane; o < issued; o += 32) landed(o);
        } else {
            const int base = __shfl_sync(~0u, tried, 0), mine = R::last(base + lane, issued == base + lane + 1);
            for (int o = max(0, base + kWarps - NS) + lane; o < base; o += 32) landed(o);
            if (lane < kWarps && mine >= 0) landed(mine);
        }
        return;
    }

    // ---------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    const uint32_t krow = lane & 15, kchunk = lane >> 4;                              // ldmatrix: keys x 16-byte chunks
    const uint32_t vrow = (lane & 7) + ((lane >> 4) & 1) * 8, vchunk = (lane >> 3) & 1;
    const float c = a.c;
    if (tid == 0) desc[blockIdx.x].n = 0;
    for (long long at = begin; at < end;) {
        // units skip .. of the row block are this share's
        const int skip = p.from(begin), n = p.to(end) - skip, u0 = p.s.u0 + skip;
        if (n == 0 && (p.s.n > 0 || p.begin < begin)) {   // a cut that left this share nothing of the block
            at = p.end();
            if (at < end) p.advance(a, nrb);
            continue;
        }
        const bool whole_block = n == p.s.n;
        const int row0 = p.rb * RB, rows = min(RB, p.r * a.group - row0);
        // Q in fragment order: fragment (kk, nt), lane (g, t): values 16 kk + 2 t, + 1 and + 8, + 9 of row 8 nt + g
        consumers_sync();
        for (int i = tid; i < D / 16 * NT * 32; i += kWarps * 32) {
            const int l = i & 31, nt = (i >> 5) % NT, kk = (i >> 5) / NT, row = nt * 8 + (l >> 2);
            uint2 v = make_uint2(0, 0);
            if (row < rows) {
                const int rr = row0 + row, tok = a.token(rr);
                const uint32_t* src = (const uint32_t*)(a.q + (p.cu0 + tok) * a.ldq + (int64_t)(p.h * a.group + rr - tok * a.group) * D +
                                                        kk * 16 + (l & 3) * 2);
                v = make_uint2(src[0], src[4]);
            }
            qs[i] = v;
        }
        consumers_sync();
        uint2 qr[D / 16 * NT];
#pragma unroll
        for (int i = 0; i < D / 16 * NT; i++) qr[i] = qs[i * 32 + lane];
        int place[NT][2];   // positions of this lane's columns (rows 8 nt + 2 t, + 1); none: before every key
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + t * 2 + j;
                place[nt][j] = row < rows ? p.len - p.r + a.token(row0 + row) : -1;
            }
        float m[NT][2], sum[NT][2], o[D / 16][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY;
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
                for (int j = 0; j < 4; j++) o[mt][nt][j] = 0.f;
        }
        // the warp's units: ordinals congruent to it
        for (int i = (warp - ordinal) & (kWarps - 1); i < n; i += kWarps) {
            const int od = ordinal + i, st = od % NS, key0 = (u0 + i) * kUnit;
            if (!dead && !tc_mbar_wait(full + st * 8, od / NS & 1)) { dead = true; if (lane == 0) atomicOr(&g_attn_error, 1); }
            dead = __any_sync(~0u, dead);
            if (dead) continue;
            const uint32_t kt = ring + st * S::kBytes, vt = kt + S::kBytes / 2;
            bool fenced = false;
            if (key0 < p.s.lo || key0 + kUnit > p.s.hi) {
                // values that no row sees may hold anything, and 0 * NaN is NaN: they become zero
                for (int j = lane; j < kUnit * D / 8; j += 32) {
                    const int row = (j / 8) % kUnit, key = key0 + row;
                    if (key < p.s.lo || key >= p.s.hi) sts128(vt + j * 16, make_uint4(0, 0, 0, 0));
                }
                __syncwarp();
                fenced = true;
            }
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[nt][j] = 0.f;
#pragma unroll
            for (int kk = 0; kk < D / 16; kk++) {
                uint32_t k4[4];
                const uint32_t ch = 2 * kk + kchunk;
                ldsm4(k4, kt + (ch >> 3) * (kUnit * 128) + krow * 128 + (((ch & 7) ^ (krow & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const uint2 b = qr[kk * NT + nt];
                    mma(s[nt], k4, b.x, b.y);
                }
            }
            const bool whole = key0 + kUnit - 1 <= p.s.p0 && key0 > p.s.p1 - a.window;   // every row sees every key
            uint32_t pb[NT][2];
            bool moved = false;
            float scale[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                if (a.cap_in != 0.f) {
                    if (a.cap_exact) {
#pragma unroll
                        for (int j = 0; j < 4; j++) s[nt][j] = capped(s[nt][j], a.cap_in, true);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; j++) s[nt][j] = capped(s[nt][j], a.cap_in, false);
                    }
                }
                if (!whole)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int key = key0 + g + (j >> 1) * 8, at_ = place[nt][j & 1];
                        if (key > at_ || key <= at_ - a.window) s[nt][j] = -INFINITY;
                    }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float x = fmaxf(s[nt][j], s[nt][j + 2]);
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                    const float mn = fmaxf(m[nt][j], x * c), mz = mn == -INFINITY ? 0.f : mn;
                    moved |= mn > m[nt][j];
                    scale[nt][j] = ex2(m[nt][j] - mz);   // 0 for the first keys
                    m[nt][j] = mn;
                    s[nt][j] = ex2(fmaf(s[nt][j], c, -mz));
                    s[nt][j + 2] = ex2(fmaf(s[nt][j + 2], c, -mz));
                    sum[nt][j] = sum[nt][j] * scale[nt][j] + (s[nt][j] + s[nt][j + 2]);
                }
                pb[nt][0] = transpose8(pack_bf16(s[nt][0], s[nt][1]));
                pb[nt][1] = transpose8(pack_bf16(s[nt][2], s[nt][3]));
            }
            if (__any_sync(~0u, moved)) {
#pragma unroll
                for (int mt = 0; mt < D / 16; mt++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int j = 0; j < 4; j++) o[mt][nt][j] *= scale[nt][j & 1];
            }
#pragma unroll
            for (int mt = 0; mt < D / 16; mt++) {
                uint32_t v4[4];
                const uint32_t ch = 2 * mt + vchunk;
                ldsm4t(v4, vt + (ch >> 3) * (kUnit * 128) + vrow * 128 + (((ch & 7) ^ (vrow & 7)) << 4));
#pragma unroll
                for (int nt = 0; nt < NT; nt++) mma(o[mt][nt], v4, pb[nt][0], pb[nt][1]);
            }
            if (fenced) tc_fence_proxy_async();
            __syncwarp();
            if (lane == 0) tc_mbar_arrive(empty + st * 8);
        }
        ordinal += n;

        // join the warps: the maxima, then the sums and accumulators scaled to the common one, kJoin fragments a pass
        if (g == 0)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) jm[warp * RB + nt * 8 + t * 2 + j] = m[nt][j];
        consumers_sync();
        float scale[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + t * 2 + j;
                float x = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; w++) x = fmaxf(x, jm[w * RB + row]);
                scale[nt][j] = ex2(m[nt][j] - (x == -INFINITY ? 0.f : x));
                float y = sum[nt][j] * scale[nt][j];
                y += __shfl_xor_sync(~0u, y, 4);
                y += __shfl_xor_sync(~0u, y, 8);
                y += __shfl_xor_sync(~0u, y, 16);
                if (g == 0) jl[warp * RB + row] = y;
                m[nt][j] = x;
            }
        auto row_sum = [&](int row) {
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) y += jl[w * RB + row];
            return y;
        };
        float* slot = slots(a.ws) + ((size_t)blockIdx.x * 2 + (skip == 0 ? 1 : 0)) * kSlot<D, RB>;
        float check = 0.f;   // NaN once a value on its way out is not finite
#pragma unroll
        for (int pass = 0; pass < (S::kFrags + kJoin - 1) / kJoin; pass++) {
            if (pass) consumers_sync();
#pragma unroll
            for (int k = 0; k < kJoin; k++) {
                const int f = pass * kJoin + k;
                if (f >= S::kFrags) break;
                float(&v)[4] = o[f / NT][f % NT];
                jo[(warp * kJoin + k) * 32 + lane] = make_float4(v[0] * scale[f % NT][0], v[1] * scale[f % NT][1],
                                                                 v[2] * scale[f % NT][0], v[3] * scale[f % NT][1]);
            }
            consumers_sync();
            const int f = pass * kJoin + warp;
            if (warp < kJoin && f < S::kFrags) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < kWarps; w++) {
                    const float4 x = jo[(w * kJoin + warp) * 32 + lane];
                    v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
                }
                const int d0 = f / NT * 16, r0 = f % NT * 8;
                if (MANY) check = fmaf(v.x + v.y + v.z + v.w, 0.f, check);
                if (whole_block) {
                    const float l0 = row_sum(r0 + t * 2), l1 = row_sum(r0 + t * 2 + 1);
                    const float i0 = l0 == 0.f ? 0.f : 1.f / l0, i1 = l1 == 0.f ? 0.f : 1.f / l1;   // no key seen: zeros
                    const uint32_t lo = transpose8(pack_bf16(v.x * i0, v.y * i1)), hi = transpose8(pack_bf16(v.z * i0, v.w * i1));
                    if (r0 + g < rows) {
                        const int rr = row0 + r0 + g, tok = a.token(rr);
                        uint32_t* dst = (uint32_t*)(a.out + (p.cu0 + tok) * a.ldo +
                                                    (int64_t)(p.h * a.group + rr - tok * a.group) * D + d0 + t * 2);
                        dst[0] = lo;
                        dst[4] = hi;
                    }
                } else {
                    float* s0 = slot + (r0 + t * 2) * D + d0 + g;
                    s0[0] = v.x; s0[D] = v.y; s0[8] = v.z; s0[D + 8] = v.w;
                }
            }
        }
        if (!whole_block) {
            if (warp == 0 && g == 0)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) slot[RB * D + nt * 8 + t * 2 + j] = m[nt][j];
            if (tid >= 32 && tid < 32 + RB) slot[RB * D + RB + tid - 32] = row_sum(tid - 32);
            if (tid == 0 && skip == 0) {
                Desc& d = desc[blockIdx.x];
                d.n = p.last_share(split, blockIdx.x) - blockIdx.x + 1;
                d.cu0 = p.cu0; d.row0 = row0; d.nrows = rows; d.h = p.h;
            }
        }
        // rows of several tokens: see row_again
        if (MANY && p.s.p0 != p.s.p1 && __builtin_expect(consumers_any(check != 0.f), 0)) rows_again<D, RB, kUnit, 0, kWarps>(a, p, skip, skip + n, blockIdx.x);
        at = p.end();
        if (at < end) p.advance(a, nrb);
    }
}

template <int D, int NT, bool MANY>
cudaError_t launch_form(const CUtensorMap& mk, const CUtensorMap& mv, const AttnArgs& a, cudaStream_t s) {
    const size_t smem = Shape<D, NT>::kSmem;
    static SmemOptIn opted;
    cudaError_t e = opted.allow((const void*)attn_rows_k<D, NT, MANY>, smem);
    if (e != cudaSuccess) return e;
    const int ctas = min(device_sms(), kMaxShares);
    e = launch(attn_rows_k<D, NT, MANY>, dim3(ctas), dim3((kWarps + 1) * 32), smem, s, mk, mv, a);
    if (e != cudaSuccess) return e;
    return a.whole ? e : launch(join_k<D, Shape<D, NT>::kRows>, dim3(ctas, NT), dim3(256), 0, s, a);
}
template <int D, int NT>
cudaError_t launch_rows(const CUtensorMap& mk, const CUtensorMap& mv, const AttnArgs& a, cudaStream_t s) {
    return a.max_rows > 1 ? launch_form<D, NT, true>(mk, mv, a, s) : launch_form<D, NT, false>(mk, mv, a, s);
}

// Rows a kv head that this kernel takes.  From 17 on its accumulators are short of registers, and its S and PV products pay
// for every eight rows; the tensor-core kernel's step costs the same up to 128.  16 rows a kv head, this kernel against that one:
// d 128 over 4 kv heads, one sequence of 512 keys 9.7 / 16.7 us, 32 of 4096 55.0 / 63.6, 4 of 16384 34.1 / 38.3; over 8, 32 of 4096
// 101 / 100; d 64 over 4: 7.7 / 13.1, 34.3 / 47.3, 22.6 / 29.1.
constexpr int kMostRows = 16;
// Where the page table holds no more keys a sequence, and there are no more blocks than CTAs, blocks are not cut: a CTA then reads
// a block's keys alone, but nothing is joined and the second launch is saved.  (Shares are not below kMinUnits then either:
// blocks under 256 keys share CTAs.)  In a stream of calls, whole against cut, 32 heads of d 128 over 8, one sequence: 500 keys
// 7.2 / 8.1 us, 1000 keys 10.3 / 9.9; 16 sequences: 9.0 / 13.3 and 15.1 / 19.9.  From Python a call is 13.8 / 16, the host's part.
constexpr int kWholeKeys = 1024;
bool few(int hq, int hkv, int max_rows) { return (int64_t)max_rows * (hq / hkv) <= kMostRows; }
int row_tiles(int hq, int hkv, int max_rows) { return max_rows * (hq / hkv) <= 8 ? 1 : 2; }

size_t attend_ws(int hq, int hkv, int d, int max_rows) {
    if (!few(hq, hkv, max_rows)) return prompt_workspace(d, (int64_t)max_rows * (hq / hkv));
    return kMaxShares * (sizeof(Desc) + 2 * (size_t)row_tiles(hq, hkv, max_rows) * 8 * (d + 2) * sizeof(float));
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_attn_decode_workspace_bytes(int hq, int hkv, int d, int max_rows) {
    return hq <= 0 || hkv <= 0 || hq % hkv || max_rows <= 0 || max_rows > 16 ? 0 : attend_ws(hq, hkv, d, max_rows);
}

int b200q_attn_decode(const b200q_paged* kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                      int window, void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (!attn_ok(kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace) || max_rows > 16) return B200Q_EINVAL;
    const int d = kv->d;
    if (workspace_bytes < attend_ws(hq, kv->hkv, d, max_rows)) return B200Q_ENOSPACE;
    if (rows == 0) return B200Q_OK;
    AttnArgs a = attn_args(*kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace);
    if (!few(hq, kv->hkv, max_rows)) return prompt_launch(*kv, a, stream);
    a.whole = (int64_t)kv->width * kv->page <= kWholeKeys && (int64_t)kv->batch * kv->hkv <= min(device_sms(), kMaxShares);
    CUtensorMap mk, mv;
    if (!kv_tensor_map(&mk, kv->k_pages, kv->k_stride, *kv, kUnit, d / 64) ||
        !kv_tensor_map(&mv, kv->v_pages, kv->v_stride, *kv, kUnit, d / 64))
        return status_from(cudaErrorInvalidValue);
    const cudaStream_t s = (cudaStream_t)stream;
    const bool one = row_tiles(hq, kv->hkv, max_rows) == 1;
    cudaError_t e;
    if (d == 128) e = one ? launch_rows<128, 1>(mk, mv, a, s) : launch_rows<128, 2>(mk, mv, a, s);
    else e = one ? launch_rows<64, 1>(mk, mv, a, s) : launch_rows<64, 2>(mk, mv, a, s);
    return status_from(e);
}

}  // extern "C"
