// Attention of prompt chunks over a paged key/value cache on the tcgen05 tensor cores (libbolt: bolt_mma.cu:1406-1724).
//
// Work is shared as attn_line.cuh says, in steps of 128 keys and row blocks of 256 rows (row = token * group + query head of
// the group, so the heads that share keys share their loads), a CTA an SM.  A block is two tiles of 128 rows.  Per step and tile
//   S = Q K^T         tcgen05.mma m128n128k16, Q and K from shared memory, S (fp32) in 128 TMEM columns
//   P = exp2(c S - m) one warpgroup a tile, one thread a row: the row's maximum and sum need no exchange
//   O += P V          P (bf16) written over S and read as the A operand from TMEM, V from shared memory as it lies in
//                     the cache ([key][d]: N-major), O (fp32) in d columns
// While one tile's warpgroup computes its exponentials, the tensor core works on the other tile.  One thread issues all
// MMAs; they execute in that order, so S of the next keys may overwrite P of the last once PV has been issued.
//
// Where no sequence has more than 128 rows a kv head (a verify window, a short chunk), a block is 128 rows and both tiles hold
// them (narrow): one takes the even steps, the other the odd ones, and their sums are joined at the end.
//
// m is not the running maximum but, as published for attention on these tensor cores, a reference at most 2^8 below it: the
// quotient is the same for any reference that neither overflows nor loses the largest terms, and O (in TMEM) is rescaled only
// when the maximum has outgrown the reference by 2^8, a few times a row instead of every step.  Probabilities are then at most
// 2^8, a row's sum at most 2^8 n.  P is rounded to bf16 (2^-8 relative at most), the only type that multiplies V's; scores,
// sums and O stay in fp32.
//
// Bound by each tile's chain: its exponentials, its PV, its next S.  8192 tokens of 32 heads over 8, d 128 (550 GFLOP): a step
// of both tiles takes 3380 cycles, per tile 1500 for the exponentials (1024 of the special-function unit), 600 for the maximum
// and its checks, 1140 from P to the next S; the tensor pipe works 2050 of them.  460 to 560 us as the power limit leaves
// 1.4 to 1.6 GHz, 980 to 1190 TFLOPS.
#include "attn_tc.cuh"

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
using namespace attn_tc;

template <bool NARROW>
constexpr int kRows = NARROW ? kTile : 2 * kTile;
constexpr int kThreads = 384;         // two softmax warpgroups; a MMA, a TMA and two Q warps
constexpr int kOver = 2;              // what a row block costs besides its steps, in steps: its first and last step's waits
constexpr int kMinShare = 1 + kOver;  // a share is not smaller, but for the division's rest: a block of one step (4: 77 tokens 14.8 us, not 11.1)

template <int D>
struct Lay {
    static constexpr int kBytes = kTile * D * 2;              // a tile of Q, K or V: [D / 64][128][128 B]
    static constexpr int kStages = D == 128 ? 2 : 4;          // of K and of V
    static constexpr int kOut = 8 * 32 * 128;                 // a warp's 32 rows of 64 columns on their way out
    static constexpr int kBars = 4 * kStages + 11;
    static constexpr int kFirst = 128;                        // the cursor at the share's start
    static constexpr size_t kSmem = 1024 + (2 + 2 * kStages) * (size_t)kBytes + kOut + kBars * 8 + 16 + kFirst;
};

template <int D, bool NARROW>
__global__ void __launch_bounds__(kThreads, 1)
attn_prompt_k(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, AttnArgs a) {
    using L = Lay<D>;
    constexpr int ROWS = kRows<NARROW>, NS = L::kStages;
    using At = Cursor<ROWS, kKeys, kOver>;
    using Line = Scan<ROWS, kKeys, kOver, kThreads>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(smem_raw), sq = (raw + 1023) & ~1023u;
    uint8_t* base = smem_raw + (sq - raw);
    const uint32_t sk = sq + 2 * L::kBytes, sv = sk + NS * L::kBytes, sout = sv + NS * L::kBytes, bars = sout + L::kOut;
    const uint32_t kfull = bars, kempty = kfull + NS * 8, vfull = kempty + NS * 8, vempty = vfull + NS * 8;
    const uint32_t qfull = vempty + NS * 8, qempty = qfull + 8, sfull = qempty + 8, pready = sfull + 16, odone = pready + 32, drain = odone + 16;
    const uint32_t tslot = bars + L::kBars * 8;
    static_assert(sizeof(typename Line::Shared) <= L::kOut, "the scan's place");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_trigger();

    const int nrb = (int)(((int64_t)a.max_rows * a.group + ROWS - 1) / ROWS);
    Line scan(*(typename Line::Shared*)(base + (sout - sq)), nrb);
    const long long total = scan.total(a, blockIdx.x == 0 ? &g_prompt_error : nullptr);
    const int share = blockIdx.x, shares = (int)min((long long)gridDim.x, (total + kMinShare - 1) / kMinShare);
    Desc* desc = (Desc*)a.ws;
    if (share >= shares) {
        if (tid == 0) desc[share].n = 0;
        return;
    }
    const Shares split(total, shares);
    const long long begin = split.start(share), end = split.start(share + 1);
    At p = scan.seek(a, begin);
    int* again = (int*)(base + (tslot - sq) + 4);   // whether a result is not finite
    At* first = (At*)(base + (tslot - sq) + 16);
    static_assert(sizeof(At) <= L::kFirst, "the cursor's place");
    // where tile t's rows begin among the sequence's (token, head) rows
    auto tile_row = [&](const At& c, int t) { return c.rb * ROWS + (NARROW ? 0 : t * kTile); };
    // tile t's part of steps from .. to - 1 of the block (counted from the block's first), as far as its rows see keys
    auto tile_steps = [&](const At& c, int t, int from, int to, int& ja, int& jb) {
        const int row0 = tile_row(c, t), rows = min(kTile, c.r * a.group - row0);
        ja = jb = 0;
        if (rows <= 0) return;
        const int p0 = c.len - c.r + a.token(row0), p1 = c.len - c.r + a.token(row0 + rows - 1);
        const int l = max(0, p0 - a.window + 1);
        if (p1 < l) return;
        ja = max(l / kKeys - c.s.u0, from);
        jb = max(min(p1 / kKeys + 1 - c.s.u0, to), ja);
    };

    if (tid == 0) {
        for (int i = 0; i < 4 * NS; i++) tc_mbar_init(bars + i * 8, 1);
        tc_mbar_init(qfull, 2);
        tc_mbar_init(qempty, 1);
        tc_mbar_init(drain, 1);
        for (int t = 0; t < 2; t++) {
            tc_mbar_init(sfull + t * 8, 1);
            tc_mbar_init(pready + t * 16, 4);
            tc_mbar_init(pready + t * 16 + 8, 4);
            tc_mbar_init(odone + t * 8, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        tma_prefetch(&mk);
        tma_prefetch(&mv);
        desc[share].n = 0;   // unless the share ends inside a block, below
        *first = p;
        *again = 0;
    }
    if (warp == 8) tmem_take(tslot);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *(volatile uint32_t*)(base + (tslot - sq));   // S at t * 128, O at 256 + t * D
    bool dead = false;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == 9) {
            KvLoader<D, NS, At> kv{sk, sv, kfull, kempty, vfull, vempty, &mk, &mv, a};
            for (; !kv.dead;) {
                kv.block(p, p.cut(begin), p.cut(end));
                if (p.end() >= end) break;
                p.advance(a, nrb);
            }
            kv.drain(&g_prompt_error);
            dead = kv.dead;
        } else if (warp >= 10) {
            // ------------------------------------------------------------ Q, a warp a tile, once the last S of the piece before is formed
            const int t = warp - 10;
            for (int k = 0;;) {
                const int n = p.cut(end) - p.cut(begin);
                if (n) {
                    if (k > 0 && !dead && !wait_for(qempty, k - 1 & 1)) dead = true;
                    dead = __any_sync(~0u, dead);
                    const int row0 = tile_row(p, t), rows = p.r * a.group - row0;
                    load_q64<D>(a, p, row0, rows, 0, sq + t * L::kBytes);
                    load_q64<D>(a, p, row0, rows, 64, sq + t * L::kBytes);
                    q_arrived();
                    __syncwarp();
                    if (lane == 0) tc_mbar_arrive(qfull);
                    k++;
                }
                if (p.end() >= end) break;
                p.advance(a, nrb);
            }
        } else {
            // ------------------------------------------------------------ MMA.  Votes on waits that ran out cost 50 cycles each
            // here, so there is one a piece; the piece is finished without further waiting.
            int o = 0, k = 0, pr[2] = {0, 0};   // steps, pieces, P tiles so far
            auto await = [&](uint32_t bar, uint32_t parity) { dead = dead || !wait_for(bar, parity); };
            while (!dead) {
                const int from = p.cut(begin), to = p.cut(end);
                if (to > from) {
                    int ja[2], jb[2];
#pragma unroll
                    for (int t = 0; t < 2; t++) tile_steps(p, t, from, to, ja[t], jb[t]);
                    auto scores = [&](int t, int st) {
                        if (elect_one()) {
                            issue_scores<D>(tmem + t * kTile, sq + t * L::kBytes, sk + st * L::kBytes);
                            umma_commit(sfull + t * 8);
                        }
                        __syncwarp();
                    };
                    await(qfull, k & 1);
                    await(kfull + o % NS * 8, o / NS & 1);
                    __syncwarp();
                    tc_fence_after();
#pragma unroll
                    for (int t = 0; t < (NARROW ? 1 : 2); t++)
                        if (ja[t] == from && jb[t] > from) scores(t, o % NS);
                    if (elect_one()) {
                        umma_commit(kempty + o % NS * 8);
                        if (from + 1 == to) umma_commit(qempty);
                    }
                    __syncwarp();
                    for (int j = from; j < to; j++, o++) {
                        const int st = o % NS, sn = (o + 1) % NS;
                        if (NARROW && j + 1 < to) {   // the other tile's scores: its product of the step before is issued
                            await(kfull + sn * 8, (o + 1) / NS & 1);
                            __syncwarp();
                            tc_fence_after();
                            scores((j + 1 - from) & 1, sn);
                            if (elect_one()) {
                                umma_commit(kempty + sn * 8);
                                if (j + 2 == to) umma_commit(qempty);
                            }
                        }
                        await(vfull + st * 8, o / NS & 1);
                        __syncwarp();
                        clear_unseen<D>(sv + st * L::kBytes, (p.s.u0 + j) * kKeys, p.s);
#pragma unroll
                        for (int t = 0; t < 2; t++) {
                            if (NARROW ? ((j - from) & 1) == t : j >= ja[t] && j < jb[t]) {
                                const bool later = NARROW ? j - from > 1 : j > ja[t];
#pragma unroll
                                for (int half = 0; half < 2; half++) {
                                    await(pready + (t * 2 + half) * 8, pr[t] & 1);
                                    __syncwarp();
                                    tc_fence_after();
                                    if (elect_one()) {
                                        issue_values<D>(tmem + 256 + t * D, tmem + t * kTile + half * 32, sv + st * L::kBytes + half * 8192, 4,
                                                        later || half > 0);
                                        if (half) umma_commit(odone + t * 8);
                                    }
                                    __syncwarp();
                                }
                                pr[t]++;
                            }
                            if (t == 1 && elect_one()) umma_commit(vempty + st * 8);
                            if (!NARROW && t == 0 && j + 1 < to) {
                                await(kfull + sn * 8, (o + 1) / NS & 1);
                                __syncwarp();
                                tc_fence_after();
                            }
                            if (!NARROW && j + 1 >= ja[t] && j + 1 < jb[t]) scores(t, sn);
                        }
                        if (!NARROW && j + 1 < to && elect_one()) {
                            umma_commit(kempty + sn * 8);
                            if (j + 2 == to) umma_commit(qempty);
                        }
                        __syncwarp();
                    }
                    k++;
                }
                dead = __any_sync(~0u, dead);
                if (p.end() >= end) break;
                p.advance(a, nrb);
            }
            if (elect_one()) umma_commit(drain);   // every MMA issued has completed before TMEM is freed
            __syncwarp();
            if (!wait_for(drain, 0)) dead = true;
            dead = __any_sync(~0u, dead);
        }
    } else {
        // ---------------------------------------------------------------- softmax: warpgroup t, thread = row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t ts = tmem + t * kTile + ((uint32_t)quarter << 21), to_ = tmem + 256 + t * D + ((uint32_t)quarter << 21);
        const uint32_t stage = sout + warp * 4096;
        const float c = a.c;
        const uint64_t c2 = pair(c, c);
        int ns = 0;   // steps of the tile so far
        // between a piece's steps the cursor lies in shared memory: the scores take the registers
        At* kept = (At*)(base + (sout - sq) + warp * 4096);
        for (;;) {
            const int from = p.cut(begin), to = p.cut(end);
            if (to > from || (p.s.n == 0 && p.begin >= begin)) {
                int n, key0, pos, w0, w1;
                {
                    int ja, jb;
                    tile_steps(p, t, from, to, ja, jb);
                    n = NARROW ? (to - from + 1 - t) / 2 : jb - ja;
                    key0 = (p.s.u0 + (NARROW ? from + t : ja)) * kKeys;
                    const int row0 = tile_row(p, t), rows = min(kTile, p.r * a.group - row0);   // may be <= 0
                    const int mrow = min(row, max(rows, 1) - 1);   // rows that are none: like the last
                    pos = p.len - p.r + a.token(row0 + mrow);
                    w0 = __shfl_sync(~0u, pos, 0);
                    w1 = __shfl_sync(~0u, pos, 31);
                }
                if (lane == 0) *kept = p;
                __syncwarp();
                float ref = -INFINITY, sum = 0.f;   // the reference, in powers of two
                for (int i = 0; i < n; i++, ns++, key0 += NARROW ? 2 * kKeys : kKeys) {
                    if (!dead && !wait_for(sfull + t * 8, ns & 1)) dead = true;   // goes on all the same: nobody waits for long
                    __syncwarp();
                    tc_fence_after();
                    Scores s;
#pragma unroll
                    for (int j = 0; j < 4; j++) tmem_ld32(ts + j * 32, s[j]);
                    tmem_ld_wait();
                    if (a.cap_in != 0.f) cap_scores(s, ts, a);
                    mask_scores(s, key0, pos, w0, w1, a.window);
                    const float top = row_top(s) * c;
                    if (__any_sync(~0u, over_reference(top, ref))) {
                        const float now = raised(top, ref), f = ex2(ref - (now == -INFINITY ? 0.f : now));
                        ref = now;
                        sum *= f;
                        if (i > 0) {
                            if (!dead && !wait_for(odone + t * 8, ns - 1 & 1)) dead = true;
                            __syncwarp();
                            tc_fence_after();
                            rescale<D>(to_, f);
                        }
                    }
                    const float z = ref == -INFINITY ? 0.f : ref;
                    const uint64_t z2 = pair(-z, -z);
                    uint64_t acc[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                    auto hand_over = [&](int half) {   // half of P: its product may begin
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) tc_mbar_arrive(pready + (t * 2 + half) * 8);
                    };
                    row_probabilities(s, c2, z2, acc, ts, hand_over);
                    float s0, s1;
                    unpair(add2(acc[0], acc[1]), s0, s1);
                    sum += s0 + s1;
                }
                // ------------------------------------------------------------ out
                p = *kept;
                __syncwarp();
                const bool whole = from == 0 && to == p.s.n;
                const int row0 = tile_row(p, t), rows = min(kTile, p.r * a.group - row0);
                const int mrow = min(row, max(rows, 1) - 1), tok = a.token(row0 + mrow);
                float mine = 1.f;   // this tile's part of the joined row
                if (NARROW) {
                    // the tiles' references and sums, then (below) the second tile's O through shared memory
                    float2* told = (float2*)(base + (sout - sq) + 2048) + row;   // behind the first warp's cursor
                    told[t * kTile] = make_float2(ref, sum);
                    asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory");
                    const float2 r0 = told[0], r1 = told[kTile];
                    const float m = fmaxf(r0.x, r1.x), z = m == -INFINITY ? 0.f : m;
                    const float f0 = ex2(r0.x - z), f1 = ex2(r1.x - z);
                    sum = r0.y * f0 + r1.y * f1;
                    mine = t ? f1 : f0;
                    ref = r0.x != r0.x || r1.x != r1.x ? NAN : m;
                }
                const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no key seen: zeros
                const long long place = (p.cu0 + tok) * a.ldo + (int64_t)(p.h * a.group + row0 + mrow - tok * a.group) * D;
                float* slot = slots(a.ws) + ((size_t)share * 2 + (from == 0 ? 1 : 0)) * kSlot<D, ROWS>;
                float top[4] = {};   // the largest sizes of the row's results
                if (n > 0) {
                    if (!dead && !wait_for(odone + t * 8, ns - 1 & 1)) dead = true;
                    __syncwarp();
                    tc_fence_after();
                }
#pragma unroll 1
                for (int c0 = 0; c0 < D; c0 += 64) {   // 64 columns at a time
                    uint32_t v[2][32];
                    if (n > 0) {
                        tmem_ld32(to_ + c0, v[0]);
                        tmem_ld32(to_ + c0 + 32, v[1]);
                        tmem_ld_wait();
                    } else
#pragma unroll
                        for (int j = 0; j < 64; j++) v[j / 32][j % 32] = 0;
                    auto look = [&] {
#pragma unroll
                        for (int y = 0; y < 32; y++) top[y & 3] = max3(top[y & 3], fabsf(val(v[y / 16][y % 16 * 2])), fabsf(val(v[y / 16][y % 16 * 2 + 1])));
                    };
                    if (NARROW) {
                        // [16 pieces of 4 columns][128 rows]: a warp's lanes side by side
                        float4* second = (float4*)(base + (sout - sq)) + row;
                        asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory");   // what was there has been read
                        if (t == 1)
#pragma unroll
                            for (int y = 0; y < 16; y++) {
                                const uint32_t* e = &v[y / 8][y % 8 * 4];
                                second[y * kTile] = make_float4(val(e[0]) * mine, val(e[1]) * mine, val(e[2]) * mine, val(e[3]) * mine);
                            }
                        asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory");
                        if (t == 1) continue;
#pragma unroll
                        for (int y = 0; y < 16; y++) {
                            uint32_t* e = &v[y / 8][y % 8 * 4];
                            const float4 x = second[y * kTile];
                            e[0] = __float_as_uint(fmaf(val(e[0]), mine, x.x));
                            e[1] = __float_as_uint(fmaf(val(e[1]), mine, x.y));
                            e[2] = __float_as_uint(fmaf(val(e[2]), mine, x.z));
                            e[3] = __float_as_uint(fmaf(val(e[3]), mine, x.w));
                        }
                        look();
                        if (whole) {
                            if (row < rows)
#pragma unroll
                                for (int ch = 0; ch < 8; ch++) {
                                    const uint32_t* e = &v[ch / 4][ch % 4 * 8];
                                    *(uint4*)(a.out + place + c0 + ch * 8) =
                                        make_uint4(pack_bf16(val(e[0]) * inv, val(e[1]) * inv), pack_bf16(val(e[2]) * inv, val(e[3]) * inv),
                                                   pack_bf16(val(e[4]) * inv, val(e[5]) * inv), pack_bf16(val(e[6]) * inv, val(e[7]) * inv));
                                }
                            continue;
                        }
                    }
                    if (!NARROW) look();
                    if (whole) {   // through shared memory, to whole lines in the stores
#pragma unroll
                        for (int ch = 0; ch < 8; ch++) {
                            const uint32_t* e = &v[ch / 4][ch % 4 * 8];
                            uint4 w;
                            w.x = pack_bf16(val(e[0]) * inv, val(e[1]) * inv);
                            w.y = pack_bf16(val(e[2]) * inv, val(e[3]) * inv);
                            w.z = pack_bf16(val(e[4]) * inv, val(e[5]) * inv);
                            w.w = pack_bf16(val(e[6]) * inv, val(e[7]) * inv);
                            sts128(sw128(stage, lane, ch), w);
                        }
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int i = j * 4 + lane / 8, ch = lane % 8;
                            const long long to_row = __shfl_sync(~0u, place, i);
                            if (quarter * 32 + i < rows)
                                *(uint4*)(a.out + to_row + c0 + ch * 8) = *(const uint4*)(base + (sw128(stage, i, ch) - sq));
                        }
                        __syncwarp();
                    } else if (row < rows) {
                        float* dst = slot + (size_t)(NARROW ? row : t * kTile + row) * D + c0;
#pragma unroll
                        for (int y = 0; y < 16; y++)
                            *(uint4*)(dst + y * 4) =
                                make_uint4(v[y / 8][y % 8 * 4], v[y / 8][y % 8 * 4 + 1], v[y / 8][y % 8 * 4 + 2], v[y / 8][y % 8 * 4 + 3]);
                    }
                }
                // rows of several tokens: see row_again
                if (p.s.p0 != p.s.p1 && row < rows && !(max3(max3(top[0], top[1], top[2]), top[3], top[3]) < INFINITY)) *again = 1;
                tc_fence_before();   // O has been read before this tile's next P is handed over
                if (NARROW) asm volatile("barrier.cta.sync.aligned 1, 256;" ::: "memory");   // the shared places have been read
                if (!whole) {
                    if (row < rows && (!NARROW || t == 0)) {
                        const int r = NARROW ? row : t * kTile + row;
                        slot[ROWS * D + r] = ref;
                        slot[ROWS * D + ROWS + r] = sum;
                    }
                    if (tid == 0 && from == 0) {
                        Desc& d = desc[share];
                        d.n = p.last_share(split, share) - share + 1;
                        d.cu0 = p.cu0; d.row0 = p.rb * ROWS; d.nrows = min(ROWS, p.r * a.group - p.rb * ROWS); d.h = p.h;
                    }
                }
            }
            if (p.end() >= end) break;
            p.advance(a, nrb);
        }
    }
    if (__any_sync(~0u, dead) && lane == 0) atomicOr(&g_prompt_error, 1);
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        tmem_free(tmem);
    }
    if (warp < 8 && *again) {   // the share's rows once more, here where no other warp's bounded wait is for these
        p = *first;
        for (;;) {
            const int from = p.cut(begin), to = p.cut(end);
            if (to > from && p.s.p0 != p.s.p1) rows_again<D, ROWS, kKeys, kOver, 8>(a, p, from, to, share);
            if (p.end() >= end) break;
            p.advance(a, nrb);
        }
    }
}

template <int D, bool NARROW>
cudaError_t launch_prompt(const b200q_paged& kv, const AttnArgs& a, cudaStream_t s) {
    using L = Lay<D>;
    static SmemOptIn opted;
    cudaError_t e = opted.allow((const void*)attn_prompt_k<D, NARROW>, L::kSmem);
    if (e != cudaSuccess) return e;
    CUtensorMap mk, mv;
    const int piece = kv.page < kKeys ? kv.page : kKeys;
    if (!kv_tensor_map(&mk, kv.k_pages, kv.k_stride, kv, piece, 1) || !kv_tensor_map(&mv, kv.v_pages, kv.v_stride, kv, piece, 1))
        return cudaErrorInvalidValue;
    const int ctas = min(device_sms(), kMaxShares);
    e = launch(attn_prompt_k<D, NARROW>, dim3(ctas), dim3(kThreads), L::kSmem, s, mk, mv, a);
    if (e != cudaSuccess) return e;
    // blocks of under four steps are not cut: nothing to join (77 tokens 11.1 us, with the launch 14.4)
    if ((int64_t)kv.width * kv.page <= 3 * kKeys) return e;
    // 16 CTAs a cut block: all of its 128 rows at once, or half of 256 (4: the verify window below 32.5 us, not 30.9; 8 as 16, ragged prompts 78.9, not 78.6)
    return launch(join_k<D, kRows<NARROW>>, dim3(ctas, 16), dim3(256), 0, s, a);
}

}  // namespace

size_t prompt_workspace(int d, int64_t rows) {
    return kMaxShares * (sizeof(Desc) + 2 * (size_t)(rows <= kTile ? kTile : 2 * kTile) * (d + 2) * sizeof(float));
}
int prompt_launch(const b200q_paged& kv, const AttnArgs& a, void* stream) {
    const cudaStream_t s = (cudaStream_t)stream;
    // 8 verify windows of 16 tokens x 7 heads over 6000 keys: narrow 31 us, with a second tile of no rows 36
    const bool narrow = (int64_t)a.max_rows * a.group <= kTile;
    if (kv.d == 128) return status_from(narrow ? launch_prompt<128, true>(kv, a, s) : launch_prompt<128, false>(kv, a, s));
    return status_from(narrow ? launch_prompt<64, true>(kv, a, s) : launch_prompt<64, false>(kv, a, s));
}

}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_attn_prompt_workspace_bytes(int hq, int hkv, int d, int rows, int max_rows, int batch) {
    if (hq <= 0 || hkv <= 0 || hq % hkv || (d != 64 && d != 128) || rows < 0 || max_rows <= 0 || batch <= 0) return 0;
    return prompt_workspace(d, (int64_t)max_rows * (hq / hkv));
}

int b200q_attn_prompt(const b200q_paged* kv, const void* q, int64_t ldq, int rows, int hq, int max_rows, float scale, float softcap,
                      int window, void* out, int64_t ldo, void* workspace, size_t workspace_bytes, void* stream) {
    if (!attn_ok(kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace)) return B200Q_EINVAL;
    if (workspace_bytes < prompt_workspace(kv->d, (int64_t)max_rows * (hq / kv->hkv))) return B200Q_ENOSPACE;
    if (rows == 0) return B200Q_OK;
    return prompt_launch(*kv, attn_args(*kv, q, ldq, rows, hq, max_rows, scale, softcap, window, out, ldo, workspace), stream);
}

}  // extern "C"
