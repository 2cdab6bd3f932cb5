// How the paged attention kernels share their work, whatever the lengths on the device are.
//
// A row block is up to ROWS rows (row = token * group + query head of the group) of one (sequence, kv head).  The keys that
// its rows see are cut into units of UNIT; the units of all row blocks stand in one line (sequence, kv head, row block in
// order), and each share of the grid takes an equal stretch of it.  A row block cut by a share's end leaves its partial
// sums in the workspace, and a second small kernel joins them in the line's order, so results do not depend on timing.
#pragma once
#include "attn.cuh"

namespace b200q {
namespace line {

constexpr int kMaxShares = 160;   // shares the workspace holds

struct Desc {   // what a share left to join: n partials of rows row0 .. of a sequence starting at row cu0, kv head h
    int n, cu0, row0, nrows, h, pad[3];
};
// a partial: O [rows][d], m [rows] (in powers of two), sum [rows]; share c's slot 2 c + 1 holds a row block's first, 2 c
// one that began in an earlier share
template <int D, int ROWS>
constexpr size_t kSlot = (size_t)ROWS * (D + 2);
template <int D, int ROWS>
constexpr size_t kWorkspace = kMaxShares * (sizeof(Desc) + 2 * kSlot<D, ROWS> * sizeof(float));
__device__ __forceinline__ float* slots(void* ws) { return (float*)((uint8_t*)ws + kMaxShares * sizeof(Desc)); }

// a row block's keys: units u0 .. u0 + n - 1 hold every key that one of its rows sees
struct Span {
    int u0, n, lo, hi, p0, p1;   // keys lo .. hi - 1; positions of its first and last row
};
template <int ROWS, int UNIT>
__device__ __forceinline__ bool row_block(const AttnArgs& a, int r, int len, int rb, Span& s) {
    const int first = rb * ROWS, all = r * a.group;
    if (first >= all) return false;
    const int last = min(first + ROWS, all) - 1;
    s.p0 = len - r + a.token(first);
    s.p1 = len - r + a.token(last);
    s.hi = max(s.p1 + 1, 0);
    s.lo = min(max(0, s.p0 - a.window + 1), s.hi);
    s.u0 = s.lo / UNIT;
    s.n = s.hi > s.lo ? (s.hi + UNIT - 1) / UNIT - s.u0 : 0;
    return true;
}
// A block's length on the line: its units (one where it sees no key: it still writes zeros) and OVER for what a block costs
// whatever its units.
template <int OVER>
__device__ __forceinline__ int cost_of(const Span& s) { return max(s.n, 1) + OVER; }

__device__ __forceinline__ void seq_sizes(const AttnArgs& a, int b, int& cu0, int& r, int& len) {
    cu0 = min(max(a.s.cu[b], 0), a.rows);
    r = min(max(a.s.cu[b + 1], cu0), a.rows) - cu0;
    len = min(max(a.s.lens[b], 0), a.s.width << a.page_log2);
}

// shares of per or per + 1 units
struct Shares {
    long long per;
    int more;   // the first `more` shares have one unit more
    __device__ __forceinline__ Shares(long long total, int n) {
        per = total < (1ll << 32) ? (long long)((unsigned)total / (unsigned)n) : total / n;
        more = (int)(total - per * n);
    }
    __device__ __forceinline__ long long start(int k) const { return per * k + min(k, more); }
    __device__ __forceinline__ int of(long long at) const {   // the share that holds position `at`
        int k = (int)(at < (1ll << 32) ? (unsigned)at / (unsigned)(per + 1) : at / (per + 1));
        while (start(k + 1) <= at) k++;
        return k;
    }
};

// Where a share stands on the line: a row block (b, h, rb), its keys, the line's position where it begins.  Every method is
// called by whole warps, all lanes alike.
template <int ROWS, int UNIT, int OVER>
struct Cursor {
    int b, h, rb, cu0, r, len;
    Span s;
    long long begin;
    bool whole;
    __device__ __forceinline__ int cost() const { return cost_of<OVER>(s); }
    __device__ __forceinline__ long long end() const { return begin + cost(); }
    // The units of the block before the line's position `at`.  Whole: all or none.  Without OVER no cut leaves fewer than four
    // units on a side, and shares have eight or more: a piece of its own costs 3900 cycles, eight units more 1250 (one sequence
    // of 1000 keys, 15.75 units a share: 9200 cycles, not 13400).  With OVER a block of under four units is not cut, and no cut
    // leaves one side without a unit; shares of two or more then have one unit at least of every block cut twice.
    __device__ __forceinline__ int cut(long long at) const {
        if (at <= begin) return 0;
        if (at >= end()) return s.n;
        const int rel = (int)(at - begin);
        if (OVER == 0) return s.n < 8 || whole ? (2 * rel < s.n ? 0 : s.n) : rel < 4 ? 0 : rel > s.n - 4 ? s.n : rel;
        if (s.n < 4) return 2 * rel < cost() ? 0 : s.n;
        const long long part = (long long)rel * s.n;
        return min(max((int)(part < (1ll << 32) ? (unsigned)part / (unsigned)cost() : part / cost()), 1), s.n - 1);
    }
    // this share's part of the block
    __device__ __forceinline__ int from(long long share_begin) const { return cut(share_begin); }
    __device__ __forceinline__ int to(long long share_end) const { return cut(share_end); }
    // the share that holds the block's last unit, given one that holds an earlier one
    __device__ __forceinline__ int last_share(const Shares& split, int share) const {
        int k = split.of(end() - 1);
        while (k > share && cut(split.start(k)) == s.n) k--;
        return k;
    }
    __device__ __forceinline__ bool block(const AttnArgs& a, int nrb) {
        return rb < nrb && row_block<ROWS, UNIT>(a, r, len, rb, s);
    }
    // to sequence b's block that holds the line's position `at`: b starts at `first`, each of its heads has a_head units
    __device__ __forceinline__ void seek(const AttnArgs& a, int nrb, long long first, long long a_head, long long at) {
        const long long rest = at - first;
        h = a_head < (1 << 21) ? (int)((unsigned)rest / (unsigned)a_head) : (int)(rest / a_head);   // below 2^31: <= 1024 heads
        begin = first + h * a_head;
        if (nrb <= 4) {
            for (rb = 0; block(a, nrb) && at >= end(); rb++) begin = end();
            return;
        }
        const int lane = threadIdx.x & 31;
        for (int rb0 = 0;; rb0 += 32) {   // 32 blocks at a time, a lane each
            rb = rb0 + lane;
            const int c = block(a, nrb) ? cost() : 0;
            int sum = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(~0u, sum, o);
                if (lane >= o) sum += v;
            }
            const unsigned past = __ballot_sync(~0u, at < begin + sum);
            if (past) {
                const int f = __ffs(past) - 1;
                begin += __shfl_sync(~0u, sum - c, f);
                rb = rb0 + f;
                block(a, nrb);
                return;
            }
            const int all = __shfl_sync(~0u, sum, 31);
            if (!all) return;   // not reached: the position lies in this head
            begin += all;
        }
    }
    __device__ __forceinline__ void advance(const AttnArgs& a, int nrb) {
        begin = end();
        rb++;
        if (block(a, nrb)) return;
        rb = 0;
        if (++h == a.hkv) {
            h = 0;
            do seq_sizes(a, ++b, cu0, r, len);
            while (r == 0);
        }
        block(a, nrb);
    }
};

// The line's units in all and, once a share's start is known, the cursor at it: an exclusive sum over the sequences, by each
// warp for itself where they are 32 or fewer (500 cycles less before the first load), else block-wide, THREADS at a time.
template <int ROWS, int UNIT, int OVER, int THREADS>
struct Scan {
    struct Shared {
        long long warp_sum[THREADS / 32], units[THREADS], start[2];   // start: units before the share's first sequence, a head's
        int seq[4];                                                    // that sequence and its sizes
    };
    Shared& sh;
    long long units, below;   // of sequence b0 + thread (each warp: b0 + lane): those of a head, those of the sequences before
    int cu0, r, len, nrb;
    __device__ __forceinline__ bool alone(const AttnArgs& a) const { return a.s.batch <= 32 && nrb <= 4; }
    __device__ __forceinline__ Scan(Shared& shared, int nrb_) : sh(shared), units(0), below(0), cu0(0), r(0), len(0), nrb(nrb_) {}

    __device__ __forceinline__ long long round(const AttnArgs& a, int b0, long long carry, int* error) {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = alone(a) ? lane : b0 + tid;
        units = 0;
        if (b < a.s.batch) {
            seq_sizes(a, b, cu0, r, len);
            if (error && (r > a.max_rows || len != a.s.lens[b])) atomicOr(error, r > a.max_rows ? 4 : 2);
        }
        Span s;
        if (nrb <= 4) {
            if (b < a.s.batch)
                for (int rb = 0; rb < nrb && row_block<ROWS, UNIT>(a, r, len, rb, s); rb++) units += cost_of<OVER>(s);
        } else {   // a warp a sequence, a lane a block
            __syncthreads();
            for (int i = warp; i < THREADS && b0 + i < a.s.batch; i += THREADS / 32) {
                int c0, ri, li;
                seq_sizes(a, b0 + i, c0, ri, li);
                long long u = 0;
                for (int rb = lane; rb < nrb && row_block<ROWS, UNIT>(a, ri, li, rb, s); rb += 32) u += cost_of<OVER>(s);
#pragma unroll
                for (int o = 16; o; o >>= 1) u += __shfl_xor_sync(~0u, u, o);
                if (lane == 0) sh.units[i] = u;
            }
            __syncthreads();
            if (b < a.s.batch) units = sh.units[tid];
        }
        long long sum = units * a.hkv;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long v = __shfl_up_sync(~0u, sum, o);
            if (lane >= o) sum += v;
        }
        if (alone(a)) {
            below = sum - units * a.hkv;
            return __shfl_sync(~0u, sum, 31);
        }
        __syncthreads();   // the sums of the round before have been read
        if (lane == 31) sh.warp_sum[warp] = sum;
        __syncthreads();
        below = carry + sum - units * a.hkv;
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) below += sh.warp_sum[w];
            carry += sh.warp_sum[w];
        }
        return carry;
    }
    __device__ __forceinline__ long long total(const AttnArgs& a, int* error) {
        long long carry = 0;
        for (int b0 = 0; b0 < a.s.batch; b0 += THREADS) carry = round(a, b0, carry, error);
        return carry;
    }
    // after total()
    __device__ __forceinline__ Cursor<ROWS, UNIT, OVER> seek(const AttnArgs& a, long long at) {
        long long carry = 0;
        Cursor<ROWS, UNIT, OVER> p;
        p.whole = a.whole;
        if (alone(a)) {
            const int from = __ffs(__ballot_sync(~0u, units > 0 && below <= at && at < below + units * a.hkv)) - 1;
            p.b = from;
            p.cu0 = __shfl_sync(~0u, cu0, from); p.r = __shfl_sync(~0u, r, from); p.len = __shfl_sync(~0u, len, from);
            p.seek(a, nrb, __shfl_sync(~0u, below, from), __shfl_sync(~0u, units, from), at);
            return p;
        }
        for (int b0 = 0; b0 < a.s.batch; b0 += THREADS) {
            if (a.s.batch > THREADS) carry = round(a, b0, carry, nullptr);   // else the round just made holds it
            if (units > 0 && below <= at && at < below + units * a.hkv) {
                sh.start[0] = below; sh.start[1] = units;
                sh.seq[0] = b0 + threadIdx.x; sh.seq[1] = cu0; sh.seq[2] = r; sh.seq[3] = len;
            }
        }
        __syncthreads();
        p.b = sh.seq[0]; p.cu0 = sh.seq[1]; p.r = sh.seq[2]; p.len = sh.seq[3];
        p.seek(a, nrb, sh.start[0], sh.start[1], at);
        return p;
    }
};

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *(uint32_t*)&v;
}

// ---------------------------------------------------------------------------------------------------------
// Infinite and NaN values.  The products multiply every value of a tile with every row's probability, and 0 times such a value
// is NaN: the value of a later token of the row block, or of one that has left a row's window, spoils rows that do not see it.
// (Values that no row of the block sees are cleared before; the rows of one token see the same keys.)  So where a result of rows
// of several tokens is not finite, the columns that such a value spoilt are added up again, key by key, by a warp a row.  Found
// by the size of the results on their way out; that and the code cost steps of several tokens 1 to 3 %, the shortest 5 (77 tokens
// 10.6 -> 11.1 us).  Looking through the values instead, by the MMA warp or an idle one, cost 2 to 17 %.  A key takes a row 250 ns:
// 8192 tokens of which the last holds NaN 54 ms, not 0.5.
// ---------------------------------------------------------------------------------------------------------
// The row at `pos` with query q: of the keys key0 .. key1 - 1, the share's part of a block with keys lo .. hi - 1, those that it
// sees.  The result lies in out (bf16, a whole block) or part (fp32, a partial by reference ref).  Columns that the row's own
// scores, or values that it sees, make NaN stay as they are.  Lanes hold D / 32 columns each: short code, since code between
// the loops costs time although it is not run.
template <int D>
__device__ __forceinline__ void row_again(const AttnArgs& a, int lo, int hi, const int* tab, int h, int pos, int key0, int key1,
                                          const __nv_bfloat16* q, __nv_bfloat16* out, float* part, float ref) {
    constexpr int V = D / 32, kAtOnce = 4;
    const int lane = threadIdx.x & 31, d0 = lane * V;
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < V; j++) bad |= (uint32_t)!(fabsf(out ? __bfloat162float(out[d0 + j]) : part[d0 + j]) < INFINITY) << j;
    if (!__any_sync(~0u, bad)) return;
    auto load = [&](const __nv_bfloat16* pages, int64_t stride, int key, float (&x)[V]) {   // zeros where the table names no page
        const int page = tab[key >> a.page_log2];
        uint32_t w[V / 2] = {};
        if (page >= 0 && page < a.pages) {
            const __nv_bfloat16* at = pages + page * stride + (((int64_t)h << a.page_log2) + (key & ((1 << a.page_log2) - 1))) * D + d0;
#pragma unroll
            for (int j = 0; j < V / 2; j++) w[j] = ((const uint32_t*)at)[j];
        }
#pragma unroll
        for (int j = 0; j < V; j++) x[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    };
    const int first = max(0, pos - a.window + 1);   // the row sees keys first .. pos
    uint32_t taint = 0;                             // columns in which a key that it does not see holds such a value
#pragma unroll 1
    for (int k = max(lo, key0); k < min(hi, key1); k++) {
        if (k >= first && k <= pos) k = pos;
        else {
            float v[V];
            load(a.vp, a.v_stride, k, v);
#pragma unroll
            for (int j = 0; j < V; j++) taint |= (uint32_t)!(fabsf(v[j]) < INFINITY) << j;
        }
    }
    bad &= taint;
    float x[V], acc[V] = {}, m = -INFINITY, sum = 0.f;   // sum: of every kAtOnce-th key, in the first lanes
#pragma unroll
    for (int j = 0; j < V; j++) x[j] = __bfloat162float(q[d0 + j]);
    const int end = min(pos + 1, key1);
#pragma unroll 1
    for (int k0 = max(first, key0); k0 < end; k0 += kAtOnce) {
        uint32_t left = bad;   // columns not NaN by a value that the row sees: those stay so
#pragma unroll
        for (int j = 0; j < V; j++) left &= ~((uint32_t)(acc[j] != acc[j]) << j);
        if (!__any_sync(~0u, left)) return;
        float k[kAtOnce][V], v[kAtOnce][V], mine = 0.f;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            load(a.kp, a.k_stride, min(k0 + i, end - 1), k[i]);
            load(a.vp, a.v_stride, min(k0 + i, end - 1), v[i]);
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            float y = 0.f;
#pragma unroll
            for (int j = 0; j < V; j++) y = fmaf(x[j], k[i][j], y);
#pragma unroll
            for (int o = 16; o; o >>= 1) y += __shfl_xor_sync(~0u, y, o);
            if (lane == i) mine = y;
        }
        // lane i: key i's exponent and probability
        if (a.cap_in != 0.f) mine = capped(mine, a.cap_in, a.cap_exact);
        mine = lane < kAtOnce && k0 + lane < end ? mine * a.c : -INFINITY;
        float top = mine;
#pragma unroll
        for (int o = 1; o < kAtOnce; o <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        top = fmaxf(m, __shfl_sync(~0u, top, 0));
        const float z = top == -INFINITY ? 0.f : top, f = ex2(m - z), e = ex2(mine - z);
        m = top;
        sum = sum * f + e;
#pragma unroll
        for (int j = 0; j < V; j++) acc[j] *= f;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const float p = __bfloat162float(__float2bfloat16_rn(__shfl_sync(~0u, e, i)));   // as the products take it
            if (k0 + i < end)
#pragma unroll
                for (int j = 0; j < V; j++) acc[j] = fmaf(p, v[i][j], acc[j]);
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    const float f = !out ? (m == -INFINITY ? 0.f : ex2(m - ref)) : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < V; j++)
        if (bad >> j & 1) {
            if (out) out[d0 + j] = __float2bfloat16_rn(acc[j] * f);
            else part[d0 + j] = acc[j] * f;
        }
}
// Rows row, row + WARPS .. of the share's part of the block at p (units from .. to - 1), by this warp
template <int D, int ROWS, int UNIT, int OVER, int WARPS>
__device__ __forceinline__ void rows_again(const AttnArgs& a, const Cursor<ROWS, UNIT, OVER>& p, int from, int to, int share) {
    const bool whole = from == 0 && to == p.s.n;
    float* slot = slots(a.ws) + ((size_t)share * 2 + (from == 0 ? 1 : 0)) * kSlot<D, ROWS>;
    const int row0 = p.rb * ROWS, rows = min(ROWS, p.r * a.group - row0);
#pragma unroll 1
    for (int row = threadIdx.x >> 5; row < rows; row += WARPS) {
        const int rr = row0 + row, tok = a.token(rr);
        const int64_t of_head = (int64_t)(p.h * a.group + rr - tok * a.group) * D;
        row_again<D>(a, p.s.lo, p.s.hi, a.s.table + p.b * a.s.ldt, p.h, p.len - p.r + tok, (p.s.u0 + from) * UNIT, (p.s.u0 + to) * UNIT,
                     a.q + (p.cu0 + tok) * a.ldq + of_head, whole ? a.out + (p.cu0 + tok) * a.ldo + of_head : nullptr, slot + row * D,
                     whole ? 0.f : slot[ROWS * D + row]);
    }
}

// The row blocks that a share's end cut: partial 0 is the share's last, the others the first of the shares after it.
// blockIdx.y takes every gridDim.y-th set of rows.  A row's partials are dealt to as many of the eight warps as rows leave
// it, their sums added in warp order.
template <int D, int ROWS>
__global__ void __launch_bounds__(256, 4) join_k(AttnArgs a) {
    constexpr int V = D / 32, kAhead = 8;
    __shared__ float weight[8][kMaxShares], part[8][D];
    pdl_wait();
    pdl_trigger();
    const Desc d = ((const Desc*)a.ws)[blockIdx.x];
    if (d.n <= 0) return;
    const float* all = slots(a.ws);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    auto slot = [&](int i) { return all + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kSlot<D, ROWS>; };
    const int most = (int)min((long long)ROWS, (long long)a.max_rows * a.group);
    const int each = most >= 5 ? 1 : most >= 3 ? 2 : most == 2 ? 4 : 8, mine = warp % each;   // warps a row
    float x[kAhead][V], m0 = 0.f, l0 = 0.f;
    auto load = [&](int r, int i0) {
#pragma unroll
        for (int k = 0; k < kAhead; k++) {
            const int i = i0 + k * each;
            if (i >= d.n) continue;
            const float* p = slot(i) + r * D + lane * V;
            if (V == 4) *(float4*)x[k] = *(const float4*)p; else *(float2*)x[k] = *(const float2*)p;
        }
    };
    for (int r0 = blockIdx.y * (8 / each); r0 < d.nrows; r0 += gridDim.y * (8 / each)) {
        const int r = r0 + warp / each;
        const bool live = r < d.nrows;
        float acc[V] = {}, sum = 0.f;
        if (live) {
            load(r, mine);   // beside the weights
            if (lane < d.n) { m0 = slot(lane)[ROWS * D + r]; l0 = slot(lane)[ROWS * D + ROWS + r]; }
            float top = lane < d.n ? m0 : -INFINITY;
            for (int i = lane + 32; i < d.n; i += 32) top = fmaxf(top, slot(i)[ROWS * D + r]);
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            const float z = top == -INFINITY ? 0.f : top;
            for (int i = lane; i < d.n; i += 32) {
                const float w = ex2((i < 32 ? m0 : slot(i)[ROWS * D + r]) - z);
                weight[warp][i] = w;
                sum += w * (i < 32 ? l0 : slot(i)[ROWS * D + ROWS + r]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
            __syncwarp();
            for (int i0 = mine; i0 < d.n; i0 += kAhead * each) {
                if (i0 != mine) load(r, i0);
#pragma unroll
                for (int k = 0; k < kAhead; k++) {
                    const int i = i0 + k * each;
                    if (i >= d.n) break;
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] = fmaf(weight[warp][i], x[k][j], acc[j]);
                }
            }
        }
        if (each > 1) {
#pragma unroll
            for (int j = 0; j < V; j++) part[warp][lane * V + j] = acc[j];
            __syncthreads();
            if (live && mine == 0)
                for (int w = 1; w < each; w++)
#pragma unroll
                    for (int j = 0; j < V; j++) acc[j] += part[warp + w][lane * V + j];
            __syncthreads();
        }
        if (live && mine == 0) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;   // no key seen: zeros
            const int rr = d.row0 + r, tok = a.token(rr);
            uint32_t* dst = (uint32_t*)(a.out + (d.cu0 + tok) * a.ldo + (int64_t)(d.h * a.group + rr - tok * a.group) * D + lane * V);
#pragma unroll
            for (int j = 0; j < V / 2; j++) dst[j] = pack_bf16(acc[2 * j] * inv, acc[2 * j + 1] * inv);
        }
        __syncwarp();
    }
}

}  // namespace line
}  // namespace b200q
