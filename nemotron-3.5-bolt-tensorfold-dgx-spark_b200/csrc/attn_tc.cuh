// Shared pieces of the paged attention kernels on the tcgen05 tensor cores: MMAs with operands in shared memory and TMEM,
// and the softmax of 128 scores of a row held by one thread.
#pragma once
#include "attn_line.cuh"
#include "ring.cuh"
#include "tcgen05.cuh"

namespace b200q {
namespace attn_tc {

using line::pack_bf16;

constexpr int kKeys = 128;   // keys of a step
constexpr int kTile = 128;   // rows of a tile

constexpr uint32_t kIdescBf16 = (1u << 4) | (1u << 7) | (1u << 10) | (128u >> 4) << 24;   // fp32 += bf16 bf16, M = 128
constexpr uint32_t kIdescQK = kIdescBf16 | (128u >> 3) << 17;
template <int D>
constexpr uint32_t kIdescPV = kIdescBf16 | (1u << 16) | ((uint32_t)D >> 3) << 17;          // B is N-major

// B operand [key][d] (N-major), 128-byte swizzle: 64-value column blocks kKeys * 128 bytes apart (leading offset), groups
// of 8 keys 1024 bytes apart (stride offset)
__device__ __forceinline__ uint64_t desc_v(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFF);
    d |= (uint64_t)((kKeys * 128) >> 4) << 16;
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
// S = Q K^T of one tile and one step, by one lane: Q [D / 64][128][128 B], K the same
template <int D>
__device__ __forceinline__ void issue_scores(uint32_t tmem_s, uint32_t q, uint32_t k) {
    const uint64_t qd = umma_desc_sw128(q), kd = umma_desc_sw128(k);
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        const uint32_t off = ((i / 4) * (kTile * 128) + (i % 4) * 32) >> 4;
        umma_ss(tmem_s, qd + off, kd + off, kIdescQK, i > 0);
    }
}
// O += P V of 16 n keys from the first of P (TMEM, 8 columns for 16 keys) and V [D / 64][128][128 B]
template <int D>
__device__ __forceinline__ void issue_values(uint32_t tmem_o, uint32_t tmem_p, uint32_t v, int n, bool accumulate) {
    const uint64_t vd = desc_v(v);
#pragma unroll
    for (int i = 0; i < n; i++) umma_ts(tmem_o, tmem_p + i * 8, vd + i * (2048 >> 4), kIdescPV<D>, accumulate || i > 0);
}
__device__ __forceinline__ void tmem_take(uint32_t slot) {   // all 512 columns, by a warp
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
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
// tc_mbar_wait, the first look without its suspend-time hint (15 cycles, not 50, where the phase is complete)
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok || tc_mbar_wait(bar, parity);
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

// ---------------------------------------------------------------------------------------------------------
// the scores of one row and 128 keys, bit patterns of fp32
// ---------------------------------------------------------------------------------------------------------
typedef uint32_t Scores[4][32];
__device__ __forceinline__ float val(uint32_t x) { return __uint_as_float(x); }

// s -> tanh(cap_in s): four packed operations two scores where all of the warp's lie below cap_near, as nearly always.
// Otherwise the special functions, in TMEM and back: unrolled over the 128 scores beside the rest, the code alone cost a tenth
// of a step that never ran it.
__device__ __forceinline__ void cap_scores(Scores& s, uint32_t tmem_s, const AttnArgs& a) {
    float m[4] = {};
#pragma unroll
    for (int y = 0; y < 32; y += 2)
#pragma unroll
        for (int j = 0; j < 4; j++) m[j] = max3(m[j], fabsf(val(s[j][y])), fabsf(val(s[j][y + 1])));
    const float far = max3(max3(m[0], m[1], m[2]), m[3], m[3]);
    if (__any_sync(~0u, !(far <= a.cap_near))) {
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
            uint32_t v[16];
            tmem_ld16(tmem_s + j * 16, v);
            tmem_ld_wait();
            if (a.cap_exact) {
#pragma unroll
                for (int y = 0; y < 16; y++) v[y] = __float_as_uint(capped(val(v[y]), a.cap_in, true));
            } else {
#pragma unroll
                for (int y = 0; y < 16; y++) v[y] = __float_as_uint(capped(val(v[y]), a.cap_in, false));
            }
            tmem_st16(tmem_s + j * 16, v);
        }
        tmem_st_wait();
#pragma unroll
        for (int j = 0; j < 4; j++) tmem_ld32(tmem_s + j * 32, s[j]);
        tmem_ld_wait();
        return;
    }
    uint64_t c[3];
#pragma unroll
    for (int k = 0; k < 3; k++) c[k] = pair(a.cap_poly[k], a.cap_poly[k]);
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int y = 0; y < 32; y += 2) {
            const uint64_t x = pair(val(s[j][y]), val(s[j][y + 1])), v = mul2(x, x);
            float lo, hi;
            unpair(mul2(x, fma2(fma2(c[2], v, c[1]), v, c[0])), lo, hi);
            s[j][y] = __float_as_uint(lo);
            s[j][y + 1] = __float_as_uint(hi);
        }
}
// Keys key0 .. key0 + 127 that the row at `pos` does not see get no part (minus infinity).  w0, w1: the positions of the
// warp's first and last row.
__device__ __forceinline__ void mask_scores(Scores& s, int key0, int pos, int w0, int w1, int window) {
    const int all = w0 - key0, any = w1 - key0;   // columns up to which all rows, some row of the warp see
    if (kKeys - 1 <= all && any - window < 0) return;
    const int last = pos - key0, first = last - window;
    auto upto = [](int j) { return j >= 31 ? ~0u : j < 0 ? 0u : (2u << j) - 1; };   // bits 0 .. j
#pragma unroll
    for (int j = 0; j < 4; j++)   // 32 columns: most are seen by all rows
        if (j * 32 + 31 > all || j * 32 <= any - window) {
            const uint32_t seen = upto(last - j * 32) & ~upto(first - j * 32);
#pragma unroll
            for (int y = 0; y < 32; y++) s[j][y] = seen & 1u << y ? s[j][y] : 0xff800000u;
        }
}
__device__ __forceinline__ float row_top(const Scores& s) {   // NaN if any is
    float m[4];
#pragma unroll
    for (int j = 0; j < 4; j++) m[j] = max3(val(s[j][0]), val(s[j][1]), val(s[j][2]));
#pragma unroll
    for (int y = 3; y < 31; y += 2)
#pragma unroll
        for (int j = 0; j < 4; j++) m[j] = max3(m[j], val(s[j][y]), val(s[j][y + 1]));
#pragma unroll
    for (int j = 0; j < 4; j++) m[j] = max3(m[j], m[j], val(s[j][31]));
    return max3(max3(m[0], m[1], m[2]), m[3], m[3]);
}
// The reference after a step whose largest exponent is `top`: raised only when it is exceeded by 2^8.  An infinite or NaN
// score makes its row NaN, by the reference.
__device__ __forceinline__ bool over_reference(float top, float ref) { return !(top <= ref + 8.f); }
__device__ __forceinline__ float raised(float top, float ref) { return !over_reference(top, ref) ? ref : top < INFINITY ? top : NAN; }
// Probabilities of 32 keys by reference z, summed in fp32 and rounded to bf16.  All by the special-function unit: a quarter of
// them by a polynomial of degree 3 relieves it, but the other pipes and the code's length gave up more (8192 tokens 490 us with
// it, 480 without; ragged prompts 81 / 78).
__device__ __forceinline__ void probabilities(const uint32_t (&s)[32], uint64_t c2, uint64_t z2, uint64_t (&acc)[2], uint32_t (&p)[16]) {
#pragma unroll
    for (int y = 0; y < 16; y++) {
        float e0, e1;
        unpair(fma2(pair(val(s[2 * y]), val(s[2 * y + 1])), c2, z2), e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        acc[y & 1] = add2(acc[y & 1], pair(e0, e1));
        p[y] = pack_bf16(e0, e1);
    }
}
// Those of the row's 128 keys to TMEM, 16 columns for 32 keys.  half(0) is called once the first 64 keys' have arrived there,
// in the shadow of the third quarter's exponentials; half(1) at the end.
template <typename F>
__device__ __forceinline__ void row_probabilities(const Scores& s, uint64_t c2, uint64_t z2, uint64_t (&acc)[2], uint32_t tmem_p, F half) {
    uint32_t p[16];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        probabilities(s[j], c2, z2, acc, p);
        if (j == 2) {
            tmem_st_wait();
            half(0);
        }
        tmem_st16(tmem_p + j * 16, p);
    }
    tmem_st_wait();
    half(1);
}
// O of the row, D columns, times f
template <int D>
__device__ __forceinline__ void rescale(uint32_t tmem_o, float f) {
#pragma unroll
    for (int j = 0; j < D / 16; j++) {
        uint32_t v[16];
        tmem_ld16(tmem_o + j * 16, v);
        tmem_ld_wait();
#pragma unroll
        for (int y = 0; y < 16; y++) v[y] = __float_as_uint(val(v[y]) * f);
        tmem_st16(tmem_o + j * 16, v);
    }
}
// values that no row sees may hold anything, and 0 * NaN is NaN: they become zero (by a warp)
template <int D>
__device__ __forceinline__ void clear_unseen(uint32_t v, int key0, const line::Span& s) {
    if (key0 >= s.lo && key0 + kKeys <= s.hi) return;
    for (int i = threadIdx.x & 31; i < kKeys * D / 8; i += 32) {
        const int key = key0 + i / 8 % kKeys;
        if (key < s.lo || key >= s.hi) sts128(v + i * 16, make_uint4(0, 0, 0, 0));
    }
    tc_fence_proxy_async();
    __syncwarp();
}
// rows row .. of one column block `block` of page `page`, kv head `head`
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* m, int row, int block, int head, int page, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(m), "r"(0), "r"(row), "r"(block), "r"(head), "r"(page), "r"(bar) : "memory");
}

// Loads of K and V by one warp: pieces of a page, a lane each.  A step's pages are looked up a step ahead.
template <int D, int NS, typename At>
struct KvLoader {
    static constexpr int kBytes = kKeys * D * 2;
    uint32_t sk, sv, kfull, kempty, vfull, vempty;
    const CUtensorMap *mk, *mv;
    const AttnArgs& a;
    int o = 0;               // steps whose copies were issued
    bool half = false;       // the wait for V's place ran out: of step o K's copies were issued
    bool dead = false, bad = false;
    // steps from .. to - 1 of the block at p
    __device__ __forceinline__ void block(const At& p, int from, int to) {
        const int lane = threadIdx.x & 31, piece = min(1 << a.page_log2, kKeys), pieces = kKeys / piece;
        const int* tab = a.s.table + p.b * a.s.ldt;
        // lane l: whether some row sees piece l of step i (apart from its page's number, which may be anything), and its page
        auto seen = [&](int i) {
            const int key = (p.s.u0 + i) * kKeys + lane * piece;
            return i < to && lane < pieces && key < p.s.hi && key + piece > p.s.lo;
        };
        auto lookup = [&](int i) { return seen(i) ? tab[((p.s.u0 + i) * kKeys + lane * piece) >> a.page_log2] : 0; };
        int next = lookup(from);
        for (int i = from; i < to; i++, o++) {
            int page = next;
            next = lookup(i + 1);
            const bool live = seen(i);
            if (live && (page < 0 || page >= a.pages)) { bad = true; page = a.pages; }   // TMA fills zeros
            const int st = Ring<NS>::stage(o), row = ((p.s.u0 + i) * kKeys + lane * piece) & ((1 << a.page_log2) - 1);
            const uint32_t bytes = __popc(__ballot_sync(~0u, live)) * piece * D * 2;
#pragma unroll
            for (int side = 0; side < 2; side++) {
                const uint32_t full = (side ? vfull : kfull) + st * 8;
                if (!wait_for((side ? vempty : kempty) + st * 8, Ring<NS>::parity(o) ^ 1)) dead = true;
                dead = __any_sync(~0u, dead);
                if (dead) { half = side == 1; return; }
                if (lane == 0) tc_mbar_arrive_tx(full, bytes);
                __syncwarp();
                if (live)
#pragma unroll
                    for (int c = 0; c < D / 64; c++)
                        tma_rows((side ? sv : sk) + st * kBytes + c * (kKeys * 128) + lane * piece * 128, side ? mv : mk, row, c, p.h, page,
                                 full);
            }
        }
    }
    // every stage's last release, and so every copy, has landed before the block ends; where a wait ran out, every copy alone
    __device__ __forceinline__ void drain(int* error) {
        using R = Ring<NS>;
        const int lane = threadIdx.x & 31;
        if (!dead)
            for (int i = R::oldest(o) + lane; i < o; i += 32)
                if (!wait_for(kempty + R::stage(i) * 8, R::parity(i)) || !wait_for(vempty + R::stage(i) * 8, R::parity(i))) dead = true;
        dead = __any_sync(~0u, dead);
        if (dead)
#pragma unroll
            for (int side = 0; side < 2; side++) {
                const int issued = o + (half && side == 0);
                for (int i = R::oldest(issued) + lane; i < issued; i += 32) wait_for((side ? vfull : kfull) + R::stage(i) * 8, R::parity(i));
            }
        if (__any_sync(~0u, bad) && lane == 0) atomicOr(error, 2);
    }
};

// Q of a tile's rows `first` .. `first + 63` into its swizzled place, by a warp: cp.async, addresses once a row.  row0: the
// tile's first row of the sequence's (token, head) rows; rows: those that are some, the others become zero.
template <int D, typename At>
__device__ __forceinline__ void load_q64(const AttnArgs& a, const At& p, int row0, int rows, int first, uint32_t dst) {
    constexpr int kLanes = D / 8;   // lanes of a row
    const int lane = threadIdx.x & 31, c = lane % kLanes;
    long long place[2];   // of rows first + lane and + 32 in q
#pragma unroll
    for (int y = 0; y < 2; y++) {
        const int rr = row0 + first + y * 32 + lane, tok = a.token(rr);
        place[y] = (p.cu0 + tok) * a.ldq + (int64_t)(p.h * a.group + rr - tok * a.group) * D;
    }
#pragma unroll
    for (int j = 0; j < 2 * kLanes; j++) {
        const int i = j * (32 / kLanes) + lane / kLanes;
        const long long from = __shfl_sync(~0u, place[j / kLanes], i & 31);
        const uint32_t to = sw128(dst + (c >> 3) * (kTile * 128), first + i, c & 7);
        if (first + i < rows) cp_async16(to, a.q + from + c * 8);
        else sts128(to, make_uint4(0, 0, 0, 0));
    }
}
__device__ __forceinline__ void q_arrived() {   // this thread's part of Q, before its word to the MMA warp
    asm volatile("cp.async.wait_all;" ::: "memory");
    tc_fence_proxy_async();
}

}  // namespace attn_tc
}  // namespace b200q
