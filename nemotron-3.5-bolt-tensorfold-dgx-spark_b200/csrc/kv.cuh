// The paged key/value cache as the append and attention kernels see it, and the ragged rows of one step.
//
// k and v: [pages][heads][page][d] bf16, every page's heads x page x d values contiguous, pages at any stride.  The
// token at position p of sequence b sits in page table[b][p / page], row p % page.  Sequence b's rows of the step are
// cu[b] .. cu[b + 1] - 1; lens[b] counts its cached tokens with the step's own, so row i of r stands at lens - r + i.
#pragma once
#include "common.cuh"

namespace b200q {

struct KvSeqs {
    const int* table;    // [batch][ldt], width entries used
    const int* lens;     // [batch]
    const int* cu;       // [batch + 1]
    int64_t ldt;
    int width, batch;
};

int device_sms();   // SMs of the current device (core.cu)

inline bool kv_page_ok(int page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }
inline int log2_of(int v) { int l = 0; while ((1 << l) < v) l++; return l; }
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// what every entry point asks of the cache and the step's description
inline bool kv_ok(const b200q_paged* p) {
    if (!p) return false;
    const int64_t one = (int64_t)p->hkv * p->page * p->d, far = (int64_t)1 << 38;
    return p->k_pages && p->v_pages && p->table && p->lens && p->cu && aligned(p->k_pages, 16) && aligned(p->v_pages, 16) &&
           aligned(p->table, 4) && aligned(p->lens, 4) && aligned(p->cu, 4) && (p->d == 64 || p->d == 128) && kv_page_ok(p->page) &&
           p->pages > 0 && p->hkv > 0 && p->hkv <= 1024 && p->width > 0 && p->ldt >= p->width &&
           (int64_t)p->width * p->page <= (1 << 30) && p->batch > 0 && p->batch <= 4096 && p->k_stride >= one &&
           p->v_stride >= one && p->k_stride % 8 == 0 && p->v_stride % 8 == 0 && p->k_stride < far && p->v_stride < far;
}
// Whether n rows of wa bytes, pa apart, and n rows of wb bytes, pb apart, share no byte.  At one pitch the rows of each may lie
// between those of the other, as views of one buffer do; at two pitches whole ranges are compared.
inline bool rows_apart(const void* a, int64_t pa, int64_t wa, const void* b, int64_t pb, int64_t wb, int64_t n) {
    const int64_t x = (int64_t)(uintptr_t)a, y = (int64_t)(uintptr_t)b;
    if (n <= 0 || x + (n - 1) * pa + wa <= y || y + (n - 1) * pb + wb <= x) return true;
    if (n == 1 || pa != pb) return false;
    const int64_t at = ((y - x) % pa + pa) % pa;
    return at >= wa && at + wb <= pa;
}
inline KvSeqs kv_seqs(const b200q_paged& p) { return {p.table, p.lens, p.cu, p.ldt, p.width, p.batch}; }

}  // namespace b200q
