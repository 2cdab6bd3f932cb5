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

inline bool kv_page_ok(int page) { return page >= 16 && page <= 256 && (page & (page - 1)) == 0; }
inline int log2_of(int v) { int l = 0; while ((1 << l) < v) l++; return l; }
inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) == 0; }

// what every entry point asks of the cache and the step's description
inline bool kv_args_ok(const void* k, const void* v, int64_t k_stride, int64_t v_stride, int pages, int page, int hkv, int d,
                       const int* table, int64_t ldt, int width, const int* lens, const int* cu, int batch) {
    return k && v && table && lens && cu && aligned(k, 16) && aligned(v, 16) && aligned(table, 4) && aligned(lens, 4) &&
           aligned(cu, 4) && (d == 64 || d == 128) && kv_page_ok(page) && pages > 0 && hkv > 0 && hkv <= 1024 && width > 0 &&
           ldt >= width && (int64_t)width * page <= (1 << 30) && batch > 0 && batch <= 4096 &&
           k_stride >= (int64_t)hkv * page * d && v_stride >= (int64_t)hkv * page * d && k_stride % 8 == 0 && v_stride % 8 == 0 &&
           k_stride < ((int64_t)1 << 38) && v_stride < ((int64_t)1 << 38);
}

}  // namespace b200q
