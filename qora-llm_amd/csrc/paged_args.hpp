// Argument checks and index arithmetic of the paged KV cache calls. Plain C++
// (no HIP header needed), so that they also build for the CPU tests.
#pragma once

#include <stdint.h>
#include <stddef.h>

#include "../../include/qora_hip.h"

#if defined(__HIPCC__)
#define QORA_HD __host__ __device__ __forceinline__
#else
#define QORA_HD inline
#endif

namespace qora {

constexpr uint32_t kPagedMaxSeqs = 4096;

// Position -> slot of its page table entry: false where the position has no
// place (negative, past the table, or a page id outside the pool).
QORA_HD bool paged_table_index(int64_t pos, uint32_t page_size, uint32_t max_pages, uint32_t* entry, uint32_t* slot) {
    if (pos < 0 || pos >= (int64_t)page_size * (int64_t)max_pages) return false;
    *entry = (uint32_t)pos / page_size;
    *slot = (uint32_t)pos - *entry * page_size;
    return true;
}

QORA_HD bool paged_page_ok(int32_t page, uint32_t num_pages) { return page >= 0 && (uint32_t)page < num_pages; }

// Element offset of one KV head's slot in the pool.
QORA_HD uint64_t paged_offset(uint64_t page_stride, uint64_t head_stride, uint64_t slot_stride, uint32_t page,
                              uint32_t head, uint32_t slot) {
    return (uint64_t)page * page_stride + (uint64_t)head * head_stride + (uint64_t)slot * slot_stride;
}

// New rows of sequence s and the first of them, from two neighbouring row
// offsets: 0 rows unless 0 <= a <= b <= rows.
QORA_HD uint32_t paged_rows_of(int32_t a, int32_t b, uint32_t rows) {
    return a >= 0 && b >= a && (uint32_t)b <= rows ? (uint32_t)(b - a) : 0u;
}

// nullptr when the pool describes memory the kernels can address: every
// (page, head, slot) row is 16-byte aligned and apart from every other one.
inline const char* paged_kv_error(const qora_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v) return "null cache";
    if (kv->kv_f16 > 1) return "kv_f16 must be 0 or 1";
    if (kv->num_pages == 0 || kv->page_size == 0 || kv->num_kv_heads == 0) return "empty page pool";
    if (kv->num_pages > 0x7FFFFFFFu || kv->page_size > 0x7FFFFFFFu || kv->num_kv_heads > 65535u)
        return "page pool too large";
    if (kv->head_dim == 0 || kv->head_dim > 128 || kv->head_dim % 8 != 0)
        return "paged caches need head_dim a multiple of 8, at most 128";
    const uint64_t al = kv->kv_f16 ? 8 : 4;          // elements in 16 bytes
    uint64_t st[3] = {kv->page_stride, kv->head_stride, kv->slot_stride};
    uint64_t n[3] = {kv->num_pages, kv->num_kv_heads, kv->page_size};
    for (int i = 0; i < 3; ++i) {
        if (st[i] >= (1ull << 40)) return "page pool stride too large";
        if (st[i] % al != 0) return "page pool strides must be multiples of 16 bytes";
    }
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) % 16 != 0) return "page pools must be 16-byte aligned";
    // from the smallest stride up, each must step over everything inside it
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j + 1 < 3; ++j)
            if (st[j] > st[j + 1]) {
                const uint64_t a = st[j], b = n[j];
                st[j] = st[j + 1];
                n[j] = n[j + 1];
                st[j + 1] = a;
                n[j + 1] = b;
            }
    uint64_t extent = kv->head_dim;
    for (int i = 0; i < 3; ++i) {
        if (n[i] == 1) continue;
        if (st[i] < extent) return "page pool strides overlap";
        if ((n[i] - 1) > ((1ull << 58) - extent) / st[i]) return "page pool too large";
        extent += (n[i] - 1) * st[i];
    }
    // rows are addressed in units of 16 bytes in 32 bits
    if (extent / al >= (1ull << 32)) return "page pool larger than 64 GiB";
    if (kv->k == kv->v) return "k and v pools are the same memory";
    return nullptr;
}

inline const char* paged_batch_error(const qora_paged_kv* kv, const qora_paged_batch* b) {
    if (!b) return "null batch";
    if (b->num_seqs > kPagedMaxSeqs) return "too many sequences in the batch";
    if (b->rows > 0x7FFFFFFFu) return "too many rows in the batch";
    if (b->num_seqs == 0 || b->rows == 0) return nullptr;       // nothing to do
    if (!b->row_start || !b->kv_len || !b->pages) return "null batch array";
    if (b->max_pages == 0) return "empty page table";
    if ((uint64_t)b->max_pages * kv->page_size > 0x7FFFFFFFull) return "page table covers more than 2^31 - 1 positions";
    return nullptr;
}

// Rows of `heads` heads: a row stride in elements that holds them, every row 16-byte aligned.
inline const char* paged_rows_error(const void* p, uint64_t ld, uint64_t heads, uint32_t hd) {
    if (!p) return "null argument";
    if (((uintptr_t)p) % 16 != 0 || ld % 4 != 0) return "rows must be 16-byte aligned";
    if (ld < heads * hd || ld >= (1ull << 30)) return "row stride does not hold the heads";
    return nullptr;
}

// Whether two arrays of `rows` rows, ld floats apart and w floats wide, share memory. Rows of the same stride
// may lie between each other (the parts of a q|k|v row).
inline bool paged_rows_meet(const void* a, uint64_t lda, uint64_t wa, const void* b, uint64_t ldb, uint64_t wb,
                            uint64_t rows) {
    if (rows == 0) return false;
    const uint64_t x = (uint64_t)(uintptr_t)a, y = (uint64_t)(uintptr_t)b;
    const uint64_t xe = x + ((rows - 1) * lda + wa) * 4, ye = y + ((rows - 1) * ldb + wb) * 4;
    if (xe <= y || ye <= x) return false;
    if (lda != ldb || (y - x) % 4 != 0) return true;
    // b's first column after a's, modulo the stride
    const uint64_t d = y >= x ? (y - x) / 4 % lda : (lda - (x - y) / 4 % lda) % lda;
    return d < wa || d + wb > lda;
}

}  // namespace qora
