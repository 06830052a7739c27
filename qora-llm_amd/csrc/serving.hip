// Kernel instantiations and launch helpers of the many-request calls (gfx950).
#include "launch.hpp"
#include "paged.hpp"

#include <algorithm>

namespace qora {

hipError_t launch_paged_append(const PagedAppendParams& in, bool f16, hipStream_t stream) {
    PagedAppendParams p = in;
    if (p.g.rows == 0 || p.g.seqs == 0) return hipSuccess;
    const bool vec = p.half % 4 == 0;
    const uint32_t w = vec ? 4u : 1u, heads = (p.q ? p.H : 0u) + p.g.KVH;
    const uint64_t units = (uint64_t)heads * ((p.g.hd - p.half) / w) + (uint64_t)p.g.KVH * (p.g.hd / w);
    const uint64_t blocks = ((uint64_t)p.g.rows * units + 255u) / 256u;
    if (units > 0x7FFFFFFFull || blocks > 0x7FFFFFFFull) return hipErrorInvalidValue;
    p.units = (uint32_t)units;
    const dim3 grid((uint32_t)blocks), block(256);
    if (f16 && vec) hipLaunchKernelGGL((paged_append_kernel<true, true>), grid, block, 0, stream, p);
    else if (f16) hipLaunchKernelGGL((paged_append_kernel<true, false>), grid, block, 0, stream, p);
    else if (vec) hipLaunchKernelGGL((paged_append_kernel<false, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_append_kernel<false, false>), grid, block, 0, stream, p);
    return hipGetLastError();
}

// Items the work is cut into: twice the CUs, two workgroups on each. (512 rows over 8192 keys, calls on one stream
// / on three: 116 / 76 us; with half as many 125 / 72; 65535 positions 67 / 37.6 and 62 / 36.5; 4096 in f32
// 51.6 / 23.1 and 52.2 / 24.3.)
static uint32_t paged_target(int cus) { return 2u * (uint32_t)std::max(1, cus); }

// Items beyond the target: every tile's last chunk may be a short one.
uint64_t paged_attn_items(uint64_t rows, uint64_t seqs, uint32_t G, uint32_t KVH, int cus) {
    return paged_target(cus) + (uint64_t)KVH * (seqs + rows * G / kPgWideRows);
}

static bool paged_wide_rows(uint64_t max_new, uint32_t G) { return max_new * G > kPgNarrowRows; }

// Items of split tiles: a tile is split when it has more than an item's share of the work, so there are at most
// `target` such tiles, and their items are at most that share's count and one more each.
static uint32_t paged_states(int cus) { return 2u * paged_target(cus) + 2u; }

uint64_t paged_attn_part_bytes(uint64_t rows, uint32_t G, uint32_t hd, int cus) {
    return (uint64_t)paged_states(cus) * pg_part_floats(hd <= 64 ? 64 : 128, paged_wide_rows(rows, G)) * sizeof(float);
}

hipError_t launch_paged_attn(const PagedAttnParams& in, bool f16, int cus, hipStream_t stream) {
    PagedAttnParams p = in;
    if (p.g.rows == 0 || p.g.seqs == 0) return hipSuccess;
    const uint32_t es = f16 ? 2u : 4u, HD = p.g.hd <= 64 ? 64u : 128u;
    p.page_u = (uint32_t)(p.g.page_stride * es / 16u);
    p.head_u = (uint32_t)(p.g.head_stride * es / 16u);
    p.slot_u = (uint32_t)(p.g.slot_stride * es / 16u);
    const bool wide = paged_wide_rows(p.g.max_new, p.G);
    p.narrow_shift = (uint32_t)__builtin_ctz(pg_narrow_keys(f16));
    p.wide_shift = (uint32_t)__builtin_ctz(pg_wide_keys(f16));
    // A narrow step (128 binary16 keys of a row or two) takes a workgroup about as long as four wide ones (64 keys of
    // 128 rows): one chunk beside 16 single tokens, calls on one stream / on three, 99.5 / 54.5 us at two, 90.9 / 52.4
    // at four, 98.5 / 52.1 at six. No item is shorter than one narrow step or four wide ones: a state to store
    // and join costs as much as that.
    p.narrow_cost = 4.f;
    p.wide_cost = 1.f;
    p.target = (float)paged_target(cus);
    p.least = 4.f;
    p.part_floats = pg_part_floats(HD, wide);
    p.states = paged_states(cus);
    const uint64_t items = paged_attn_items(p.g.rows, p.g.seqs, p.G, p.g.KVH, cus);
    if (items > kPgMaxItems) return hipErrorInvalidValue;
    const dim3 grid((uint32_t)items), block(256);
#define QORA_PAGED(HD_, F_, W_)                                                                                     \
    do {                                                                                                            \
        if (p.g.seqs > kWave) hipLaunchKernelGGL((paged_attn_kernel<HD_, F_, W_, true>), grid, block, 0, stream, p); \
        else hipLaunchKernelGGL((paged_attn_kernel<HD_, F_, W_, false>), grid, block, 0, stream, p);                \
    } while (0)
#define QORA_PAGED_W(HD_, F_) \
    do {                      \
        if (wide) QORA_PAGED(HD_, F_, true); else QORA_PAGED(HD_, F_, false); \
    } while (0)
    if (HD == 128 && f16) QORA_PAGED_W(128, true);
    else if (HD == 128) QORA_PAGED_W(128, false);
    else if (f16) QORA_PAGED_W(64, true);
    else QORA_PAGED_W(64, false);
#undef QORA_PAGED_W
#undef QORA_PAGED
    return hipGetLastError();
}

}  // namespace qora
