// Kernel instantiations and launch helpers of the many-request calls (gfx950).
#include "launch.hpp"
#include "lora.hpp"
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

hipError_t launch_paged_attn(const PagedAttnParams& p, bool f16, hipStream_t stream) {
    if (p.g.rows == 0 || p.g.seqs == 0) return hipSuccess;
    const dim3 grid(p.g.rows, p.H), block(64);
    if (f16) hipLaunchKernelGGL((paged_attn_row_kernel<true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((paged_attn_row_kernel<false>), grid, block, 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_lora_shrink(const LoraParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(lora_shrink_kernel, dim3(p.rows), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_lora_expand(const LoraParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(lora_expand_kernel, dim3(p.rows, (p.n + 255u) / 256u), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace qora
