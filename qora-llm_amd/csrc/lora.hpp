// Low-rank adapters of many requests beside a shared projection (gfx950).
#pragma once

#include "common.hpp"
#include "params.hpp"

namespace qora {

// u[t][r] = sum_k x[t][k] A_e[k][r], one block per row, a wave per rank column.
__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p) {
    const uint32_t t = blockIdx.x, lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int32_t e = p.row_adapter[t];
    if (e < 0 || (uint32_t)e >= p.count) return;
    const LoraEntry a = p.entries[e];
    const float* x = p.x + (uint64_t)t * p.k;
    for (uint32_t r = wave; r < a.rp; r += 4u) {
        float s = 0.f;
        for (uint32_t k = lane; k < p.k; k += kWave) s = fmaf(x[k], h2f(a.at[(uint64_t)r * p.k + k]), s);
        s = wave_sum(s);
        if (lane == 0) p.u[(uint64_t)t * p.rp + r] = s;
    }
}

// y[t][j] += scale_e sum_r u[t][r] B_e[r][j]
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p) {
    const uint32_t t = blockIdx.x, j = blockIdx.y * 256u + threadIdx.x;
    const int32_t e = p.row_adapter[t];
    if (e < 0 || (uint32_t)e >= p.count || j >= p.n) return;
    const LoraEntry a = p.entries[e];
    float s = 0.f;
    for (uint32_t r = 0; r < a.rp; ++r) s = fmaf(p.u[(uint64_t)t * p.rp + r], h2f(a.bt[(uint64_t)j * a.rp + r]), s);
    p.y[(uint64_t)t * p.n + j] += a.scale * s;
}

}  // namespace qora
