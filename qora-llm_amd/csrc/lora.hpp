// Low-rank adapters of many requests beside a shared projection (gfx950):
//   y[t] = x[t] W + s_e (x[t] A_e) B_e,  e = row_adapter[t].
// Two steps around the shared product: u = x A_e of every row with an adapter
// (lora_shrink), and y += s_e u B_e (lora_expand). Rows come in blocks of 16, the
// height of a matrix tile; a block runs once for each distinct adapter among its
// rows, on all 16 rows, and keeps the rows that are the adapter's. So rows
// of one adapter side by side (a prompt) read it once per block, and a batch of single
// tokens reads each adapter about once, in whatever order the rows come.
// Both steps multiply on the bfloat16 matrix cores (v_mfma_f32_16x16x32_bf16): the
// float32 side is cut into three bfloat16 parts and the binary16 side into two, both
// exactly, and the five products above 2^-24 are kept; sums are float32, no scale
// or exponent is needed, and a row's sums do not depend on its neighbours.
// What bounds them is latency: a decode step's adapters are a few MB that each come
// once, so the work is spread over slots (one block per distinct adapter), K slices and
// columns, and the steps ride in the launches of the few-token GEMM (its product in
// front, its sum of K slices behind) instead of two of their own.
#pragma once

#include "common.hpp"
#include "params.hpp"
#include "prefill_small.hpp"

namespace qora {

typedef __bf16 lr_bf8 __attribute__((ext_vector_type(8)));

// Three bfloat16 parts of eight float32 values.
__device__ __forceinline__ void lr_cut(const float* v, v4u32* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
        p[0][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        const uint32_t a2 = __float_as_uint(v[2 * i] - __uint_as_float(a & 0xFFFF0000u));
        const uint32_t b2 = __float_as_uint(v[2 * i + 1] - __uint_as_float(b & 0xFFFF0000u));
        p[1][i] = __builtin_amdgcn_perm(b2, a2, 0x07060302u);
        const float a3 = __uint_as_float(a2) - __uint_as_float(a2 & 0xFFFF0000u);
        const float b3 = __uint_as_float(b2) - __uint_as_float(b2 & 0xFFFF0000u);
        p[2][i] = __builtin_amdgcn_perm(__float_as_uint(b3), __float_as_uint(a3), 0x07060302u);
    }
}

// Two bfloat16 parts (8 and 3 bits) of eight binary16 values.
__device__ __forceinline__ void lr_cut16(const v4u32& w, v4u32* p) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = f16lo(w[i]), y = f16hi(w[i]);
        const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
        p[0][i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
        const float a2 = x - __uint_as_float(a & 0xFFFF0000u), b2 = y - __uint_as_float(b & 0xFFFF0000u);
        p[1][i] = __builtin_amdgcn_perm(__float_as_uint(b2), __float_as_uint(a2), 0x07060302u);
    }
}

__device__ __forceinline__ f32x4v lr_mma(const v4u32* x, const v4u32* w, f32x4v c) {
    auto mm = [&](const v4u32& a, const v4u32& b) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lr_bf8, a), __builtin_bit_cast(lr_bf8, b), c, 0, 0, 0);
    };
    mm(x[2], w[0]);
    mm(x[1], w[1]);
    mm(x[0], w[1]);
    mm(x[1], w[0]);
    mm(x[0], w[0]);
    return c;
}

// The row block's adapters: lane i % 16's row, -1 without one; and the rows that are
// the first of their adapter, as a mask of 16.
__device__ __forceinline__ int32_t lr_rows(const LoraParams& p, uint32_t rb, uint32_t* firsts) {
    const uint32_t lane = threadIdx.x & (kWave - 1), i = lane % 16u, t = rb * 16u + i;
    int32_t a = p.row_adapter[min(t, p.rows - 1u)];
    if (t >= p.rows || a < 0 || (uint32_t)a >= p.count) a = -1;
    bool first = a >= 0;
#pragma unroll
    for (uint32_t j = 0; j < 15u; ++j) {
        const int32_t b = __builtin_amdgcn_readlane(a, (int)j);
        if (j < i && b == a) first = false;
    }
    *firsts = (uint32_t)__ballot(first) & 0xFFFFu;
    return a;
}

// The n-th of them.
__device__ __forceinline__ int32_t lr_nth(int32_t mine, uint32_t firsts, uint32_t n) {
    for (uint32_t i = 0; i < n; ++i) firsts &= firsts - 1u;
    return __builtin_amdgcn_readlane(mine, __builtin_ctz(firsts));
}

__device__ __forceinline__ LoraEntry lr_entry(const LoraParams& p, int32_t e) {
    LoraEntry a = p.entries[e];
    a.at = sgpr_ptr(a.at);
    a.bt = sgpr_ptr(a.bt);
    a.rp = __builtin_amdgcn_readfirstlane(a.rp);
    return a;
}

constexpr uint32_t kLoraShrinkLds = 4u * 16u * 64u * 4u;

// u[z][t][r] = sum over K slice z of x[t][k] A_e[k][r], block (slot, z, row block): the slot's
// distinct adapters slot, slot + slots, ... Wave w takes k = 128 w .. + 127 of every 512, up to
// 64 ranks at a time; the waves' sums are joined in LDS in wave order.
__device__ __forceinline__ void lora_shrink_block(const LoraParams& p, uint32_t slot, uint32_t z, uint32_t rb, float* red) {
    const uint32_t t = threadIdx.x, lane = t & (kWave - 1), g = lane / 16u, li = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    uint32_t firsts;
    const int32_t mine = lr_rows(p, rb, &firsts);
    const uint32_t n = (uint32_t)__popc(firsts);
    const uint32_t kb = z * p.kper, ke = min(p.k, kb + p.kper);
    const float* x = p.x + (uint64_t)min(rb * 16u + li, p.rows - 1u) * p.k;
    const bool vec = pf_al(p.x, 16);
    for (uint32_t d = slot; d < n; d += p.slots) {
        const int32_t e = lr_nth(mine, firsts, d);
        const LoraEntry a = lr_entry(p, e);
        for (uint32_t c0 = 0; c0 < a.rp; c0 += 64u) {
            f32x4v acc[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = f32x4v{0.f, 0.f, 0.f, 0.f};
            for (uint32_t k0 = kb + wave * 128u; k0 < ke; k0 += 512u) {
                float xv[4][8];
                v4u32 av[4][4];
#pragma unroll
                for (uint32_t s = 0; s < 4; ++s) {
                    const uint32_t k = k0 + 32u * s + 8u * g;
                    const bool in = k0 + 32u * s < ke;       // (k and ke are multiples of 32)
                    const uint32_t kc = in ? k : kb + 8u * g;
                    if (vec) {
                        const float4 u = *reinterpret_cast<const float4*>(x + kc), v = *reinterpret_cast<const float4*>(x + kc + 4);
                        xv[s][0] = u.x; xv[s][1] = u.y; xv[s][2] = u.z; xv[s][3] = u.w;
                        xv[s][4] = v.x; xv[s][5] = v.y; xv[s][6] = v.z; xv[s][7] = v.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) xv[s][i] = x[kc + i];
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) xv[s][i] = in ? xv[s][i] : 0.f;
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c)
                        if (c0 + 16u * c < a.rp)
                            av[c][s] = ld_global<v4u32>(a.at + (uint64_t)(c0 + 16u * c + li) * p.k + kc);
                }
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    v4u32 xp[3];
                    lr_cut(xv[s], xp);
#pragma unroll
                    for (uint32_t c = 0; c < 4; ++c)
                        if (c0 + 16u * c < a.rp) {
                            v4u32 wp[2];
                            lr_cut16(av[c][s], wp);
                            acc[c] = lr_mma(xp, wp, acc[c]);
                        }
                }
            }
            __syncthreads();                                 // (red is read from the round before)
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c)
                *reinterpret_cast<f32x4v*>(red + wave * 1024u + (16u * c + li) * 16u + 4u * g) = acc[c];
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                // (column-major: a lane's four rows are one 16-byte store)
                const uint32_t row = t % 16u, c = t / 16u + 16u * i, at = c * 16u + row;
                const int32_t whose = __shfl(mine, (int)row, kWave);
                if (whose == e && c0 + c < a.rp)
                    p.u[((uint64_t)z * p.rows + rb * 16u + row) * p.rp + c0 + c] =
                        ((red[at] + red[1024u + at]) + red[2048u + at]) + red[3072u + at];
            }
        }
    }
}

__global__ __launch_bounds__(256) void lora_shrink_kernel(LoraParams p) {
    __shared__ __align__(16) float red[kLoraShrinkLds / 4];
    lora_shrink_block(p, blockIdx.x, blockIdx.y, blockIdx.z, red);
}

// The few-token GEMM and the adapters' first step in one launch: the first
// p.slots * p.nz * row blocks workgroups are the latter's.
template <int TM, bool Q4>
__global__ __launch_bounds__(256) void lora_gemm_small_kernel(PfSmallParams q, LoraParams p, uint32_t nshrink, uint32_t nx) {
    __shared__ __align__(16) char smem[PfSmallLds<TM, Q4>::bytes > kLoraShrinkLds ? PfSmallLds<TM, Q4>::bytes : kLoraShrinkLds];
    if (blockIdx.x < nshrink) {
        const uint32_t b = blockIdx.x / p.slots;
        lora_shrink_block(p, blockIdx.x % p.slots, b % p.nz, b / p.nz, reinterpret_cast<float*>(smem));
    } else {
        const uint32_t b = blockIdx.x - nshrink;
        pf_gemm_small_block<TM, Q4>(q, b % nx, b / nx, smem);
    }
}

// y[t][j] += s_e sum_r u[t][r] B_e[r][j], block (columns, row block).
// FEW: 32 columns, the four waves taking the distinct adapters in turn and joining their
// sums (single tokens: up to 16 adapters a block, so few that the columns have to fill the
// chip); y is the sum of q.splits K slices of the product when q.splits > 1, in
// pf_sum_splits_kernel's order. Else 64 columns a wave.
template <bool FEW>
__global__ __launch_bounds__(256) void lora_expand_kernel(LoraParams p, const float* part, uint32_t splits) {
    constexpr uint32_t CT = FEW ? 2 : 4;                     // 16-column tiles of a wave
    __shared__ __align__(16) float red[FEW ? 4 * 16 * 32 : 4];
    const uint32_t t = threadIdx.x, lane = t & (kWave - 1), g = lane / 16u, li = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t rb = blockIdx.y, n0 = FEW ? blockIdx.x * 32u : blockIdx.x * 256u + wave * 64u;
    uint32_t firsts;
    const int32_t mine = lr_rows(p, rb, &firsts);
    const uint32_t n = (uint32_t)__popc(firsts);
    if (!FEW && (n == 0 || n0 >= p.n)) return;
    const float scale = mine >= 0 ? p.entries[mine].scale : 0.f;
    // FEW: the product's values of this thread's two outputs, on their way while the adapters are
    const uint32_t row2 = t / 16u, col2 = n0 + 2u * (t % 16u);
    const uint64_t at2 = (uint64_t)min(rb * 16u + row2, p.rows - 1u) * p.n + min(col2, p.n - 2u);
    float y0 = 0.f, y1 = 0.f;
    if constexpr (FEW) {
        if (splits > 1u) {
            const uint64_t total = (uint64_t)p.rows * p.n;
            for (uint32_t z = 0; z < splits; z += 4u) {
                float2 q[4];
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const float2*>(part + (uint64_t)min(z + u, splits - 1u) * total + at2);
#pragma unroll
                for (uint32_t u = 0; u < 4; ++u)
                    if (z + u < splits) {
                        y0 = z + u ? y0 + q[u].x : q[u].x;
                        y1 = z + u ? y1 + q[u].y : q[u].y;
                    }
            }
        } else {
            y0 = p.y[at2];
            y1 = p.y[at2 + 1];
        }
    }
    f32x4v acc[CT];
#pragma unroll
    for (uint32_t c = 0; c < CT; ++c) acc[c] = f32x4v{0.f, 0.f, 0.f, 0.f};
    for (uint32_t d = FEW ? wave : 0u; d < n; d += FEW ? 4u : 1u) {
        const int32_t e = lr_nth(mine, firsts, d);
        const LoraEntry a = lr_entry(p, e);
        const bool own = mine == e;
        for (uint32_t r0 = 0; r0 < a.rp; r0 += 32u) {
            const bool in = r0 + 8u * g < a.rp;
            const uint32_t rc = in ? r0 + 8u * g : 0u;
            v4u32 bv[CT];
#pragma unroll
            for (uint32_t c = 0; c < CT; ++c)
                bv[c] = ld_global<v4u32>(a.bt + (uint64_t)min(n0 + 16u * c + li, p.n - 1u) * a.rp + rc);
            float uv[8];
            const float* ur = p.u + (uint64_t)min(rb * 16u + li, p.rows - 1u) * p.rp + rc;
#pragma unroll
            for (int i = 0; i < 8; ++i) uv[i] = 0.f;
            for (uint32_t z = 0; z < p.nz; ++z) {
                const float4 u = *reinterpret_cast<const float4*>(ur + (uint64_t)z * p.rows * p.rp);
                const float4 v = *reinterpret_cast<const float4*>(ur + (uint64_t)z * p.rows * p.rp + 4);
                uv[0] += u.x; uv[1] += u.y; uv[2] += u.z; uv[3] += u.w;
                uv[4] += v.x; uv[5] += v.y; uv[6] += v.z; uv[7] += v.w;
            }
            // (rows of other adapters, and ranks past rp, may hold anything)
#pragma unroll
            for (int i = 0; i < 8; ++i) uv[i] = own && in ? uv[i] : 0.f;
            v4u32 up[3];
            lr_cut(uv, up);
#pragma unroll
            for (uint32_t c = 0; c < CT; ++c) {
                v4u32 wp[2], w = bv[c];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = in ? w[i] : 0u;
                lr_cut16(w, wp);
                acc[c] = lr_mma(up, wp, acc[c]);
            }
        }
    }
    if constexpr (FEW) {
#pragma unroll
        for (uint32_t c = 0; c < CT; ++c)
            *reinterpret_cast<f32x4v*>(red + wave * 512u + (16u * c + li) * 16u + 4u * g) = acc[c];
        __syncthreads();
        if (rb * 16u + row2 >= p.rows || col2 >= p.n) return;
        const uint32_t at = 2u * (t % 16u) * 16u + row2, bt = at + 16u;   // (column-major)
        const float s = __shfl(scale, (int)row2, kWave);
        const bool has = __shfl(mine, (int)row2, kWave) >= 0;
        if (has) {
            // (a row has one adapter: one wave's sum, the others are zero)
            y0 += s * ((red[at] + red[512u + at]) + (red[1024u + at] + red[1536u + at]));
            y1 += s * ((red[bt] + red[512u + bt]) + (red[1024u + bt] + red[1536u + bt]));
        }
        p.y[at2] = y0;
        p.y[at2 + 1] = y1;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t row = rb * 16u + 4u * g + r;
            const float s = __shfl(scale, (int)(4u * g + r), kWave);
            const bool has = __shfl(mine, (int)(4u * g + r), kWave) >= 0;
#pragma unroll
            for (uint32_t c = 0; c < CT; ++c) {
                const uint32_t col = n0 + 16u * c + li;
                if (row < p.rows && has && col < p.n) p.y[(uint64_t)row * p.n + col] += s * acc[c][r];
            }
        }
    }
}

}  // namespace qora
