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

// The adapter of row first + lane and its entry, e = -1 without one; lanes from `rows` on have none.
// The entries of all rows come in one load, so that a block's adapters cost it no further trip to memory.
struct LrMine {
    int32_t e;
    LoraEntry a;
};

__device__ __forceinline__ LrMine lr_mine(const LoraParams& p, uint32_t first, uint32_t rows) {
    const uint32_t lane = threadIdx.x & (kWave - 1), t = first + lane;
    const int32_t e = p.row_adapter[min(t, p.rows - 1u)];
    LrMine m;
    m.e = lane < rows && t < p.rows && e >= 0 && (uint32_t)e < p.count ? e : -1;
    m.a = p.entries[max(m.e, 0)];
    return m;
}

// The next distinct adapter of `rest` (lanes whose row is still to do), taken out of it; its entry in scalar registers.
__device__ __forceinline__ int32_t lr_next(const LrMine& m, uint64_t* rest, LoraEntry* a) {
    const int w = __builtin_ctzll(*rest);
    const int32_t e = __builtin_amdgcn_readlane(m.e, w);
    *rest &= ~__ballot(m.e == e);
    auto word = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, w); };
    auto ptr = [&](const uint16_t* q) {
        const uint64_t v = (uint64_t)q;
        return reinterpret_cast<const uint16_t*>((uint64_t)word((uint32_t)v) | ((uint64_t)word((uint32_t)(v >> 32)) << 32));
    };
    a->at = ptr(m.a.at);
    a->bt = ptr(m.a.bt);
    a->rp = word(m.a.rp);
    a->scale = __uint_as_float(word(__float_as_uint(m.a.scale)));
    return e;
}

constexpr uint32_t kLoraSlices = 8;                          // K slices of x . A at most
constexpr uint32_t kLoraRanks = 32;                          // ranks of a workgroup of the first step
constexpr uint32_t kLoraShrinkLds = 4u * 16u * kLoraRanks * 4u;

// Workgroups of the first step per K slice and row block.
__host__ __device__ __forceinline__ uint32_t lora_slots(const LoraParams& p) { return p.slots * (p.rp32 / kLoraRanks); }

// A wave's part of x A^T for 16 rows and 16 NC ranks from c0 on: k = kb + 128 wave .. + 127 of every 512. x: the lane's row.
template <bool VEC, int NC>
__device__ __forceinline__ void lora_shrink_wave(const float* x, const LoraEntry& a, uint32_t K, uint32_t c0, uint32_t kb,
                                                 uint32_t ke, uint32_t wave, f32x4v* acc) {
    const uint32_t lane = threadIdx.x & (kWave - 1), g = lane / 16u, li = lane % 16u;
    for (uint32_t k0 = kb + wave * 128u; k0 < ke; k0 += 512u) {
        float xv[4][8];
        v4u32 av[NC][4];
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
            const uint32_t kc = (k0 + 32u * s < ke ? k0 + 32u * s : kb) + 8u * g;   // (k, kb and ke are multiples of 32)
            if constexpr (VEC) {
                const float4 u = *reinterpret_cast<const float4*>(x + kc), v = *reinterpret_cast<const float4*>(x + kc + 4);
                xv[s][0] = u.x; xv[s][1] = u.y; xv[s][2] = u.z; xv[s][3] = u.w;
                xv[s][4] = v.x; xv[s][5] = v.y; xv[s][6] = v.z; xv[s][7] = v.w;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) xv[s][i] = x[kc + i];
            }
#pragma unroll
            for (uint32_t c = 0; c < NC; ++c)
                av[c][s] = ld_global<v4u32>(a.at + (uint64_t)min(c0 + 16u * c + li, a.rp - 1u) * K + kc);
        }
#pragma unroll
        for (uint32_t s = 0; s < 4; ++s) {
            const bool in = k0 + 32u * s < ke;
#pragma unroll
            for (int i = 0; i < 8; ++i) xv[s][i] = in ? xv[s][i] : 0.f;
            v4u32 xp[3];
            lr_cut(xv[s], xp);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                v4u32 wp[2];
                lr_cut16(av[c][s], wp);
                acc[c] = lr_mma(xp, wp, acc[c]);
            }
        }
    }
}

// u[z][t][r] = sum over K slice z of x[t][k] A_e[k][r], block (slot, z, row block): the slot's
// distinct adapters slot / chunks, + slots, ... of 32 ranks (chunk slot % chunks); the waves' sums are joined in
// LDS in wave order. With one slice and p.uh set they go out as two binary16 parts on a
// power-of-two scale of the row's 32 (uh, ul, ue): the second step of a prompt reads them once per column block,
// and then multiplies what it loads. VEC: x starts on 16 bytes.
template <bool VEC>
__device__ __forceinline__ void lora_shrink_rows(const LoraParams& p, uint32_t slot, uint32_t z, uint32_t rb, float* red) {
    const uint32_t t = threadIdx.x, lane = t & (kWave - 1), g = lane / 16u, li = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const LrMine mine = lr_mine(p, rb * 16u, 16u);
    uint64_t rest = __ballot(mine.e >= 0);
    const uint32_t kb = z * p.kper, ke = min(p.k, kb + p.kper);
    const float* x = p.x + (uint64_t)min(rb * 16u + li, p.rows - 1u) * p.k;
    const uint32_t chunks = p.rp32 / kLoraRanks, c0 = (slot % chunks) * kLoraRanks;
    slot /= chunks;
    {
        for (uint32_t d = 0; rest; ++d) {
            LoraEntry a;
            const int32_t e = lr_next(mine, &rest, &a);
            if (d % p.slots != slot) continue;
            if (c0 >= a.rp) continue;
            f32x4v acc[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[c] = f32x4v{0.f, 0.f, 0.f, 0.f};
            if (a.rp - c0 <= 16u) lora_shrink_wave<VEC, 1>(x, a, p.k, c0, kb, ke, wave, acc);
            else lora_shrink_wave<VEC, 2>(x, a, p.k, c0, kb, ke, wave, acc);
            __syncthreads();                                 // (red is read from the round before)
#pragma unroll
            for (uint32_t c = 0; c < 2; ++c)
                *reinterpret_cast<f32x4v*>(red + wave * 512u + (16u * c + li) * 16u + 4u * g) = acc[c];
            __syncthreads();
            // (column-major: a lane's four rows are one 16-byte store)
            const uint32_t row = t % 16u;
            const bool keep = __shfl(mine.e, (int)row, kWave) == e;
            float v[2], amax = 0.f;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t at = (t / 16u + 16u * i) * 16u + row;
                v[i] = ((red[at] + red[512u + at]) + red[1024u + at]) + red[1536u + at];
                if (c0 + t / 16u + 16u * i < a.rp) amax = fmaxf(amax, fabsf(v[i]));
            }
            const uint64_t r = rb * 16u + row;
            if (!p.uh) {
#pragma unroll
                for (uint32_t i = 0; i < 2; ++i) {
                    const uint32_t c = c0 + t / 16u + 16u * i;
                    if (keep && c < a.rp) p.u[((uint64_t)z * p.rows + r) * p.rp + c] = v[i];
                }
                continue;
            }
            __syncthreads();
            red[t] = amax;
            __syncthreads();
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) amax = fmaxf(amax, red[16u * i + row]);
            const int ex = pf_row_exponent(amax);
            if (keep && t < 16u) p.ue[r * chunks + c0 / kLoraRanks] = ex;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t c = c0 + t / 16u + 16u * i;
                if (keep && c < a.rp)
                    pf_split(v[i], ex, reinterpret_cast<_Float16*>(p.uh) + r * p.rp + c,
                             reinterpret_cast<_Float16*>(p.ul) + r * p.rp + c);
            }
        }
    }
}

// Workgroup b of lora_slots(p) * p.nz * row blocks: K slices fastest (with eight each XCD's L2 holds one of A and x),
// slots last (those of a number of adapters that few blocks have do nothing: with slots fastest the others met on two
// XCDs of eight, 256 rows over 11008 rows of K 40.6 us against 19.9).
__device__ __forceinline__ void lora_shrink_block(const LoraParams& p, uint32_t b, float* red) {
    const uint32_t nrb = (p.rows + 15u) / 16u, z = b % p.nz, rb = b / p.nz % nrb, slot = b / p.nz / nrb;
    if (pf_al(p.x, 16)) lora_shrink_rows<true>(p, slot, z, rb, red);
    else lora_shrink_rows<false>(p, slot, z, rb, red);
}

// The few-token GEMM and the adapters' first step in one launch: the first
// lora_slots(p) * p.nz * row blocks workgroups are the latter's.
template <int TM, bool Q4>
__global__ __launch_bounds__(256) void lora_gemm_small_kernel(PfSmallParams q, LoraParams p, uint32_t nshrink, uint32_t nx) {
    __shared__ __align__(16) char smem[PfSmallLds<TM, Q4>::bytes > kLoraShrinkLds ? PfSmallLds<TM, Q4>::bytes : kLoraShrinkLds];
    if (blockIdx.x < nshrink) {
        lora_shrink_block(p, blockIdx.x, reinterpret_cast<float*>(smem));
    } else {
        const uint32_t b = blockIdx.x - nshrink;
        pf_gemm_small_block<TM, Q4>(q, b % nx, b / nx, smem);
    }
}

// s_e u B_e of 16 TM rows first .. and CT 16-column tiles from u's two binary16 parts (B as it is, two products
// of v_mfma_f32_16x16x32_f16): add() takes a value of the product for row 16 i + 4 (lane / 16) + r and tile c.
// mine: lr_mine of the rows; cols as below.
template <int TM, int CT>
struct LoraTile {
    f32x4v sum[TM][CT];
    bool has[TM][4];

    __device__ __forceinline__ float add(float v, int i, int r, int c) const { return has[i][r] ? v + sum[i][c][r] : v; }

    __device__ __forceinline__ void get(const LoraParams& p, uint32_t first, const LrMine& mine, const uint32_t* cols) {
        const uint32_t lane = threadIdx.x & (kWave - 1), g = lane / 16u, li = lane % 16u;
        int32_t own[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            own[i] = __shfl(mine.e, (int)(16u * i + li), kWave);
#pragma unroll
            for (int c = 0; c < CT; ++c) sum[i][c] = f32x4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int r = 0; r < 4; ++r) has[i][r] = __shfl(mine.e, (int)(16u * i + 4u * g + r), kWave) >= 0;
        }
        const uint32_t nch = p.rp32 / kLoraRanks;
        uint64_t rest = __ballot(mine.e >= 0);
        while (rest) {
            LoraEntry a;
            const int32_t e = lr_next(mine, &rest, &a);
            for (uint32_t c0 = 0; c0 < a.rp; c0 += 2u * kLoraRanks) {
                v4u32 bv[2][CT], uh[2][TM], ul[2][TM];
                int ex[2][TM][4];
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) {
                    const uint32_t rc = min(c0 + kLoraRanks * s + 8u * g, a.rp - 8u);
#pragma unroll
                    for (int c = 0; c < CT; ++c) bv[s][c] = ld_global<v4u32>(a.bt + (uint64_t)min(cols[c], p.n - 1u) * a.rp + rc);
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        const uint64_t at = (uint64_t)min(first + 16u * i + li, p.rows - 1u) * p.rp + rc;
                        uh[s][i] = ld_global<v4u32>(p.uh + at);
                        ul[s][i] = ld_global<v4u32>(p.ul + at);
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            ex[s][i][r] = p.ue[(uint64_t)min(first + 16u * i + 4u * g + r, p.rows - 1u) * nch +
                                               min(c0 / kLoraRanks + s, nch - 1u)];
                    }
                }
#pragma unroll
                for (uint32_t s = 0; s < 2; ++s) {
                    const bool in = c0 + kLoraRanks * s + 8u * g < a.rp;
                    if (c0 + kLoraRanks * s >= a.rp) break;
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        // (rows of other adapters, and ranks past rp, may hold anything)
                        const uint32_t keep = own[i] == e && in ? ~0u : 0u;
                        bool mine_r[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            uh[s][i][x] &= keep;
                            ul[s][i][x] &= keep;
                            mine_r[x] = __shfl(mine.e, (int)(16u * i + 4u * g + x), kWave) == e;
                        }
#pragma unroll
                        for (int c = 0; c < CT; ++c) {
                            const half8v b = __builtin_bit_cast(half8v, bv[s][c]);
                            f32x4v acc = f32x4v{0.f, 0.f, 0.f, 0.f};
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, ul[s][i]), b, acc, 0, 0, 0);
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, uh[s][i]), b, acc, 0, 0, 0);
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                sum[i][c][r] = mine_r[r] ? sum[i][c][r] + a.scale * ldexpf(acc[r], ex[s][i][r]) : sum[i][c][r];
                        }
                    }
                }
            }
        }
    }
};

// u B_e (without the scale) of 16 rows first .., whose adapters `mine` holds (lr_mine), from the K slices' sums; cols[c]:
// the column whose B this lane holds in tile c (past n: any that is not used). The rows' distinct adapters from
// number d0 on, every step-th.
template <int CT>
__device__ __forceinline__ void lora_few_tile(const LoraParams& p, uint32_t first, const LrMine& mine, const uint32_t* cols,
                                              f32x4v* acc, uint32_t d0, uint32_t step) {
    const uint32_t lane = threadIdx.x & (kWave - 1), g = lane / 16u, li = lane % 16u;
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = f32x4v{0.f, 0.f, 0.f, 0.f};
    const int32_t own = __shfl(mine.e, (int)li, kWave);
    uint64_t rest = __ballot(mine.e >= 0);
    for (uint32_t d = 0; rest; ++d) {
        LoraEntry a;
        const int32_t e = lr_next(mine, &rest, &a);
        if (d % step != d0) continue;
        for (uint32_t r0 = 0; r0 < a.rp; r0 += 32u) {
            const bool in = r0 + 8u * g < a.rp;
            const uint32_t rc = in ? r0 + 8u * g : 0u;
            v4u32 bv[CT];
#pragma unroll
            for (int c = 0; c < CT; ++c) bv[c] = ld_global<v4u32>(a.bt + (uint64_t)min(cols[c], p.n - 1u) * a.rp + rc);
            float uv[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            for (uint32_t z0 = 0; z0 < p.nz; z0 += 4u) {     // four slices in flight
                float4 u[4], v[4];
#pragma unroll
                for (uint32_t z = 0; z < 4; ++z) {
                    const uint64_t row = (uint64_t)min(z0 + z, p.nz - 1u) * p.rows + min(first + li, p.rows - 1u);
                    u[z] = *reinterpret_cast<const float4*>(p.u + row * p.rp + rc);
                    v[z] = *reinterpret_cast<const float4*>(p.u + row * p.rp + rc + 4);
                }
#pragma unroll
                for (uint32_t z = 0; z < 4; ++z) {
                    if (z0 + z >= p.nz) continue;
                    uv[0] += u[z].x; uv[1] += u[z].y; uv[2] += u[z].z; uv[3] += u[z].w;
                    uv[4] += v[z].x; uv[5] += v[z].y; uv[6] += v[z].z; uv[7] += v[z].w;
                }
            }
            // (rows of other adapters, and ranks past rp, may hold anything)
#pragma unroll
            for (int x = 0; x < 8; ++x) uv[x] = own == e && in ? uv[x] : 0.f;
            v4u32 up[3];
            lr_cut(uv, up);
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                v4u32 w = bv[c], wp[2];
#pragma unroll
                for (int x = 0; x < 4; ++x) w[x] = in ? w[x] : 0u;
                lr_cut16(w, wp);
                acc[c] = lr_mma(up, wp, acc[c]);
            }
        }
    }
}

// y[t][j] = product + s_e sum_r u[t][r] B_e[r][j], block (32 CG columns, 16 rows); the product is y or, with
// splits > 1, the sum of its K slices in part, in the order of the kernels that sum them without adapters.
// The 8 / CG waves of 32 columns take the distinct adapters of the block's rows in turn (single tokens: up to
// 16, which one wave would wait for one after the other).
template <int CG>
__global__ __launch_bounds__(512) void lora_expand_kernel(LoraParams p, const float* part, uint32_t splits) {
    constexpr int CT = 2;                                    // 16-column tiles of a wave
    constexpr uint32_t W = 8u / CG;
    __shared__ __align__(16) float red[8 * 16 * 32];
    const uint32_t t = threadIdx.x, lane = t & (kWave - 1), g = lane / 16u, li = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t rb = blockIdx.y, n0 = blockIdx.x * 32u * CG;
    const uint64_t total = (uint64_t)p.rows * p.n;
    uint32_t cols[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) cols[c] = n0 + wave / W * 32u + 16u * c + li;
    const LrMine mine = lr_mine(p, rb * 16u, 16u);
    // thread: row t / 32, columns t % 32 and 32 further; the product's values on their way while the adapters are
    const uint32_t row = t / 32u;
    const bool on = rb * 16u + row < p.rows;
    const uint64_t at = (uint64_t)min(rb * 16u + row, p.rows - 1u) * p.n;
    uint64_t to[CG];
    float y[CG];
#pragma unroll
    for (int j = 0; j < CG; ++j) {
        to[j] = at + min(n0 + 32u * j + t % 32u, p.n - 1u);  // (n is a multiple of 32)
        y[j] = 0.f;
    }
    if (on) {
        if (splits > 1u) {
            constexpr uint32_t Z = 8u / CG;
            for (uint32_t z = 0; z < splits; z += Z) {
                float q[CG][Z];
#pragma unroll
                for (uint32_t u = 0; u < Z; ++u)
#pragma unroll
                    for (int j = 0; j < CG; ++j) q[j][u] = part[(uint64_t)min(z + u, splits - 1u) * total + to[j]];
#pragma unroll
                for (uint32_t u = 0; u < Z; ++u)
#pragma unroll
                    for (int j = 0; j < CG; ++j)
                        if (z + u < splits) y[j] = z + u ? y[j] + q[j][u] : q[j][u];
            }
        } else {
#pragma unroll
            for (int j = 0; j < CG; ++j) y[j] = p.y[to[j]];
        }
    }
    f32x4v acc[CT];
    lora_few_tile<CT>(p, rb * 16u, mine, cols, acc, wave % W, W);
#pragma unroll
    for (int c = 0; c < CT; ++c)
        *reinterpret_cast<f32x4v*>(red + wave * 512u + (16u * c + li) * 16u + 4u * g) = acc[c];
    __syncthreads();
    // the wave of the row's adapter: its number among the distinct ones, by first row, modulo the waves
    uint64_t rest = __ballot(mine.e >= 0);
    const int32_t e = __shfl(mine.e, (int)row, kWave);
    const float s = __shfl(mine.a.scale, (int)row, kWave);
    uint32_t w = 0, d = 0;
    while (rest) {
        LoraEntry a;
        if (lr_next(mine, &rest, &a) == e) w = d;
        ++d;
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < CG; ++j) {
        if (n0 + 32u * j >= p.n) break;
        if (e >= 0) y[j] = fmaf(s, red[(j * W + w % W) * 512u + (t % 32u) * 16u + row], y[j]);   // (column-major)
        p.y[to[j]] = y[j];
    }
}

}  // namespace qora
