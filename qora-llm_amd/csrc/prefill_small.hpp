// What the prefill's kernels and the few-token GEMM share (operand splitting,
// row pieces), and the few-token GEMM itself: templates and inline functions
// only, for every file that builds a kernel around them.
#pragma once

#include "common.hpp"
#include "params.hpp"

namespace qora {

typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));

// Power-of-two exponent e with |v| * 2^-e < 2^15 for every |v| <= amax.
__device__ __forceinline__ int pf_row_exponent(float amax) {
    int E = 0;
    (void)frexpf(amax, &E);      // amax < 2^E (E = 0 for amax = 0)
    return E - 15;
}

__device__ __forceinline__ void pf_split(float v, int e, _Float16* hi, _Float16* lo) {
    const float s = ldexpf(v, -e);
    const _Float16 h = (_Float16)s;
    *hi = h;
    *lo = (_Float16)(s - (float)h);
}

template <int NT>
__device__ __forceinline__ float pf_block_max(float v, float* red) {
    v = wave_max(v);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    __syncthreads();
    if (lane == 0) red[wave] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int w = 1; w < NT / kWave; ++w) m = fmaxf(m, red[w]);
    return m;
}

// Row chunks of the register-cached producers: thread t of NT owns the runs
// of four consecutive elements starting at 4 (t + NT i). A row whose length,
// stride and pointers are multiples of four elements (16 bytes of fp32, 8 of
// binary16) moves as vectors (VEC); any other row element by element, with
// the same values. Elements past the row end read as 0 and are not written.
// Loads are branch-free (indexes clamped into the row, the value then
// selected), so all of a thread's loads are in flight together.
__device__ __forceinline__ bool pf_al(const void* a, uintptr_t m) { return ((uintptr_t)a & (m - 1)) == 0; }

template <bool VEC>
__device__ __forceinline__ void pf_load4(const float* x, uint32_t j, uint32_t n, float* v) {
    if constexpr (VEC) {                            // n is a positive multiple of 4
        const float4 a = *reinterpret_cast<const float4*>(x + min(j, n - 4u));
        const bool in = j < n;
        v[0] = in ? a.x : 0.f;
        v[1] = in ? a.y : 0.f;
        v[2] = in ? a.z : 0.f;
        v[3] = in ? a.w : 0.f;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float a = x[min(j + (uint32_t)c, n - 1u)];
            v[c] = j + c < n ? a : 0.f;
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void pf_gamma4(const uint16_t* g, uint32_t j, uint32_t n, float* v) {
    if constexpr (VEC) {
        const uint2 a = *reinterpret_cast<const uint2*>(g + min(j, n - 4u));
        const bool in = j < n;
        v[0] = in ? h2f((uint16_t)(a.x & 0xFFFFu)) : 0.f;
        v[1] = in ? h2f((uint16_t)(a.x >> 16)) : 0.f;
        v[2] = in ? h2f((uint16_t)(a.y & 0xFFFFu)) : 0.f;
        v[3] = in ? h2f((uint16_t)(a.y >> 16)) : 0.f;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float a = h2f(g[min(j + (uint32_t)c, n - 1u)]);
            v[c] = j + c < n ? a : 0.f;
        }
    }
}

template <bool VEC>
__device__ __forceinline__ void pf_store4(float* x, uint32_t j, uint32_t n, const float* v) {
    if constexpr (VEC) {
        if (j < n) *reinterpret_cast<float4*>(x + j) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (j + c < n) x[j + c] = v[c];
    }
}

template <bool VEC>
__device__ __forceinline__ void pf_split4(const float* v, int e, _Float16* xh, _Float16* xl, uint32_t j, uint32_t n) {
    typedef _Float16 half4v __attribute__((ext_vector_type(4)));
    if constexpr (VEC) {
        if (j >= n) return;
        half4v h, l;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float sv = ldexpf(v[c], -e);
            h[c] = (_Float16)sv;
            l[c] = (_Float16)(sv - (float)h[c]);
        }
        *reinterpret_cast<half4v*>(xh + j) = h;
        *reinterpret_cast<half4v*>(xl + j) = l;
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (j + c < n) pf_split(v[c], e, xh + j + c, xl + j + c);
    }
}

// The exponent f of the scales of one K slice, from their largest magnitude
// bits: s 2^-f < 2^12 as above, f kept between -5 and 5 so that 2^-f, 1032 2^-f
// and (q - 8) 2^-f are binary16 values (s is a multiple of 2^-24, so
// s (q - 8) 2^5 still splits exactly into two of them).
__device__ __forceinline__ int pf_scale_exp(uint32_t mx) {
    const int e = (int)((mx >> 10) & 0x1F);
    return max((e == 0 ? -14 : e - 14) - 12, -5);
}

// ---------------------------------------------------------------------------
// GEMM of a few tokens (T <= 16 TM) on the reference layout, x in fp32: one
// launch and, when K is split, a sum over the slices. The numerics are those of
// pf_gemm2_kernel (x and w in two binary16 parts, three products, fp32 sums),
// with the row and group exponents taken per K slice.
// Block: 4 waves over every token x 128 columns x one K slice of at most KP
// rows. The block splits its x slice into LDS itself (rows padded by 16 bytes:
// conflict-free fragment reads) and never synchronises again: each wave runs
// over its 32 columns with D steps of weights in flight, a lane holding
//   Q4:  dword li / 4 of rows 8 kq + 2 (li % 4), + 1 (64 B a row per block); the
//        quad exchanges them (DPP broadcasts), so that byte li of the 8 rows
//        gives the B fragments of columns 2 li and 2 li + 1;
//   F16: columns 2 li, 2 li + 1 of rows 8 kq .. + 7.
// What bounds it: at 24 tokens, 11008 -> 2048, the weight stream's latency (352
// blocks of 33 KB) and two launches: 13.9 us a call against 30.7 on the packed
// path, which split x, found the groups' exponents (two launches), packed,
// multiplied and summed in six.
// ---------------------------------------------------------------------------
template <int TM, bool Q4>
struct PfSmallLds {
    static constexpr int BM = 16 * TM;
    static constexpr int KP = TM == 4 ? 256 : 512;
    static constexpr int XS = KP + 8;               // halves per LDS row
    _Float16 xs[2][BM * XS];
    _Float16 ss[Q4 ? 4 : 1][Q4 ? KP : 8];
    int xes[BM];
    static constexpr uint32_t bytes = 2u * (2u * BM * XS + (Q4 ? 4u * KP : 8u)) + 4u * BM;
};

// Workgroup (bx, by) of the launch below, on `smem` of PfSmallLds (16-byte aligned).
template <int TM, bool Q4>
__device__ __forceinline__ void pf_gemm_small_block(const PfSmallParams& p, uint32_t bx, uint32_t by, char* smem) {
    using Lds = PfSmallLds<TM, Q4>;
    static_assert(sizeof(Lds) == Lds::bytes, "no padding");
    constexpr int BM = Lds::BM;
    constexpr int KP = Lds::KP;
    constexpr int TPR = 256 / BM;                   // threads per x row
    constexpr int NF = KP / (4 * TPR);              // float4 per thread
    constexpr int XS = Lds::XS;
    constexpr int D = Q4 ? 8 : 4;                   // steps of weights in flight
    Lds& lds = *reinterpret_cast<Lds*>(smem);
    auto& xs = lds.xs;
    auto& ss = lds.ss;
    auto& xes = lds.xes;

    const int t = threadIdx.x;
    const int lane = t & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t li = (uint32_t)lane % 16u, kq = (uint32_t)lane / 16u;
    const uint32_t K = p.k, N = p.n, G = N / 32u;
    const uint32_t grp = bx * 4u + (uint32_t)wave;
    const uint32_t gc = min(grp, G - 1u);           // (a wave past the last group works on it and stores nothing)
    const uint32_t kb = by * p.kper;
    const uint32_t ke = min(K, kb + p.kper);
    const uint32_t steps = (ke - kb) / 32u;

    struct WStep {
        uint32_t w[Q4 ? 2 : 8];
    };
    auto load_w = [&](uint32_t s) {
        WStep q;
        const uint32_t r0 = kb + min(s, steps - 1u) * 32u + 8u * kq;
        if constexpr (Q4) {
            const uint8_t* b = p.w + (uint64_t)(r0 + 2u * (li % 4u)) * (N / 2u) + gc * 16u + (li / 4u) * 4u;
            q.w[0] = *reinterpret_cast<const uint32_t*>(b);
            q.w[1] = *reinterpret_cast<const uint32_t*>(b + N / 2u);
        } else {
            const uint8_t* b = p.w + ((uint64_t)r0 * N + gc * 32u + 2u * li) * 2u;
#pragma unroll
            for (int r = 0; r < 8; ++r) q.w[r] = *reinterpret_cast<const uint32_t*>(b + (uint64_t)r * N * 2u);
        }
        return q;
    };
    WStep wr[D];
#pragma unroll
    for (int d = 0; d < D; ++d) wr[d] = load_w((uint32_t)d);

    // the slice's scales of the wave's group, and x (rows past T read row T - 1)
    uint32_t sv[Q4 ? KP / 64 : 1];
    if constexpr (Q4) {
#pragma unroll
        for (int i = 0; i < KP / 64; ++i) {
            const uint32_t r = kb + (uint32_t)lane + 64u * (uint32_t)i;
            sv[i] = p.scales[(uint64_t)min(r, ke - 1u) * G + gc];
            if (r >= ke) sv[i] = 0;
        }
    }
    const uint32_t xr = (uint32_t)t / TPR, xq = (uint32_t)t % TPR;
    const float* xp = p.x + (uint64_t)min(xr, p.T - 1u) * K + kb;
    const uint32_t kn = ke - kb;
    float xv[NF][4];
    const bool vec = pf_al(p.x, 16);                // K and kb are multiples of 32
#pragma unroll
    for (int i = 0; i < NF; ++i) {
        const uint32_t j = 4u * (xq + (uint32_t)TPR * (uint32_t)i);
        if (vec) pf_load4<true>(xp, j, kn, xv[i]);
        else pf_load4<false>(xp, j, kn, xv[i]);
    }
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < NF; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) amax = fmaxf(amax, fabsf(xv[i][c]));
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) amax = fmaxf(amax, __shfl_xor(amax, o, kWave));
    const int xe = pf_row_exponent(amax);
    if (xq == 0) xes[xr] = xe;
#pragma unroll
    for (int i = 0; i < NF; ++i)
        pf_split4<true>(xv[i], xe, &xs[0][xr * XS], &xs[1][xr * XS], 4u * (xq + (uint32_t)TPR * (uint32_t)i), kn);
    int fw = 0;
    if constexpr (Q4) {
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < KP / 64; ++i) mx = max(mx, sv[i] & 0x7FFFu);
        fw = pf_scale_exp(wave_max_u32(mx));
        const float f = ldexpf(1.0f, -fw);
#pragma unroll
        for (int i = 0; i < KP / 64; ++i) ss[wave][lane + 64 * i] = (_Float16)(h2f((uint16_t)sv[i]) * f);
    }
    __syncthreads();

    f32x4v acc[TM][2];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4v{0.f, 0.f, 0.f, 0.f};
    const uint32_t bsel = (li % 4u) | 0x0C000C00u | ((4u + li % 4u) << 16);
    auto compute = [&](const WStep& q, uint32_t s) {
        half8v bh[2], bl[2];
        if constexpr (Q4) {
            const half8v s8 = *reinterpret_cast<const half8v*>(&ss[wave][s * 32u + 8u * kq]);
            const v4u32 s4 = __builtin_bit_cast(v4u32, s8);
            const half2v b_lo = {(_Float16)1032.0f, (_Float16)1032.0f}, b_hi = {(_Float16)72.0f, (_Float16)72.0f};
            v4u32 h0, h1, l0, l1;
            auto pair = [&](int j, uint32_t e0, uint32_t e1) {
                const uint32_t by = __builtin_amdgcn_perm(e1, e0, bsel);    // byte li of rows 2 j and 2 j + 1
                const half2v q0 = __builtin_bit_cast(half2v, (by & 0x000F000Fu) | 0x64006400u) - b_lo;
                const half2v q1 = __builtin_bit_cast(half2v, (by & 0x00F000F0u) | 0x54005400u) - b_hi;
                const uint32_t sj = s4[j];
                const half2v sc = __builtin_bit_cast(half2v, sj);
                const half2v a0 = q0 * sc, a1 = q1 * sc;
                h0[j] = __builtin_bit_cast(uint32_t, a0);
                h1[j] = __builtin_bit_cast(uint32_t, a1);
                l0[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q0, sc, -a0));
                l1[j] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q1, sc, -a1));
            };
            // lane j of each quad holds rows 8 kq + 2 j, + 1
            pair(0, dpp_u32<0x00>(q.w[0]), dpp_u32<0x00>(q.w[1]));
            pair(1, dpp_u32<0x55>(q.w[0]), dpp_u32<0x55>(q.w[1]));
            pair(2, dpp_u32<0xAA>(q.w[0]), dpp_u32<0xAA>(q.w[1]));
            pair(3, dpp_u32<0xFF>(q.w[0]), dpp_u32<0xFF>(q.w[1]));
            bh[0] = __builtin_bit_cast(half8v, h0);
            bh[1] = __builtin_bit_cast(half8v, h1);
            bl[0] = __builtin_bit_cast(half8v, l0);
            bl[1] = __builtin_bit_cast(half8v, l1);
        } else {
            v4u32 h0, h1;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h0[j] = __builtin_amdgcn_perm(q.w[2 * j + 1], q.w[2 * j], 0x05040100u);
                h1[j] = __builtin_amdgcn_perm(q.w[2 * j + 1], q.w[2 * j], 0x07060302u);
            }
            bh[0] = __builtin_bit_cast(half8v, h0);
            bh[1] = __builtin_bit_cast(half8v, h1);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const uint32_t o = ((uint32_t)i * 16u + li) * XS + s * 32u + 8u * kq;
            const half8v ah = *reinterpret_cast<const half8v*>(&xs[0][o]);
            const half8v al = *reinterpret_cast<const half8v*>(&xs[1][o]);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh[j], acc[i][j], 0, 0, 0);
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh[j], acc[i][j], 0, 0, 0);
                if constexpr (Q4) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl[j], acc[i][j], 0, 0, 0);
            }
        }
    };
    // D steps a round, the next round's loads going out as a slot is used
    // (past the slice the last step is loaded again and not used)
    for (uint32_t s0 = 0; s0 < steps; s0 += D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const uint32_t s = s0 + (uint32_t)d;
            if (s < steps) compute(wr[d], s);
            if (s0 + D < steps) wr[d] = load_w(s + D);
        }
    }

    if (grp >= G) return;
    const uint32_t c = grp * 32u + 2u * li;
    float* y = p.splits > 1 ? p.part + (uint64_t)by * p.T * N : p.y;
    const bool al8 = pf_al(y, 8);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t row = (uint32_t)i * 16u + kq * 4u + (uint32_t)r;
            if (row >= p.T) continue;
            const int e = xes[row] + fw;
            const float v0 = ldexpf(acc[i][0][r], e), v1 = ldexpf(acc[i][1][r], e);
            float* d = y + (uint64_t)row * N + c;
            if (al8) {
                *reinterpret_cast<float2*>(d) = make_float2(v0, v1);
            } else {
                d[0] = v0;
                d[1] = v1;
            }
        }
}

template <int TM, bool Q4>
__global__ __launch_bounds__(256) void pf_gemm_small_kernel(PfSmallParams p) {
    __shared__ __align__(16) char smem[PfSmallLds<TM, Q4>::bytes];
    pf_gemm_small_block<TM, Q4>(p, blockIdx.x, blockIdx.y, smem);
}

}  // namespace qora
