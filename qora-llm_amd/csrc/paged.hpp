// Paged KV cache of many requests: append with the position rotation, and
// causal attention of a batch's new rows (gfx950).
#pragma once

#include "common.hpp"
#include "paged_args.hpp"
#include "params.hpp"

namespace qora {

// Sequence of a row: the last s with row_start[s] <= row, by a search that
// narrows the range 64-fold per load (one load for up to 64 sequences). The
// whole wave takes part; `row` is the same in all lanes. row_start[0] > row:
// sequence 0, whose own range then does not hold the row.
__device__ __forceinline__ uint32_t paged_seq_of(const PagedParams& g, uint32_t row) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    uint32_t lo = 0, n = g.seqs;
    while (n > 1u) {
        const uint32_t step = (n + kWave - 1u) / kWave;
        const uint32_t at = lane * step;
        const bool before = at < n && g.row_start[lo + min(at, n - 1u)] <= (int32_t)row;
        const uint32_t c = (uint32_t)__popcll(__ballot(before));
        const uint32_t skip = (c ? c - 1u : 0u) * step;
        lo += min(skip, n - 1u);
        n = min(step, n - min(skip, n - 1u));
    }
    return lo;
}

// ---------------------------------------------------------------------------
// Append (apply_rope_raw, gemv.rs:757-778, and the cache rows of
// gemv.rs:1062-1083): thread = one unit of a row, four dims of a head and, where
// they are rotated, their four partners half a rotation away, so that q_out
// may be q. Units of a row: (H + KVH) heads of hd/4 - half/4 (rotated pairs
// first), then KVH heads of hd/4 for v.
// ---------------------------------------------------------------------------
template <bool F16KV>
__device__ __forceinline__ void paged_store4(void* pool, uint64_t at, const float4& a) {
    if constexpr (F16KV) {
        *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(pool) + at) =
            make_uint2((uint32_t)f2h(a.x) | ((uint32_t)f2h(a.y) << 16), (uint32_t)f2h(a.z) | ((uint32_t)f2h(a.w) << 16));
    } else {
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(pool) + at) = a;
    }
}

// V: half is a multiple of 4 (pairs of 16-byte units); else one dim a unit.
template <bool F16KV, bool V>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendParams p) {
    constexpr uint32_t W = V ? 4u : 1u;                      // dims of a unit
    const PagedParams& g = p.g;
    const uint64_t u0 = (uint64_t)blockIdx.x * 256u + (threadIdx.x & ~(kWave - 1u));
    const uint32_t row0 = (uint32_t)min(u0 / p.units, (uint64_t)g.rows - 1u);   // the wave's first row
    uint32_t s = paged_seq_of(g, row0);
    const uint64_t uid = u0 + (threadIdx.x & (kWave - 1u));
    const uint32_t row = (uint32_t)min(uid / p.units, (uint64_t)0xFFFFFFFFu);
    if (row >= g.rows) return;
    const uint32_t u = (uint32_t)(uid - (uint64_t)row * p.units);
    while (s + 1u < g.seqs && g.row_start[s + 1u] <= (int32_t)row) ++s;
    // the unit's place in the row
    const uint32_t per = (g.hd - p.half) / W, rot = p.half / W, heads = (p.q ? p.H : 0u) + g.KVH;
    uint32_t head, d;                                        // head of q | k | v, first dim
    bool pair = false;
    if (u < heads * per) {
        head = u / per;
        const uint32_t i = u - head * per;
        pair = i < rot;
        d = (pair ? i : i + rot) * W;
    } else {
        const uint32_t i = u - heads * per, pv = g.hd / W;
        head = heads + i / pv;
        d = (i % pv) * W;
    }
    const uint32_t nq = p.q ? p.H : 0u;
    const bool is_q = head < nq, is_k = !is_q && head < heads;
    const uint32_t hh = is_q ? head : is_k ? head - nq : head - heads;   // within q, k or v
    const float* src = is_q ? p.q + (uint64_t)row * p.ldq : is_k ? p.kin + (uint64_t)row * p.ldk : p.vin + (uint64_t)row * p.ldv;
    src += (uint64_t)hh * g.hd + d;
    float a[W], b[W];
    if constexpr (V) {
        const float4 v = *reinterpret_cast<const float4*>(src);
        a[0] = v.x; a[1] = v.y; a[2] = v.z; a[3] = v.w;
        if (pair) {
            const float4 w = *reinterpret_cast<const float4*>(src + p.half);
            b[0] = w.x; b[1] = w.y; b[2] = w.z; b[3] = w.w;
        }
    } else {
        a[0] = src[0];
        if (pair) b[0] = src[p.half];
    }
    const int32_t rb = g.row_start[s], re = g.row_start[s + 1u];
    if (paged_rows_of(rb, re, g.rows) == 0 || (int32_t)row < rb || (int32_t)row >= re) return;
    const int64_t pos = (int64_t)g.kv_len[s] - (re - (int32_t)row);
    uint32_t entry, slot;
    if (!paged_table_index(pos, g.page_size, g.max_pages, &entry, &slot)) return;
    if (p.half && (uint64_t)pos >= p.rope_positions) return;
    const int32_t page = g.pages[(uint64_t)s * g.max_pages + entry];
    if (!paged_page_ok(page, g.num_pages)) return;
    if (pair) {
        const float* ct = p.cos_t + (uint64_t)pos * p.half + d;
        const float* st = p.sin_t + (uint64_t)pos * p.half + d;
#pragma unroll
        for (uint32_t i = 0; i < W; ++i) {
            const float x = a[i], y = b[i], c = ct[i], sn = st[i];
            a[i] = x * c - y * sn;
            b[i] = y * c + x * sn;
        }
    }
    auto put = [&](uint32_t dd, const float* v) {
        if (is_q) {
            float* o = p.q_out + (uint64_t)row * p.ldqo + (uint64_t)hh * g.hd + dd;
            if constexpr (V) *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
            else o[0] = v[0];
            return;
        }
        void* pool = is_k ? g.k : g.v;
        const uint64_t at = paged_offset(g.page_stride, g.head_stride, g.slot_stride, (uint32_t)page, hh, slot) + dd;
        if constexpr (V) paged_store4<F16KV>(pool, at, make_float4(v[0], v[1], v[2], v[3]));
        else if constexpr (F16KV) reinterpret_cast<uint16_t*>(pool)[at] = f2h(v[0]);
        else reinterpret_cast<float*>(pool)[at] = v[0];
    };
    put(d, a);
    if (pair) put(d + p.half, b);
}

// ---------------------------------------------------------------------------
// Attention, one wave per (row, query head): 64 positions a step, a lane
// scoring one of them, then the lanes over the dims.
// ---------------------------------------------------------------------------
template <bool F16KV>
__global__ __launch_bounds__(64) void paged_attn_row_kernel(PagedAttnParams p) {
    __shared__ float qs[kAttnMaxHd];
    __shared__ float es[kWave];
    __shared__ uint64_t offs[kWave];
    const PagedParams& g = p.g;
    const uint32_t row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const uint32_t s = paged_seq_of(g, row);
    const int32_t rb = g.row_start[s], re = g.row_start[s + 1u];
    if (paged_rows_of(rb, re, g.rows) == 0 || (int32_t)row < rb || (int32_t)row >= re) return;
    if (row - (uint32_t)rb >= g.max_new) return;
    const int64_t pos = (int64_t)g.kv_len[s] - (re - (int32_t)row);
    const uint32_t nk = (uint32_t)max((int64_t)0, min(pos + 1, (int64_t)g.page_size * g.max_pages));
    const float* q = p.q + (uint64_t)row * p.ldq + (uint64_t)h * g.hd;
    for (uint32_t d = lane; d < g.hd; d += kWave) qs[d] = q[d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
    for (uint32_t k0 = 0; k0 < nk; k0 += kWave) {
        uint32_t entry = 0, slot = 0;
        bool on = k0 + lane < nk && paged_table_index(k0 + lane, g.page_size, g.max_pages, &entry, &slot);
        uint64_t at = 0;
        float sc = -INFINITY;
        if (on) {
            const int32_t page = g.pages[(uint64_t)s * g.max_pages + entry];
            on = paged_page_ok(page, g.num_pages);
            if (on) {
                at = paged_offset(g.page_stride, g.head_stride, g.slot_stride, (uint32_t)page, h / p.G, slot);
                float dot = 0.f;
                for (uint32_t d = 0; d < g.hd; ++d) {
                    const float kv = F16KV ? h2f(reinterpret_cast<const uint16_t*>(g.k)[at + d])
                                           : reinterpret_cast<const float*>(g.k)[at + d];
                    dot = fmaf(qs[d], kv, dot);
                }
                sc = dot * p.scale;
            }
        }
        const float mn = fmaxf(m, wave_max(sc));
        const float mref = mn == -INFINITY ? 0.f : mn;
        const float f = expf(m - mref), e = on ? expf(sc - mref) : 0.f;
        l = l * f + wave_sum(e);
        m = mn;
        const uint64_t live = __ballot(on);
        __syncthreads();
        es[lane] = e;
        offs[lane] = at;
        __syncthreads();
        o[0] *= f;
        o[1] *= f;
        for (uint32_t j = 0; j < (uint32_t)kWave; ++j) {
            if (!((live >> j) & 1u)) continue;
#pragma unroll
            for (uint32_t i = 0; i < 2; ++i) {
                const uint32_t d = lane + kWave * i;
                if (d >= g.hd) continue;
                const float v = F16KV ? h2f(reinterpret_cast<const uint16_t*>(g.v)[offs[j] + d])
                                      : reinterpret_cast<const float*>(g.v)[offs[j] + d];
                o[i] = fmaf(es[j], v, o[i]);
            }
        }
    }
    const float inv = nk && m > -INFINITY ? 1.0f / l : (m == m ? 0.f : m);
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
        const uint32_t d = lane + kWave * i;
        if (d < g.hd) p.out[(uint64_t)row * p.ldo + (uint64_t)h * g.hd + d] = o[i] * inv;
    }
}

}  // namespace qora
