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
// first), then KVH heads of hd/4 for v. Bound by its traffic (prompts of 4000 rows, 83 MB: 13 to 16 us, a
// large copy's rate) and, for single tokens, by the trip row offsets, length, page (32 rows: 3.7 us).
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
// Attention. The query rows of a sequence that share a KV head are flattened,
// row i = token i / G of head i % G, so every group size fills the matrix
// tiles alike, and are cut into tiles; a tile's keys are cut into chunks, and a
// (sequence, chunk, tile, KV head) is one workgroup's item. What the item
// numbers mean is worked out on the device from the batch's arrays by every
// wave (two loads and a scan over the sequences, no second launch and no
// host copy), with chunk lengths such that all items together are about
// p.target of equal cost: a batch of one long request splits far, many
// requests hardly, and a captured graph follows its arrays.
//   Narrow items (at most 16 rows: single tokens): four waves walk the keys in
//   turn, each with K and V of its own keys straight from the cache in
//   registers, and join their states at the end.
//   Wide items (128 rows): four waves of 32 rows share key tiles in LDS.
// Both keep the running maximum and sum of each row's softmax in float32 and
// hold the scores transposed (S^T = K Q^T, then O^T += V^T P^T), so that a row's
// state lives in its own lanes and its weights never leave them.
// Numerics: the matrix cores take two-byte operands. Over a binary16 cache K and V
// are exact, q (on a power-of-two scale of its row) and the weights (times 2^15)
// are split into two binary16 parts (22 bits). Over a float32 cache narrow items split every
// operand into three bfloat16 parts by cutting its bits (exact: 3 x 8 = 24) and keep the six
// products above 2^-24, which cost nothing beside the loads; wide items, bound by the products,
// split K and V into two binary16 parts too, on a power-of-two scale of each key's own, and keep
// three products. Sums are float32.
// ---------------------------------------------------------------------------
typedef _Float16 pg_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 pg_bf8 __attribute__((ext_vector_type(8)));
typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef float pg_f4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));

constexpr uint32_t kPgNarrowRows = 16, kPgWideRows = 128;
// keys of a step: a narrow item's four waves, a wide item's tile
__host__ __device__ constexpr uint32_t pg_narrow_keys(bool f16) { return f16 ? 128u : 64u; }
__host__ __device__ constexpr uint32_t pg_wide_keys(bool f16) { return f16 ? 64u : 32u; }
// floats of an item's state in the workspace
__host__ __device__ constexpr uint32_t pg_part_floats(uint32_t HD, bool wide) {
    return wide ? kPgWideRows * HD + 512u : kPgNarrowRows * HD + 32u;
}

struct PagedItem {
    uint32_t s, kvh, tile, chunk;
    uint32_t tiles, chunks;
    uint32_t per;              // steps of a chunk
    uint32_t first, state;     // item of the tile's chunk 0, and where its state goes if it is split
    uint32_t row0, n, len;     // the sequence's first row, its rows, keys any of them sees
    int64_t pos0;              // position of its first row
    uint32_t narrow;
};

// A sequence's part of the plan.
struct PagedSeqPlan {
    uint32_t row0, n, len, tiles, steps;
    int64_t pos0;
    bool narrow;
};

__device__ __forceinline__ PagedSeqPlan paged_seq_plan(const PagedAttnParams& p, uint32_t s) {
    const PagedParams& g = p.g;
    PagedSeqPlan q{};
    const uint32_t c = min(s, g.seqs - 1u);
    const int32_t a = g.row_start[c], b = g.row_start[c + 1u], L = g.kv_len[c];
    const uint32_t all = s < g.seqs ? paged_rows_of(a, b, g.rows) : 0u;
    q.n = min(all, g.max_new);
    q.row0 = (uint32_t)a;
    q.pos0 = (int64_t)L - (int64_t)all;
    const int64_t cap = (int64_t)g.page_size * g.max_pages;
    q.len = (uint32_t)max((int64_t)0, min(min((int64_t)L, cap), q.pos0 + (int64_t)q.n));
    const uint64_t M = (uint64_t)q.n * p.G;
    q.narrow = M <= kPgNarrowRows;
    q.tiles = q.narrow ? (q.n ? 1u : 0u) : (uint32_t)((M + kPgWideRows - 1u) / kPgWideRows);
    const uint32_t sh = q.narrow ? p.narrow_shift : p.wide_shift;
    q.steps = (q.len + (1u << sh) - 1u) >> sh;
    return q;
}

// Inclusive sum over the wave's lanes, by DPP: within rows of 16, then row 0's and 2's last lane into the
// next row, then lane 31's into the upper half.
__device__ __forceinline__ uint32_t pg_scan(uint32_t v) {
    v += dpp_u32<0x111>(v);    // row_shr:1 (lanes without a source add 0)
    v += dpp_u32<0x112>(v);
    v += dpp_u32<0x114>(v);
    v += dpp_u32<0x118>(v);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1 and 3
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2 and 3
    return v;
}

// What the four waves of a workgroup tell each other of a plan of more than 64 sequences.
struct PagedPlanLds {
    float cost[4];
    uint32_t items[4], split[4];
    uint32_t ok;
    PagedItem it;
};

// The item of number `item`; false if there is none. All threads take part, and every workgroup of the grid gets the
// same plan. Up to 64 sequences each wave plans by itself, without a barrier. Of more, every wave takes a quarter:
// its cost, then its items, and the wave whose quarter holds the item looks for it (1024 tokens over 100 positions:
// 160 us with all of it in every wave, 108 so). MANY: more than 64, in kernels of their own (in one kernel for both the
// others took 2 us longer: 32 tokens over up to 8192 positions 44 us against 42).
template <bool MANY>
__device__ __forceinline__ bool paged_item(const PagedAttnParams& p, uint32_t item, PagedItem* it, PagedPlanLds* lds) {
    const uint32_t lane = threadIdx.x & (kWave - 1);
    const uint32_t seqs = p.g.seqs;
    auto cost_of = [&](const PagedSeqPlan& q) {
        return (float)q.tiles * (float)q.steps * (q.narrow ? p.narrow_cost : p.wide_cost);
    };
    float share = 0.f;
    auto set_share = [&](float total) { share = fmaxf(total * (float)p.g.KVH / p.target, p.least); };
    auto chunks_of = [&](const PagedSeqPlan& q, uint32_t* per) {
        // A wide tile's states are joined one after the other, by the waves that have rows: c chunks of its steps cost
        // the longest item about steps / c + c waves / 8 steps. (32 rows over 16000 positions, one stream: 99 us with a
        // chunk for each item's share, 63 with this least length; over an f32 cache 187 and 97.)
        const float waves = fminf(ceilf((float)q.n * (float)p.G / 32.f), 4.f);
        const float per_f = ceilf(fmaxf(share / (q.narrow ? p.narrow_cost : p.wide_cost),
                                        q.narrow ? 1.f : __builtin_amdgcn_sqrtf((float)q.steps * waves * 0.125f)));
        *per = min((uint32_t)fminf(fmaxf(per_f, 1.f), 1e9f), max(q.steps, 1u));
        return max((q.steps + *per - 1u) / *per, 1u);
    };
    // (more than any grid has: such a sequence is left out below, and so is what follows it)
    auto items_of = [&](const PagedSeqPlan& q, uint32_t chunks) {
        return (uint32_t)min((uint64_t)p.g.KVH * q.tiles * chunks, (uint64_t)kPgMaxItems);
    };
    uint64_t base = 0, split = 0;                             // items before the sequences b .., those of them that are split
    // looks among sequences b .. b + 63 (lane's plan: q); 0: not there, 1: found, 2: there, but left out
    auto find = [&](const PagedSeqPlan& q, uint32_t b) {
        uint32_t per;
        const uint32_t chunks = chunks_of(q, &per), mine = items_of(q, chunks);
        const uint32_t sum = pg_scan(mine), apart = pg_scan(chunks > 1u ? mine : 0u);
        const uint64_t end = base + sum, begin = end - mine;
        const uint64_t hit = __ballot(item >= begin && item < end);
        if (!hit) {
            base += (uint32_t)__builtin_amdgcn_readlane((int)sum, kWave - 1);
            split += (uint32_t)__builtin_amdgcn_readlane((int)apart, kWave - 1);
            return 0;
        }
        const int w = __builtin_ctzll(hit);
        auto u = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, w); };
        const uint64_t e0 = base + u(sum), b0 = e0 - u(mine);
        // row offsets that are none can ask for more items than the grid has, or states than the workspace: all of
        // such a sequence is left out
        const uint64_t s1 = split + u(apart);
        if (e0 > gridDim.x || (u(chunks) > 1u && s1 > p.states)) return 2;
        it->s = b + (uint32_t)w;
        it->tiles = u(q.tiles);
        it->chunks = u(chunks);
        it->per = u(per);
        it->row0 = u(q.row0);
        it->n = u(q.n);
        it->len = u(q.len);
        it->pos0 = (int64_t)((uint64_t)u((uint32_t)(uint64_t)q.pos0) | ((uint64_t)u((uint32_t)((uint64_t)q.pos0 >> 32)) << 32));
        it->narrow = u(q.narrow ? 1u : 0u);
        // KV head fastest (a head's items keep to the same XCDs' L2), then the tiles that share a chunk of keys
        uint32_t r = item - (uint32_t)b0;
        it->kvh = r % p.g.KVH;
        r /= p.g.KVH;
        it->tile = r % it->tiles;
        it->chunk = r / it->tiles;
        it->first = (uint32_t)b0 + it->tile * p.g.KVH + it->kvh;
        it->state = it->chunks > 1u ? (uint32_t)(s1 - u(mine)) + it->tile * p.g.KVH + it->kvh : 0u;
        return 1;
    };
    if constexpr (!MANY) {
        const PagedSeqPlan q = paged_seq_plan(p, lane);
        set_share(wave_sum(cost_of(q)));
        return find(q, 0) == 1;
    }
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t quarter = ((seqs + 4u * kWave - 1u) / (4u * kWave)) * kWave;
    const uint32_t s0 = wave * quarter, s1 = min(seqs, s0 + quarter);
    const PagedSeqPlan q0 = paged_seq_plan(p, s0 + lane);     // (kept: up to 256 sequences are read once)
    float cost = cost_of(q0);
#pragma unroll 4
    for (uint32_t b = s0 + kWave; b < s1; b += kWave) cost += cost_of(paged_seq_plan(p, b + lane));
    cost = wave_sum(cost);
    if (lane == 0) lds->cost[wave] = cost;
    __syncthreads();
    set_share((lds->cost[0] + lds->cost[1]) + (lds->cost[2] + lds->cost[3]));
    uint32_t items = 0, apart = 0;                            // (no more than kPgMaxItems a lane: the sums fit 32 bits)
    auto count = [&](const PagedSeqPlan& q) {
        uint32_t per;
        const uint32_t chunks = chunks_of(q, &per), mine = items_of(q, chunks);
        items = min(items + mine, kPgMaxItems);
        apart = min(apart + (chunks > 1u ? mine : 0u), kPgMaxItems);
    };
    count(q0);
#pragma unroll 4
    for (uint32_t b = s0 + kWave; b < s1; b += kWave) count(paged_seq_plan(p, b + lane));
    items = pg_scan(items);
    apart = pg_scan(apart);
    if (lane == kWave - 1) {
        lds->items[wave] = items;
        lds->split[wave] = apart;
    }
    if (threadIdx.x == 0) lds->ok = 0;
    __syncthreads();
    uint64_t before = 0;
    bool here = false;
    for (uint32_t w = 0; w < 4; ++w) {
        const uint32_t n = __builtin_amdgcn_readfirstlane((int)lds->items[w]);
        if (w == wave && item >= before && item < before + n) here = true;
        if (w < wave) {
            base += n;
            split += (uint32_t)__builtin_amdgcn_readfirstlane((int)lds->split[w]);
        }
        before += n;
    }
    if (item >= before) return false;
    if (here) {
        int found = 0;
        PagedSeqPlan next = q0;
        for (uint32_t b = s0; b < s1 && !found; b += kWave) {
            const PagedSeqPlan q = next;
            if (b + kWave < s1) next = paged_seq_plan(p, b + kWave + lane);   // (on its way while these are looked through)
            found = find(q, b);
        }
        if (found == 1 && lane == 0) {
            lds->it = *it;
            lds->ok = 1;
        }
    }
    __syncthreads();
    if (!__builtin_amdgcn_readfirstlane((int)lds->ok)) return false;
    static_assert(sizeof(PagedItem) % 4 == 0, "copied by words");
    const uint32_t* from = reinterpret_cast<const uint32_t*>(&lds->it);
    uint32_t words[sizeof(PagedItem) / 4];
#pragma unroll
    for (uint32_t i = 0; i < sizeof(PagedItem) / 4; ++i) words[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)from[i]);
    *it = __builtin_bit_cast(PagedItem, words);
    return true;
}

// Where a key's row starts, in units of 16 bytes from the pool's first byte
// (32 bits reach 64 GB), and whether it is there.
__device__ __forceinline__ uint32_t paged_row_unit(const PagedAttnParams& p, uint32_t kvh, int32_t page, uint32_t slot) {
    return (uint32_t)page * p.page_u + kvh * p.head_u + slot * p.slot_u;
}

// x = hi + lo in binary16 for two values: hi cut (v_cvt_pkrtz), lo the rounded rest.
__device__ __forceinline__ void pg_split2(float a, float b, uint32_t* hi, uint32_t* lo) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    *hi = __builtin_bit_cast(uint32_t, h);
    const half2v r = {(_Float16)(a - (float)h[0]), (_Float16)(b - (float)h[1])};
    *lo = __builtin_bit_cast(uint32_t, r);
}

// Three bfloat16 parts of two values, packed (a low, b high): cutting 8 bits at a time is exact.
__device__ __forceinline__ void pg_cut2(float a, float b, uint32_t* p1, uint32_t* p2, uint32_t* p3) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    *p1 = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    const float a2 = a - __uint_as_float(ua & 0xFFFF0000u), b2 = b - __uint_as_float(ub & 0xFFFF0000u);
    const uint32_t va = __float_as_uint(a2), vb = __float_as_uint(b2);
    *p2 = __builtin_amdgcn_perm(vb, va, 0x07060302u);
    const float a3 = a2 - __uint_as_float(va & 0xFFFF0000u), b3 = b2 - __uint_as_float(vb & 0xFFFF0000u);
    *p3 = __builtin_amdgcn_perm(__float_as_uint(b3), __float_as_uint(a3), 0x07060302u);
}

// The last of a tile's chunks to arrive joins their states: every chunk's state is stored past this
// XCD's L2 (agent scope) before its arrival is counted; the counter is zero again afterwards.
__device__ __forceinline__ bool paged_arrive(uint32_t* count, uint32_t live, uint32_t* shared) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // this wave's state is in place
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t n = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n == live - 1u) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *shared = n;
    }
    __syncthreads();
    return *shared == live - 1u;
}

using pg_u64 = unsigned long long;
__device__ __forceinline__ void pg_put2(float* p, float a, float b) {
    const pg_u64 v = (pg_u64)__float_as_uint(a) | ((pg_u64)__float_as_uint(b) << 32);
    __hip_atomic_store(reinterpret_cast<pg_u64*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 pg_get2(const float* p) {
    const pg_u64 v = __hip_atomic_load(reinterpret_cast<const pg_u64*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// Largest of the values of each aligned group of N = 16 or 32 lanes, in every lane of it.
template <int N>
__device__ __forceinline__ uint32_t pg_group_max(uint32_t v) {
    static_assert(N == 16 || N == 32, "16- or 32-lane groups");
    v = max(v, dpp_u32<0xB1>(v));     // quad_perm [1,0,3,2]
    v = max(v, dpp_u32<0x4E>(v));     // quad_perm [2,3,0,1]
    v = max(v, dpp_u32<0x141>(v));    // row_half_mirror
    v = max(v, dpp_u32<0x140>(v));    // row_mirror
    if constexpr (N == 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max((uint32_t)a[0], (uint32_t)a[1]);
    }
    return v;
}

// A word of a vector by value (a bit cast of the element itself would read element 0).
__device__ __forceinline__ uint32_t pg_word(const v4u32& x, int i) { return x[i]; }

// Binary16 words / float32 words that are infinite or NaN.
template <bool F16>
__device__ __forceinline__ bool pg_not_finite(uint32_t w) {
    if constexpr (F16) return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
    else return (w & 0x7F800000u) == 0x7F800000u;
}

// One value of the pool, as float.
template <bool F16>
__device__ __forceinline__ float pg_value(const void* pool, uint32_t unit, uint32_t d) {
    const char* b = reinterpret_cast<const char*>(pool) + ((uint64_t)unit << 4);
    if constexpr (F16) return h2f(reinterpret_cast<const uint16_t*>(b)[d]);
    else return reinterpret_cast<const float*>(b)[d];
}

// A value that the compiler takes as new here: what is derived from it below is computed
// where it is used instead of being kept in registers over a loop.
__device__ __forceinline__ uint32_t pg_fresh(uint32_t v) {
    asm volatile("" : "+v"(v));
    return v;
}
using pg_lds_p = __attribute__((address_space(3))) char*;
template <typename T>
__device__ __forceinline__ T pg_lds(uint32_t at) {
    return *reinterpret_cast<__attribute__((address_space(3))) T*>(at);
}

// 16 bytes a lane from memory to LDS, lane l's to dst + 16 l (dst the same in the
// wave), without a register between. As a statement of its own, so that LDS reads
// of the other buffer are not held back for it: the caller waits (pg_loads_done)
// before the barrier that hands the tile over.
__device__ __forceinline__ void pg_load_lds(uint64_t src, uint32_t dst) {
    const uint32_t base = __builtin_amdgcn_readfirstlane(dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(base), "v"(src) : "m0", "memory");
}
__device__ __forceinline__ void pg_loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- narrow items ----
// Wave w takes keys NK (4 i + w) .. of the chunk, NK = 32 (float32: 16) a step.
// Lane (g, li) = (l / 16, l % 16): the scores of row li for keys 16 c + 4 g + r
// (v_mfma_f32_16x16x32: A = K rows, B = q rows), so V^T P^T needs V of those
// keys in lane group g: the lane loads dims HD / 16 li .. of each and pairs the keys up with
// v_perm (32 for 32 keys x 128 dims, no LDS). K of the next step goes out once the scores have
// used K's registers, V's likewise; page ids are read two steps ahead. Bound by the reads: 32 tokens at up
// to 8192 binary16 positions, 241 MB, 42 us; 16 at up to 4096 in float32, 140 MB, 23 us.
template <int HD, bool F16>
__device__ __forceinline__ void paged_narrow(const PagedAttnParams& p, const PagedItem& it, float* red, uint32_t* shared) {
    constexpr uint32_t NK = pg_narrow_keys(F16) / 4u;
    constexpr int KC = NK / 16;                              // 16-key score tiles
    constexpr int QC = HD / 32;                              // 32-deep steps of q.k
    constexpr int DL = HD / 16;                              // dims of V a lane holds
    constexpr int NP = F16 ? 2 : 3;                          // parts of q and the weights
    constexpr uint32_t ES = F16 ? 2u : 4u;
    constexpr int VR = 4 * KC;                               // V rows of a lane
    constexpr int VW = DL * (int)ES / 4;                     // words of one
    const PagedParams& g = p.g;
    const uint32_t t = threadIdx.x, lane = t % kWave, g4 = lane / 16u, li = lane % 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint32_t M = it.n * p.G, hd = g.hd;
    const uint32_t kbeg = it.chunk * it.per * (4u * NK);
    const uint32_t kend = min(it.len, kbeg + it.per * (4u * NK));
    const uint32_t rr = min(li, M - 1u), tok = rr / p.G, head = it.kvh * p.G + rr % p.G;
    const float* qrow = p.q + (uint64_t)(it.row0 + tok) * p.ldq + (uint64_t)head * hd;
    const int32_t* table = g.pages + (uint64_t)it.s * g.max_pages;
    const char* kpool = reinterpret_cast<const char*>(g.k);
    const char* vpool = reinterpret_cast<const char*>(g.v);
    const uint32_t kl = lane % NK;                           // the key whose place this lane looks up

    auto page_of = [&](uint32_t k0) {                        // (past the end: some entry that is not used)
        return table[min(k0 + kl, max(kend, 1u) - 1u) / g.page_size];
    };
    // the lane's key's row (pool row 0 where it is not there), and which keys are
    auto unit_of = [&](uint32_t k0, int32_t page, uint32_t* live) {
        const uint32_t key = k0 + kl;
        const bool on = key < kend && paged_page_ok(page, g.num_pages);
        *live = (uint32_t)(__ballot(on) & ((1ull << NK) - 1ull));
        return on ? paged_row_unit(p, it.kvh, page, key % g.page_size) : it.kvh * p.head_u;
    };
    auto row_at = [&](uint32_t unit, uint32_t key) {
        return (uint64_t)(uint32_t)__builtin_amdgcn_ds_bpermute((int)(4u * key), (int)unit) << 4;
    };
    constexpr int KW = F16 ? 1 : 2;                          // 16-byte loads of 8 dims
    v4u32 kr[KC][QC][KW];
    uint32_t vr[VR][VW];
    auto load_k = [&](uint32_t unit) {
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const char* b = kpool + row_at(unit, 16u * c + li);
#pragma unroll
            for (int st = 0; st < QC; ++st) {
                const uint32_t d = 32u * st + 8u * g4;
                const char* a = b + (d < hd ? d : 0u) * ES;   // (dims past hd: q is zero there)
#pragma unroll
                for (int w = 0; w < KW; ++w) kr[c][st][w] = ld_global<v4u32>(a + 16 * w);
            }
        }
    };
    auto load_v = [&](uint32_t unit) {
        const uint32_t d = li * DL < hd ? li * DL : 0u;
#pragma unroll
        for (int b = 0; b < VR; ++b) {
            const char* a = vpool + row_at(unit, 16u * (b / 4) + 4u * g4 + b % 4) + d * ES;
            if constexpr (VW == 2) {
                const v2u32 x = ld_global<v2u32>(a);
                vr[b][0] = x[0];
                vr[b][1] = x[1];
            } else {
#pragma unroll
                for (int w = 0; w < VW / 4; ++w) {
                    const v4u32 x = ld_global<v4u32>(a + 16 * w);
#pragma unroll
                    for (int i = 0; i < 4; ++i) vr[b][4 * w + i] = x[i];
                }
            }
        }
    };

    uint32_t k0 = kbeg + wave * NK;
    int32_t page = page_of(k0), page1 = page_of(k0 + 4u * NK);
    float qv[QC][8];
#pragma unroll
    for (int st = 0; st < QC; ++st) {
        const uint32_t d = 32u * st + 8u * g4;
        const float4 a = *reinterpret_cast<const float4*>(qrow + (d < hd ? d : 0u));
        const float4 b = *reinterpret_cast<const float4*>(qrow + (d < hd ? d : 0u) + 4);
        const bool in = d < hd;
        qv[st][0] = in ? a.x : 0.f; qv[st][1] = in ? a.y : 0.f; qv[st][2] = in ? a.z : 0.f; qv[st][3] = in ? a.w : 0.f;
        qv[st][4] = in ? b.x : 0.f; qv[st][5] = in ? b.y : 0.f; qv[st][6] = in ? b.z : 0.f; qv[st][7] = in ? b.w : 0.f;
    }
    uint32_t live, live1;
    uint32_t unit = unit_of(k0, page, &live);
    load_k(unit);
    load_v(unit);
    v4u32 qp[NP][QC];
    float qf = p.scale * 1.4426950408889634f;                // scores in log2 units
    {
        float amax = 0.f;
#pragma unroll
        for (int st = 0; st < QC; ++st)
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(qv[st][i]));
        int e = 0;
        if constexpr (F16) {
            (void)frexpf(max_row_slots(amax), &e);
            e -= 15;
            qf *= ldexpf(1.f, e);
        }
#pragma unroll
        for (int st = 0; st < QC; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[3];
                if constexpr (F16) pg_split2(ldexpf(qv[st][2 * i], -e), ldexpf(qv[st][2 * i + 1], -e), &w[0], &w[1]);
                else pg_cut2(qv[st][2 * i], qv[st][2 * i + 1], &w[0], &w[1], &w[2]);
#pragma unroll
                for (int a = 0; a < NP; ++a) qp[a][st][i] = w[a];
            }
    }
    const int64_t qpos64 = it.pos0 + (int64_t)tok;
    const int32_t qpos = (int32_t)max((int64_t)-1, min(qpos64, (int64_t)0x7FFFFFFF));
    constexpr float kBoost = F16 ? 15.f : 0.f;               // weights times 2^15 (binary16's range)
    float m = -INFINITY, l = 0.f;
    pg_f4 o[DL];
#pragma unroll
    for (int e = 0; e < DL; ++e) o[e] = pg_f4{0.f, 0.f, 0.f, 0.f};

    for (; k0 < kend; k0 += 4u * NK) {
        const int32_t page2 = page_of(k0 + 8u * NK);
        // ---- scores ----
        pg_f4 sacc[KC];
#pragma unroll
        for (int c = 0; c < KC; ++c) sacc[c] = pg_f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < QC; ++st) {
            if constexpr (F16) {
#pragma unroll
                for (int a = 0; a < 2; ++a)
#pragma unroll
                    for (int c = 0; c < KC; ++c)
                        sacc[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_half8, kr[c][st][0]),
                                                                         __builtin_bit_cast(pg_half8, qp[a][st]), sacc[c], 0, 0, 0);
            } else {
                v4u32 kp[3];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[3];
                    const v4u32 x = kr[0][st][i / 2];
                    pg_cut2(__uint_as_float(x[2 * (i % 2)]), __uint_as_float(x[2 * (i % 2) + 1]), &w[0], &w[1], &w[2]);
#pragma unroll
                    for (int a = 0; a < 3; ++a) kp[a][i] = w[a];
                }
#pragma unroll
                for (int a = 2; a >= 0; --a)
#pragma unroll
                    for (int b = 2 - a; b >= 0; --b)
                        sacc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pg_bf8, kp[a]),
                                                                          __builtin_bit_cast(pg_bf8, qp[b][st]), sacc[0], 0, 0, 0);
            }
        }
        const uint32_t k1 = k0 + 4u * NK;
        const uint32_t unit1 = unit_of(k1, page1, &live1);
        load_k(unit1);
        // ---- masks: keys that are not there, and rows before a key ----
        const uint32_t all = (uint32_t)((1ull << NK) - 1ull);
        const bool full = live == all && (int64_t)(k0 + NK - 1u) <= it.pos0;
        float sv[KC][4];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) sv[c][r] = sacc[c][r] * qf;
        if (!full) {
#pragma unroll
            for (int c = 0; c < KC; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t key = 16u * c + 4u * g4 + r;
                    if (!((live >> key) & 1u) || (int32_t)(k0 + key) > qpos) sv[c][r] = -INFINITY;
                }
        }
        // ---- running softmax of row li ----
        float mx = sv[0][0];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = fmaxf(mx, sv[c][r]);
        mx = max_row_slots(mx);
        const float mn = fmaxf(m, mx);
        const float mref = mn == -INFINITY ? 0.f : mn;
        if (__ballot(mn > m)) {
            const float f = __builtin_amdgcn_exp2f(m - mref);
            l *= f;
#pragma unroll
            for (int e = 0; e < DL; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[e][r] *= f;
        }
        m = mn;
        float ev[KC][4];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                ev[c][r] = __builtin_amdgcn_exp2f(sv[c][r] - mref + kBoost);
                l += ev[c][r];
            }
        // ---- values: rows nobody sees read as zero; a row that only some see must not
        // meet the others' zero weights when it is not finite ----
        if (!full) {
            uint32_t bad = 0;
#pragma unroll
            for (int b = 0; b < VR; ++b) {
                const uint32_t key = 16u * (b / 4) + 4u * g4 + b % 4;
                const bool on = (live >> key) & 1u;
                bool nf = false;
#pragma unroll
                for (int w = 0; w < VW; ++w) {
                    vr[b][w] = on ? vr[b][w] : 0u;
                    nf = nf || pg_not_finite<F16>(vr[b][w]);
                }
                // (a lane past hd holds dims 0 ..: the same row)
                const uint64_t who = __ballot(nf && (int64_t)(k0 + key) > it.pos0);
#pragma unroll
                for (int gg = 0; gg < 4; ++gg)
                    if ((who >> (16 * gg)) & 0xFFFFull) bad |= 1u << (16 * (b / 4) + 4 * gg + b % 4);
            }
            if (bad) {
#pragma unroll
                for (int b = 0; b < VR; ++b)
                    if ((bad >> (16u * (b / 4) + 4u * g4 + b % 4)) & 1u)
#pragma unroll
                        for (int w = 0; w < VW; ++w) vr[b][w] = 0u;
                for (uint32_t rest = bad; rest; rest &= rest - 1u) {
                    const uint32_t key = (uint32_t)__builtin_ctz(rest);
                    float mine = 0.f;
#pragma unroll
                    for (int c = 0; c < KC; ++c)
#pragma unroll
                        for (int r = 0; r < 4; ++r) mine = (uint32_t)(4 * c + r) == 4u * (key / 16u) + key % 4u ? ev[c][r] : mine;
                    const float w = __shfl(mine, (int)(16u * ((key % 16u) / 4u) + li), kWave);
                    const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)unit, (int)key);
                    if ((int32_t)(k0 + key) <= qpos) {
#pragma unroll
                        for (int e = 0; e < DL; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const uint32_t d = DL * (4u * g4 + r) + e;
                                if (d < hd) o[e][r] = fmaf(w, pg_value<F16>(g.v, at, d), o[e][r]);
                            }
                    }
                }
            }
        }
        // ---- O^T += V^T P^T ----
        if constexpr (F16) {
            v4u32 pp[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t h, w;
                pg_split2(ev[i / 2][2 * (i % 2)], ev[i / 2][2 * (i % 2) + 1], &h, &w);
                pp[0][i] = h;
                pp[1][i] = w;
            }
#pragma unroll
            for (int e2 = 0; e2 < DL / 2; ++e2) {
                v4u32 v0, v1;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v0[i] = __builtin_amdgcn_perm(vr[2 * i + 1][e2], vr[2 * i][e2], 0x05040100u);
                    v1[i] = __builtin_amdgcn_perm(vr[2 * i + 1][e2], vr[2 * i][e2], 0x07060302u);
                }
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    const pg_half8 pb = __builtin_bit_cast(pg_half8, pp[a]);
                    o[2 * e2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_half8, v0), pb, o[2 * e2], 0, 0, 0);
                    o[2 * e2 + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pg_half8, v1), pb, o[2 * e2 + 1], 0, 0, 0);
                }
            }
        } else {
            v2u32 pp[3];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t w[3];
                pg_cut2(ev[0][2 * i], ev[0][2 * i + 1], &w[0], &w[1], &w[2]);
#pragma unroll
                for (int a = 0; a < 3; ++a) pp[a][i] = w[a];
            }
#pragma unroll
            for (int e = 0; e < DL; ++e) {
                v2u32 vp[3];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    uint32_t w[3];
                    pg_cut2(__uint_as_float(vr[2 * i][e]), __uint_as_float(vr[2 * i + 1][e]), &w[0], &w[1], &w[2]);
#pragma unroll
                    for (int a = 0; a < 3; ++a) vp[a][i] = w[a];
                }
#pragma unroll
                for (int a = 2; a >= 0; --a)
#pragma unroll
                    for (int b = 2 - a; b >= 0; --b)
                        o[e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(pg_s4, vp[a]),
                                                                         __builtin_bit_cast(pg_s4, pp[b]), o[e], 0, 0, 0);
            }
        }
        load_v(unit1);
        unit = unit1;
        live = live1;
        page1 = page2;
    }

    // ---- the four waves' states: thread = row t / 16, dims DL (t % 16) .. ----
    constexpr uint32_t LD = HD + 4;                          // padded LDS row
    float* rm = red + 4u * 16u * LD;                         // [wave][row] m, then l
    l = sum_row_slots(l);
#pragma unroll
    for (int e = 0; e < DL; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) red[(wave * 16u + li) * LD + DL * (4u * g4 + r) + e] = o[e][r];
    if (g4 == 0) {
        rm[wave * 16u + li] = m;
        rm[64u + wave * 16u + li] = l;
    }
    __syncthreads();
    const uint32_t row = t / 16u, d0 = DL * (t % 16u);
    float M0 = -INFINITY, L0 = 0.f, acc[DL];
#pragma unroll
    for (int w = 0; w < 4; ++w) M0 = fmaxf(M0, rm[w * 16u + row]);
    const float mr = M0 == -INFINITY ? 0.f : M0;
#pragma unroll
    for (int d = 0; d < DL; ++d) acc[d] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = __builtin_amdgcn_exp2f(rm[w * 16u + row] - mr);
        L0 = fmaf(f, rm[64u + w * 16u + row], L0);
#pragma unroll
        for (int d = 0; d < DL; ++d) acc[d] = fmaf(f, red[(w * 16u + row) * LD + d0 + d], acc[d]);
    }
    if (it.chunks > 1u) {
        const uint32_t stride = it.tiles * g.KVH;            // items of a tile's neighbouring chunks
        auto state = [&](uint32_t c) { return p.part + (uint64_t)(it.state + c * stride) * p.part_floats; };
        if (row < M) {
            float* d = state(it.chunk);
#pragma unroll
            for (int i = 0; i < DL; i += 2) pg_put2(d + row * HD + d0 + i, acc[i], acc[i + 1]);
            if (t % 16u == 0) pg_put2(d + 16u * HD + 2u * row, M0, L0);
        }
        if (!paged_arrive(p.count + it.first, it.chunks, shared)) return;
        if (row >= M) return;
        // eight states in flight at a time, with a running maximum
        constexpr uint32_t B = 8;
        float mx = -INFINITY;
        L0 = 0.f;
#pragma unroll
        for (int d = 0; d < DL; ++d) acc[d] = 0.f;
        for (uint32_t c0 = 0; c0 < it.chunks; c0 += B) {
            float2 ml[B], x[B][DL / 2];
#pragma unroll
            for (uint32_t c = 0; c < B; ++c) {
                const float* b = state(min(c0 + c, it.chunks - 1u));
                ml[c] = pg_get2(b + 16u * HD + 2u * row);
#pragma unroll
                for (int i = 0; i < DL / 2; ++i) x[c][i] = pg_get2(b + row * HD + d0 + 2 * i);
            }
            float mn = mx;
#pragma unroll
            for (uint32_t c = 0; c < B; ++c) mn = fmaxf(mn, ml[c].x);
            const float mf = mn == -INFINITY ? 0.f : mn, g0 = __builtin_amdgcn_exp2f(mx - mf);
            mx = mn;
            L0 *= g0;
#pragma unroll
            for (int d = 0; d < DL; ++d) acc[d] *= g0;
#pragma unroll
            for (uint32_t c = 0; c < B; ++c) {
                if (c0 + c >= it.chunks) break;
                const float f = __builtin_amdgcn_exp2f(ml[c].x - mf);
                L0 = fmaf(f, ml[c].y, L0);
#pragma unroll
                for (int i = 0; i < DL / 2; ++i) {
                    acc[2 * i] = fmaf(f, x[c][i].x, acc[2 * i]);
                    acc[2 * i + 1] = fmaf(f, x[c][i].y, acc[2 * i + 1]);
                }
            }
        }
    }
    if (row >= M || d0 >= hd) return;
    const float inv = L0 == 0.f ? 0.f : 1.0f / L0;           // a row that sees nothing: zeros
    float* out = p.out + (uint64_t)(it.row0 + row / p.G) * p.ldo + (uint64_t)(it.kvh * p.G + row % p.G) * hd + d0;
#pragma unroll
    for (int i = 0; i < DL; i += 4)
        *reinterpret_cast<float4*>(out + i) = make_float4(acc[i] * inv, acc[i + 1] * inv, acc[i + 2] * inv, acc[i + 3] * inv);
}

// ---- wide items ----
// Wave w holds rows 32 w .. of the tile as columns of 32 x 32 products: S^T = K Q^T
// (v_mfma_f32_32x32x16), lane (h, c) = (l / 32, l % 32) with row c's scores of keys
// 8 j + 4 h + r, then O^T += V^T P^T with V^T from transposing LDS reads
// (ds_read_b64_tr_b16: 4 keys x 16 dims of a row-major tile). Over a binary16 cache the tile
// goes from the cache to LDS past the registers, one tile ahead, two buffers and one barrier
// a tile; a float32 tile is loaded into registers a tile ahead and split into two binary16 parts
// a key on the way to LDS. 16-byte pieces of an LDS row are permuted by the row so that neither the
// reads of 32 keys' pieces nor the transposing reads of 4 keys meet in a bank.
// What bounds a chunk of 512 rows over 8192 keys is the matrix cores' two (three) products and
// the softmax's vector instructions beside them, about as many cycles: 71 us over a binary16 cache,
// 0.94 PFLOP/s of products (a large library product: 1.07). 64-row tiles would read each
// LDS piece for half the products, which is all the LDS can give.
template <int HD>
__device__ __forceinline__ uint32_t pg_swz_k(uint32_t row) {
    return HD == 128 ? row & 15u : (row >> 1) & 7u;
}
template <int HD>
__device__ __forceinline__ uint32_t pg_swz_v(uint32_t row) {
    return HD == 128 ? ((row & 3u) << 2) | ((row >> 2) & 3u) : (((row >> 1) & 1u) << 2) | ((row >> 2) & 3u);
}

template <int HD, bool F16>
__device__ __forceinline__ void paged_wide(const PagedAttnParams& p, const PagedItem& it, char* smem, uint32_t* shared) {
    constexpr uint32_t KT = pg_wide_keys(F16);
    constexpr int KB = KT / 32;                              // 32-key score tiles
    constexpr int QS = HD / 16;                              // 16-deep steps of q.k
    constexpr int OD = HD / 32;                              // 32-dim output tiles
    constexpr int KP = F16 ? 1 : 2;                          // parts of k and v (two of q and the weights)
    constexpr uint32_t ES = F16 ? 2u : 4u;
    constexpr uint32_t CPR = HD / 8;                         // 16-byte pieces of an LDS row
    constexpr uint32_t TB = KT * HD * 2u;                    // bytes of a tile part in LDS
    const PagedParams& g = p.g;
    const uint32_t t = threadIdx.x, lane = t % kWave, h = lane / 32u, li = lane % 32u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t / kWave);
    const uint64_t M = (uint64_t)it.n * p.G;
    const uint32_t hd = g.hd;
    const uint32_t r0 = it.tile * kPgWideRows;               // first flattened row of the tile
    const uint32_t nrow = (uint32_t)min((uint64_t)kPgWideRows, M - r0);
    // keys that the tile's last row sees bound its chunks
    const int64_t last_pos = it.pos0 + (int64_t)((r0 + nrow - 1u) / p.G);
    const uint32_t klen = (uint32_t)max((int64_t)0, min((int64_t)it.len, last_pos + 1));
    const uint32_t ckeys = it.per * KT;                      // (at most the sequence's keys and a step: 32 bits)
    const uint32_t lives = max(1u, (klen + ckeys - 1u) / ckeys);
    if (it.chunk >= lives) return;
    const uint32_t kbeg = it.chunk * ckeys, kend = min(klen, kbeg + ckeys);
    const bool wave_on = wave * 32u < nrow;
    const uint32_t rr = r0 + min(wave * 32u + li, nrow - 1u);
    const uint32_t tok = rr / p.G, head = it.kvh * p.G + rr % p.G;
    const float* qrow = p.q + (uint64_t)(it.row0 + tok) * p.ldq + (uint64_t)head * hd;
    const int32_t* table = g.pages + (uint64_t)it.s * g.max_pages;
    const int64_t first_pos = it.pos0 + (int64_t)((r0 + min(wave * 32u, nrow - 1u)) / p.G);   // of the wave's rows
    const int32_t qpos = (int32_t)max((int64_t)-1, min(it.pos0 + (int64_t)tok, (int64_t)0x7FFFFFFF));

    const uint32_t kl = lane % KT;
    auto page_of = [&](uint32_t k0) { return table[min(k0 + kl, max(kend, 1u) - 1u) / g.page_size]; };
    auto unit_of = [&](uint32_t k0, int32_t page, uint64_t* live) {
        const uint32_t key = k0 + kl;
        const bool on = key < kend && paged_page_ok(page, g.num_pages);
        *live = __ballot(on) & (KT == 64u ? ~0ull : (1ull << (KT % 64u)) - 1ull);
        return on ? paged_row_unit(p, it.kvh, page, key % g.page_size) : it.kvh * p.head_u;
    };
    const uint32_t kt0 = (uint32_t)(uintptr_t)(pg_lds_p)smem;   // binary16: [buffer]; float32: [part]
    const uint32_t vt0 = kt0 + 2u * TB;
    float* const kexp = reinterpret_cast<float*>(smem + 4u * TB);   // float32: 2^e of each key's k, then e of its v
    float* const vexp = kexp + KT;
    constexpr int NL = (int)(KT * HD * ES / 16u / 256u);     // 16-byte pieces of K (and V) a thread moves
    v4u32 kreg[F16 ? 1 : NL], vreg[F16 ? 1 : NL];
    auto load_tile = [&](uint32_t unit, uint32_t buf) {
        const uint32_t ln = pg_fresh(lane);
#pragma unroll
        for (int j = 0; j < NL; ++j) {
            constexpr uint32_t PR = F16 ? CPR : HD / 4;       // pieces of a cache row
            constexpr uint32_t RW = kWave / PR;               // rows of 64 pieces
            const uint32_t row = (wave * NL + (uint32_t)j) * RW + ln / PR, c = ln % PR;
            const uint32_t u = (uint32_t)__builtin_amdgcn_ds_bpermute((int)(4u * row), (int)unit);
            if constexpr (F16) {
                // LDS takes a wave's pieces in lane order: the permutation is in which piece a lane loads
                uint32_t ck = c ^ pg_swz_k<HD>(row), cv = c ^ pg_swz_v<HD>(row);
                ck = 8u * ck < hd ? ck : 0u;
                cv = 8u * cv < hd ? cv : 0u;
                const uint32_t d = buf * TB + (wave * NL + (uint32_t)j) * 1024u;
                pg_load_lds((uint64_t)g.k + ((uint64_t)(u + ck) << 4), kt0 + d);
                pg_load_lds((uint64_t)g.v + ((uint64_t)(u + cv) << 4), vt0 + d);
            } else {
                const uint64_t at = (uint64_t)(u + (4u * c < hd ? c : 0u)) << 4;
                kreg[j] = ld_global<v4u32>(reinterpret_cast<const char*>(g.k) + at);
                vreg[j] = ld_global<v4u32>(reinterpret_cast<const char*>(g.v) + at);
            }
        }
    };
    // float32: a row's HD / 4 lanes share its exponent (of its largest finite value), then two parts of four dims
    auto store_tile = [&]() {
        if constexpr (!F16) {
            const uint32_t ln = pg_fresh(lane);
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                constexpr uint32_t PR = HD / 4, RW = kWave / PR;
                const uint32_t row = (wave * NL + (uint32_t)j) * RW + ln / PR, c = ln % PR;
                const uint32_t ak = kt0 + (row * CPR + ((c / 2u) ^ pg_swz_k<HD>(row))) * 16u + (c % 2u) * 8u;
                const uint32_t av = vt0 + (row * CPR + ((c / 2u) ^ pg_swz_v<HD>(row))) * 16u + (c % 2u) * 8u;
                auto put = [&](const v4u32& x, uint32_t at) {
                    // (magnitudes compare as integers; a row that holds a value that is not finite looks again without those)
                    auto most = [&](uint32_t lim) {
                        uint32_t u = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t y = pg_word(x, i) & 0x7FFFFFFFu;
                            u = max(u, y < lim ? y : 0u);
                        }
                        return pg_group_max<PR>(u);
                    };
                    uint32_t u = most(~0u);
                    if (__ballot(u >= 0x7F800000u)) u = most(0x7F800000u);
                    const int e = max((int)(u >> 23) - 141, -100);   // |v| 2^-e < 2^15 (smaller rows: 2^-100 stays in range)
                    uint32_t a[2], b[2];
                    pg_split2(ldexpf(__uint_as_float(pg_word(x, 0)), -e), ldexpf(__uint_as_float(pg_word(x, 1)), -e), &a[0], &a[1]);
                    pg_split2(ldexpf(__uint_as_float(pg_word(x, 2)), -e), ldexpf(__uint_as_float(pg_word(x, 3)), -e), &b[0], &b[1]);
#pragma unroll
                    for (uint32_t q = 0; q < 2; ++q)
                        *reinterpret_cast<__attribute__((address_space(3))) v2u32*>(at + q * TB) = v2u32{a[q], b[q]};
                    return e;
                };
                const int ek = put(kreg[j], ak), ev = put(vreg[j], av);
                if (c == 0) {
                    kexp[row] = ldexpf(1.f, ek);
                    vexp[row] = (float)ev;
                }
            }
        }
    };

    int32_t page = page_of(kbeg), page1 = page_of(kbeg + KT);
    v4u32 qp[2][QS];
    float qf = p.scale * 1.4426950408889634f;
    {
        float qv[QS][8], amax = 0.f;
#pragma unroll
        for (int st = 0; st < QS; ++st) {
            const uint32_t d = 16u * st + 8u * h;
            const bool in = d < hd;
            const float4 a = *reinterpret_cast<const float4*>(qrow + (in ? d : 0u));
            const float4 b = *reinterpret_cast<const float4*>(qrow + (in ? d : 0u) + 4);
            qv[st][0] = in ? a.x : 0.f; qv[st][1] = in ? a.y : 0.f; qv[st][2] = in ? a.z : 0.f; qv[st][3] = in ? a.w : 0.f;
            qv[st][4] = in ? b.x : 0.f; qv[st][5] = in ? b.y : 0.f; qv[st][6] = in ? b.z : 0.f; qv[st][7] = in ? b.w : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(qv[st][i]));
        }
        int e = 0;
        amax = fmaxf(amax, __shfl_xor(amax, 32, kWave));
        (void)frexpf(amax, &e);
        e = max(e - 15, -100);
        qf *= ldexpf(1.f, e);
#pragma unroll
        for (int st = 0; st < QS; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t hi, lo;
                pg_split2(ldexpf(qv[st][2 * i], -e), ldexpf(qv[st][2 * i + 1], -e), &hi, &lo);
                qp[0][st][i] = hi;
                qp[1][st][i] = lo;
            }
    }
    // Weights go into the products times 2^15 (binary16's range). Over a float32 cache each key's values have an
    // exponent of their own, which its weight takes on: 2^(score + e_v - top + 15), top the row's running maximum of
    // score + e_v over the keys it sees, so that no key, however large, costs another its bits.
    constexpr float kBoost = 15.f;
    float m = -INFINITY, top = -INFINITY, l = 0.f;
    pg_f16 o[OD];
#pragma unroll
    for (int d = 0; d < OD; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = 0.f;

    uint64_t live, live1 = 0;
    uint32_t unit = unit_of(kbeg, page, &live);
    // (nothing may be on its way to LDS when the workgroup ends: a tile of rows at negative positions only has no keys)
    if (kbeg < kend) load_tile(unit, 0);
    uint32_t buf = 0;
    // LDS places: K piece 2 st + h of key li is at kl0 ^ 32 st; the V piece of dim tile d, keys 8 j .. (with the
    // lane's part of them) at vl0 ^ (64 d + 32 j), rows further by whole rows
    const uint32_t kl0 = (li * CPR + (h ^ pg_swz_k<HD>(li))) * 16u;
    const uint32_t l16 = lane % 16u, vrow = 4u * h + l16 / 4u;
    const uint32_t vl0 = (vrow * CPR + ((2u * ((lane / 16u) % 2u) + (l16 % 4u) / 2u) ^ pg_swz_v<HD>(vrow))) * 16u + (l16 % 2u) * 8u;
    auto v_frag = [&](uint32_t vl, int t4, int d) {
        v4u32 a;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t at = (vl ^ (64u * d + 32u * j)) + (16u * t4 + 8u * j) * CPR * 16u;
            const v2u32 x = __builtin_bit_cast(v2u32, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                          reinterpret_cast<__attribute__((address_space(3))) pg_s4*>(at)));
            a[2 * j] = x[0];
            a[2 * j + 1] = x[1];
        }
        return a;
    };
    for (uint32_t k0 = kbeg; k0 < kend; k0 += KT) {
        if constexpr (!F16) {
            __syncthreads();                                 // the previous tile is consumed
            store_tile();
        }
        if constexpr (F16) pg_loads_done();
        __syncthreads();
        const int32_t page2 = page_of(k0 + 2u * KT);
        const uint32_t unit1 = unit_of(k0 + KT, page1, &live1);
        if (k0 + KT < kend) load_tile(unit1, buf ^ 1u);
        const uint32_t kt = kt0 + (F16 ? buf * TB : 0u);
        const uint32_t vt = vt0 + (F16 ? buf * TB : 0u);
        const uint64_t live_now = live;
        const uint32_t unit_now = unit;
        buf ^= 1u;
        unit = unit1;
        live = live1;
        page1 = page2;
        if (!wave_on) continue;
        // ---- scores ----
        const uint32_t kl = kt + pg_fresh(kl0);             // (a multiple of 128 bytes apart: the pieces' bits stay free)
        pg_f16 sacc[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) sacc[b][v] = 0.f;
#pragma unroll
        for (int st = 0; st < QS; ++st) {
            v4u32 kf[KP][KB];
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const uint32_t at = (kl ^ (32u * st)) + 32u * b * CPR * 16u;
#pragma unroll
                for (int q = 0; q < KP; ++q) kf[q][b] = pg_lds<v4u32>(at + q * TB);
            }
            auto mm = [&](const v4u32* k, const v4u32& q) {
#pragma unroll
                for (int b = 0; b < KB; ++b)
                    sacc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pg_half8, k[b]),
                                                                     __builtin_bit_cast(pg_half8, q), sacc[b], 0, 0, 0);
            };
            mm(kf[0], qp[0][st]);
            if constexpr (KP == 2) mm(kf[1], qp[0][st]);
            mm(kf[0], qp[1][st]);
        }
        // float32: the keys' own scales, and their values' exponents
        float ve[F16 ? 1 : 16];
        const float qs = F16 ? qf : 1.f;
        if constexpr (!F16) {
#pragma unroll
            for (int v = 0; v < 16; v += 4) {
                const float4 ks = *reinterpret_cast<const float4*>(kexp + 2 * v + 4u * h);
                const float4 vs = *reinterpret_cast<const float4*>(vexp + 2 * v + 4u * h);
                sacc[0][v] *= ks.x * qf; sacc[0][v + 1] *= ks.y * qf; sacc[0][v + 2] *= ks.z * qf; sacc[0][v + 3] *= ks.w * qf;
                ve[v] = vs.x; ve[v + 1] = vs.y; ve[v + 2] = vs.z; ve[v + 3] = vs.w;
            }
        }
        // ---- masks and running softmax of row li: keys 32 b + 8 (v / 4) + 4 h + v % 4 ----
        const uint64_t all = KT == 64u ? ~0ull : (1ull << (KT % 64u)) - 1ull;
        const bool full = live_now == all && (int64_t)(k0 + KT - 1u) <= first_pos;
        if (!full) {
            const uint32_t h4 = 4u * pg_fresh(h);
            const uint64_t there = live_now >> h4;
            // keys up to the row's position
            const int64_t reach = (int64_t)qpos - (int64_t)k0 - (int64_t)h4;
            const int32_t most = (int32_t)max((int64_t)-1, min(reach, (int64_t)64));
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int v = 0; v < 16; ++v) {
                    const int key = 32 * b + 8 * (v / 4) + v % 4;
                    const bool on = ((there >> key) & 1ull) && key <= most;
                    sacc[b][v] = on ? sacc[b][v] : -INFINITY;
                }
        }
        float mx = sacc[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int v = 0; v < 16; ++v) mx = fmaxf(mx, sacc[b][v]);
        {
            const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])) * qs;
        }
        const float mn = fmaxf(m, mx);
        const float mref = mn == -INFINITY ? 0.f : mn;
        float tn = mn;                                       // the weights' own maximum
        if constexpr (!F16) {
            float tx = sacc[0][0] + ve[0];
#pragma unroll
            for (int v = 1; v < 16; ++v) tx = fmaxf(tx, sacc[0][v] + ve[v]);
            const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(tx), __float_as_uint(tx), false, false);
            tn = fmaxf(top, fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1])));
        }
        const float tref = tn == -INFINITY ? 0.f : tn;
        if (__ballot(tn > top || mn > m)) {
            const float f = __builtin_amdgcn_exp2f(top - tref);
            l *= __builtin_amdgcn_exp2f(m - mref);
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[d][v] *= f;
        }
        m = mn;
        top = tn;
        const float shift = kBoost - tref;                   // a weight on its values' scale: 2^(score qs + shift)
        // ---- values: keys nobody sees read as zero, and a key that only some of the rows see
        // must not meet the others' zero weights when its values are not finite ----
        const uint32_t vl = vt + pg_fresh(vl0);
        uint64_t use = all;
        if (!full) {
            use = live_now;
            uint64_t bad = 0;
            // keys past the wave's first row
            const int64_t ahead = first_pos + 1 - (int64_t)k0;
            const uint64_t later = ahead >= 64 ? 0ull : ahead <= 0 ? ~0ull : ~0ull << ahead;
            if (use & later) {
#pragma unroll
                for (int t4 = 0; t4 < 2 * KB; ++t4)
#pragma unroll
                    for (int d = 0; d < OD; ++d) {
                        const v4u32 a = v_frag(vl, t4, d);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            // (a float32's first part carries it)
                            const uint32_t x = (a[i / 2] >> (16 * (i % 2))) & 0x7C00u;
                            const uint64_t who = __ballot(x == 0x7C00u);
                            const uint32_t key = 16u * t4 + 8u * (i / 4) + i % 4;
                            if (who & 0xFFFFFFFFull) bad |= 1ull << key;
                            if (who >> 32) bad |= 1ull << (key + 4u);
                        }
                    }
                bad &= use & later;
                use &= ~bad;
                for (uint64_t rest = bad; rest; rest &= rest - 1ull) {
                    const uint32_t key = (uint32_t)__builtin_ctzll(rest);
                    const uint32_t want = (key / 16u) * 8u + 4u * ((key % 16u) / 8u) + key % 4u;   // register of the weight
                    float mine = 0.f;
                    const float sh = __uint_as_float(pg_fresh(__float_as_uint(shift)));
#pragma unroll
                    for (int b = 0; b < KB; ++b)
#pragma unroll
                        for (int v = 0; v < 16; ++v) {
                            const float e = __builtin_amdgcn_exp2f(fmaf(sacc[b][v], qs, sh));
                            mine = (uint32_t)(16 * b + v) == want ? e : mine;
                        }
                    const float w = __shfl(mine, (int)(32u * ((key / 4u) % 2u) + li), kWave);
                    const uint32_t at = (uint32_t)__builtin_amdgcn_readlane((int)unit_now, (int)key);
                    if ((int32_t)(k0 + key) <= qpos) {
                        const uint32_t hf = 4u * pg_fresh(h);
#pragma unroll
                        for (int d = 0; d < OD; ++d)
#pragma unroll
                            for (int v = 0; v < 16; ++v) {
                                const uint32_t dim = 32u * d + 8u * (v / 4) + hf + v % 4;
                                if (dim < hd) o[d][v] = fmaf(w, pg_value<F16>(g.v, at, dim), o[d][v]);
                                __builtin_amdgcn_sched_barrier(0);   // (rare: one value in a register at a time)
                            }
                    }
                }
            }
        }
        v4u32 pp[2][2 * KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            float ls = 0.f;
#pragma unroll
            for (int v = 0; v < 16; v += 2) {
                float e[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if constexpr (F16) {
                        e[i] = __builtin_amdgcn_exp2f(fmaf(sacc[b][v + i], qs, shift));
                        ls += e[i];
                    } else {
                        ls += __builtin_amdgcn_exp2f(sacc[b][v + i] - mref);
                        e[i] = __builtin_amdgcn_exp2f(sacc[b][v + i] + ve[v + i] + shift);
                    }
                }
                uint32_t hi, lo;
                pg_split2(e[0], e[1], &hi, &lo);
                pp[0][2 * b + v / 8][(v % 8) / 2] = hi;
                pp[1][2 * b + v / 8][(v % 8) / 2] = lo;
            }
            l += ls;
        }
        // ---- O^T += V^T P^T ----
        // (one copy of this for whole and for masked tiles: two took the registers of q)
        const uint64_t there = use >> (4u * h);
#pragma unroll
        for (int t4 = 0; t4 < 2 * KB; ++t4) {
            v4u32 keep = {~0u, ~0u, ~0u, ~0u};
            constexpr int DG = KP == 1 || OD == 1 ? OD : OD / 2;   // dim tiles whose pieces are in registers at a time
#pragma unroll
            for (int d0 = 0; d0 < OD; d0 += DG) {
                v4u32 a[DG][KP];
#pragma unroll
                for (int d = 0; d < DG; ++d)
#pragma unroll
                    for (int q = 0; q < KP; ++q) a[d][q] = v_frag(vl + q * TB, t4, d0 + d);
                if (use != all) {
                    if (d0 == 0) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const uint32_t key = 16u * t4 + 8u * (i / 4) + i % 4;
                            if (!((there >> key) & 1ull)) keep[i / 2] &= i % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                        }
                    }
#pragma unroll
                    for (int d = 0; d < DG; ++d)
#pragma unroll
                        for (int q = 0; q < KP; ++q) a[d][q] &= keep;
                }
                auto mm = [&](int q, const v4u32& w) {
#pragma unroll
                    for (int d = 0; d < DG; ++d)
                        o[d0 + d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(pg_half8, a[d][q]),
                                                                           __builtin_bit_cast(pg_half8, w), o[d0 + d], 0, 0, 0);
                };
                mm(0, pp[0][t4]);
                if constexpr (KP == 2) mm(1, pp[0][t4]);
                mm(0, pp[1][t4]);
            }
        }
    }
    if constexpr (!F16) {
        // from the values' scale to the weights' 2^(score - m)
        const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(top - kBoost - m);
#pragma unroll
        for (int d = 0; d < OD; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d][v] *= f;
    }
    {
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = __uint_as_float(w[0]) + __uint_as_float(w[1]);
    }
    if (lives > 1u) {
        // states in lane order: piece (wave, j) of 64 lanes x 16 bytes, then m, l a lane
        constexpr uint32_t NJ = HD / 8;
        const uint32_t stride = it.tiles * g.KVH;
        auto state = [&](uint32_t c) { return p.part + (uint64_t)(it.state + c * stride) * p.part_floats; };
        if (wave_on) {
            float* b = state(it.chunk);
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float* x = b + ((wave * NJ + 4u * d + q) * kWave + lane) * 4u;
                    pg_put2(x, o[d][4 * q], o[d][4 * q + 1]);
                    pg_put2(x + 2, o[d][4 * q + 2], o[d][4 * q + 3]);
                }
            pg_put2(b + kPgWideRows * HD + (wave * kWave + lane) * 2u, m, l);
        }
        if (!paged_arrive(p.count + it.first, lives, shared)) return;
        if (!wave_on) return;
        // a state at a time (its loads together), with a running maximum
        float mx = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int d = 0; d < OD; ++d)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
        for (uint32_t c = 0; c < lives; ++c) {
            const float* b = state(c);
            const float2 ml = pg_get2(b + kPgWideRows * HD + (wave * kWave + lane) * 2u);
            float2 x[OD][8];
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float* y = b + ((wave * NJ + 4u * d + q) * kWave + lane) * 4u;
                    x[d][2 * q] = pg_get2(y);
                    x[d][2 * q + 1] = pg_get2(y + 2);
                }
            const float mn = fmaxf(mx, ml.x), mf = mn == -INFINITY ? 0.f : mn;
            const float f0 = __builtin_amdgcn_exp2f(mx - mf), f = __builtin_amdgcn_exp2f(ml.x - mf);
            mx = mn;
            l = fmaf(f, ml.y, l * f0);
#pragma unroll
            for (int d = 0; d < OD; ++d)
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    o[d][2 * q] = fmaf(f, x[d][q].x, o[d][2 * q] * f0);
                    o[d][2 * q + 1] = fmaf(f, x[d][q].y, o[d][2 * q + 1] * f0);
                }
        }
    }
    if (!wave_on || wave * 32u + li >= nrow) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;             // a row that sees nothing: zeros
    float* out = p.out + (uint64_t)(it.row0 + tok) * p.ldo + (uint64_t)head * hd;
#pragma unroll
    for (int d = 0; d < OD; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t dim = 32u * d + 8u * q + 4u * h;
            if (dim < hd)
                *reinterpret_cast<float4*>(out + dim) =
                    make_float4(o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv);
        }
}

// WIDE false: every sequence has at most 16 rows a KV head (single tokens), and
// the kernel is built without the wide items' registers and LDS.
template <int HD, bool F16, bool WIDE, bool MANY>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedAttnParams p) {
    constexpr uint32_t kNarrowLds = (4u * 16u * (HD + 4u) + 128u) * 4u;
    constexpr uint32_t kWideLds = 4u * pg_wide_keys(F16) * HD * 2u + (F16 ? 0u : pg_wide_keys(F16) * 8u);
    __shared__ __align__(256) char smem[WIDE && kWideLds > kNarrowLds ? kWideLds : kNarrowLds];
    __shared__ uint32_t shared;
    __shared__ PagedPlanLds plan;
    PagedItem it;
    if (!paged_item<MANY>(p, blockIdx.x, &it, &plan)) return;
    if constexpr (WIDE) {
        if (!it.narrow) {
            paged_wide<HD, F16>(p, it, smem, &shared);
            return;
        }
    } else if (!it.narrow) {
        return;
    }
    paged_narrow<HD, F16>(p, it, reinterpret_cast<float*>(smem), &shared);
}

}  // namespace qora
