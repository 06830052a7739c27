// The paged cache's argument checks and index arithmetic on the CPU: random
// small pools against a brute-force look for rows that meet, every refusal,
// and places of positions at the edges.
#include "../../qora-llm_amd/csrc/paged_args.hpp"

#include <cstdio>
#include <cstdlib>
#include <set>

using namespace qora;

static int fails = 0;
#define CHECK(x)                                              \
    do {                                                      \
        if (!(x)) {                                           \
            std::printf("line %d: %s\n", __LINE__, #x);       \
            ++fails;                                          \
        }                                                     \
    } while (0)

static uint64_t state = 88172645463325252ull;
static uint32_t rnd(uint32_t n) {
    state ^= state << 13;
    state ^= state >> 7;
    state ^= state << 17;
    return (uint32_t)(state >> 33) % n;
}

static bool rows_meet(const qora_paged_kv& kv) {
    std::set<uint64_t> seen;
    for (uint32_t p = 0; p < kv.num_pages; ++p)
        for (uint32_t h = 0; h < kv.num_kv_heads; ++h)
            for (uint32_t s = 0; s < kv.page_size; ++s) {
                const uint64_t at = paged_offset(kv.page_stride, kv.head_stride, kv.slot_stride, p, h, s);
                for (uint32_t d = 0; d < kv.head_dim; ++d)
                    if (!seen.insert(at + d).second) return true;
            }
    return false;
}

int main() {
    alignas(16) static float mem[2][16];
    qora_paged_kv ok{};
    ok.k = mem[0];
    ok.v = mem[1];
    ok.num_pages = 3;
    ok.page_size = 4;
    ok.num_kv_heads = 2;
    ok.head_dim = 8;
    ok.page_stride = 64;
    ok.head_stride = 32;
    ok.slot_stride = 8;
    CHECK(!paged_kv_error(&ok));
    CHECK(paged_kv_error(nullptr));
    int good = 0, refused = 0;
    for (int i = 0; i < 20000; ++i) {
        qora_paged_kv kv = ok;
        kv.kv_f16 = rnd(2);
        kv.num_pages = 1 + rnd(3);
        kv.page_size = 1 + rnd(4);
        kv.num_kv_heads = 1 + rnd(3);
        kv.head_dim = 8 * (1 + rnd(2));
        kv.page_stride = 8 * rnd(20);
        kv.head_stride = 8 * rnd(20);
        kv.slot_stride = 8 * rnd(20);
        const bool bad = paged_kv_error(&kv) != nullptr;
        // every accepted pool's rows are apart (some that are apart in no nested order are refused too)
        CHECK(bad || !rows_meet(kv));
        (bad ? refused : good)++;
    }
    CHECK(good > 500 && refused > 500);
    auto with = [&](auto f) {
        qora_paged_kv kv = ok;
        f(kv);
        return paged_kv_error(&kv) != nullptr;
    };
    CHECK(with([](qora_paged_kv& x) { x.k = nullptr; }));
    CHECK(with([](qora_paged_kv& x) { x.v = nullptr; }));
    CHECK(with([](qora_paged_kv& x) { x.v = x.k; }));
    CHECK(with([](qora_paged_kv& x) { x.k = (char*)x.k + 4; }));
    CHECK(with([](qora_paged_kv& x) { x.kv_f16 = 2; }));
    CHECK(with([](qora_paged_kv& x) { x.num_pages = 0; }));
    CHECK(with([](qora_paged_kv& x) { x.page_size = 0; }));
    CHECK(with([](qora_paged_kv& x) { x.num_kv_heads = 0; }));
    CHECK(with([](qora_paged_kv& x) { x.head_dim = 0; }));
    CHECK(with([](qora_paged_kv& x) { x.head_dim = 12; }));
    CHECK(with([](qora_paged_kv& x) { x.head_dim = 136; }));
    CHECK(with([](qora_paged_kv& x) { x.num_pages = 0xFFFFFFFFu; }));
    CHECK(with([](qora_paged_kv& x) { x.page_stride = 66; }));
    CHECK(with([](qora_paged_kv& x) { x.kv_f16 = 1; x.slot_stride = 12; }));
    CHECK(with([](qora_paged_kv& x) { x.page_stride = ~0ull - 15; }));
    CHECK(with([](qora_paged_kv& x) { x.num_pages = 0x7FFFFFFFu; x.page_stride = (1ull << 40) - 16; }));

    int32_t arr[4] = {0, 1, 2, 3};
    qora_paged_batch b{arr, arr, arr, 2, 3, 10, 0};
    CHECK(!paged_batch_error(&ok, &b));
    CHECK(paged_batch_error(&ok, nullptr));
    auto wb = [&](auto f) {
        qora_paged_batch x = b;
        f(x);
        return paged_batch_error(&ok, &x) != nullptr;
    };
    CHECK(wb([](qora_paged_batch& x) { x.row_start = nullptr; }));
    CHECK(wb([](qora_paged_batch& x) { x.kv_len = nullptr; }));
    CHECK(wb([](qora_paged_batch& x) { x.pages = nullptr; }));
    CHECK(wb([](qora_paged_batch& x) { x.max_pages = 0; }));
    CHECK(wb([](qora_paged_batch& x) { x.max_pages = 0x20000000u; }));
    CHECK(wb([](qora_paged_batch& x) { x.rows = 0x80000000u; }));
    CHECK(wb([](qora_paged_batch& x) { x.num_seqs = kPagedMaxSeqs + 1; }));
    CHECK(!wb([](qora_paged_batch& x) { x.num_seqs = 0; x.pages = nullptr; }));

    uint32_t e = 9, s = 9;
    CHECK(!paged_table_index(-1, 4, 3, &e, &s) && !paged_table_index(12, 4, 3, &e, &s));
    CHECK(!paged_table_index(INT64_MIN, 4, 3, &e, &s) && !paged_table_index(INT64_MAX, 4, 3, &e, &s));
    CHECK(paged_table_index(0, 4, 3, &e, &s) && e == 0 && s == 0);
    CHECK(paged_table_index(11, 4, 3, &e, &s) && e == 2 && s == 3);
    CHECK(paged_table_index(0x7FFFFFFEll, 1, 0x7FFFFFFFu, &e, &s) && e == 0x7FFFFFFEu && s == 0);
    CHECK(paged_page_ok(0, 3) && paged_page_ok(2, 3) && !paged_page_ok(3, 3) && !paged_page_ok(-1, 3) &&
          !paged_page_ok(INT32_MIN, 3));
    // past 32 bits: the last row of a large pool
    CHECK(paged_offset(1ull << 20, 1ull << 16, 128, 1u << 20, 3, 500) == (1ull << 40) + (3ull << 16) + 64000ull);
    CHECK(paged_rows_of(0, 5, 5) == 5 && paged_rows_of(2, 2, 5) == 0 && paged_rows_of(3, 2, 5) == 0 &&
          paged_rows_of(-1, 2, 5) == 0 && paged_rows_of(0, 6, 5) == 0 && paged_rows_of(INT32_MIN, INT32_MAX, 5) == 0);
    CHECK(!paged_rows_error(mem, 16, 2, 8) && paged_rows_error(nullptr, 16, 2, 8) && paged_rows_error(mem, 12, 2, 8) &&
          paged_rows_error(mem, 18, 2, 8) && paged_rows_error((char*)mem + 8, 16, 2, 8) &&
          paged_rows_error(mem, 1ull << 40, 2, 8));
    // rows against a brute-force look for a shared float
    static float f[4096];
    int meet = 0;
    for (int i = 0; i < 20000; ++i) {
        const uint64_t wa = 1 + rnd(12), wb = 1 + rnd(12), rows = 1 + rnd(6);
        const uint64_t lda = wa + rnd(16), ldb = rnd(2) ? lda : wb + rnd(16);
        if (ldb < wb) continue;
        const float *a = f + 1000 + rnd(80), *b = f + 1000 + rnd(80);
        bool shared = false;
        for (uint64_t r = 0; r < rows; ++r)
            for (uint64_t q = 0; q < rows; ++q) {
                const float *x = a + r * lda, *y = b + q * ldb;
                shared = shared || (x < y + wb && y < x + wa);
            }
        const bool said = paged_rows_meet(a, lda, wa, b, ldb, wb, rows);
        CHECK(said || !shared);                      // (what meets in no row may be refused where the strides differ)
        if (lda == ldb && said && !shared) ++meet;   // or wraps around the end of the last row
    }
    CHECK(meet < 400);
    float qkv[3][48];
    CHECK(!paged_rows_meet(qkv[0], 48, 16, qkv[0] + 16, 48, 16, 3) && !paged_rows_meet(qkv[0] + 32, 48, 16, qkv[0], 48, 16, 3));
    CHECK(paged_rows_meet(qkv[0], 48, 16, qkv[0] + 15, 48, 16, 3) && paged_rows_meet(qkv[0], 48, 16, qkv[0], 48, 16, 3));
    CHECK(paged_rows_meet(qkv[0], 16, 16, qkv[0] + 16, 48, 16, 3) && !paged_rows_meet(qkv[0], 48, 16, qkv[2] + 16, 48, 16, 0));
    std::printf(fails ? "%d failed\n" : "all cases held\n", fails);
    return fails != 0;
}
