"""qora_hip_paged_attn_run against softmax attention in float64: one row to
chunks, head shapes, page sizes, layouts, rows that see nothing, what masked
and stale slots hold, batches of very different rows, replays and refusals."""
import ctypes

import numpy as np
import pytest

from helpers import device, rng
from paged_util import EPS32, Batch, Pool, attention64

pytestmark = pytest.mark.gpu

RAGGED = [(1, 1), (5, 5), (0, 7), (0, 0), (3, 40), (1, 333), (17, 17), (2, 64), (1, 65), (40, 100), (1, 16), (4, 1000)]
CASES = [
    # kv, order, page, H, KVH, hd, seqs
    ("f16", "head", 16, 16, 4, 128, RAGGED),
    ("f32", "head", 16, 16, 4, 128, RAGGED),
    ("f16", "slot", 24, 12, 4, 128, RAGGED),
    ("f32", "slot", 100, 8, 8, 64, RAGGED),
    ("f16", "outer", 1, 4, 2, 64, RAGGED),
    ("f32", "outer", 3, 4, 2, 64, RAGGED),
    ("f16", "head", 16, 5, 1, 40, RAGGED),
    ("f32", "head", 16, 6, 2, 72, RAGGED),
    ("f16", "head", 64, 20, 1, 128, RAGGED),           # more query heads than a tile of rows
    ("f32", "slot", 16, 3, 3, 8, RAGGED),
    ("f16", "head", 256, 16, 4, 128, [(1, 5000)]),
    ("f32", "head", 256, 16, 4, 128, [(1, 3000), (1, 2)]),
    ("f16", "head", 16, 16, 4, 128, [(1, 1 + 37 * i) for i in range(40)]),
    ("f16", "head", 16, 4, 2, 64, [((i % 3 > 0) * 1, 3 + i % 50) for i in range(150)]),
    ("f16", "head", 64, 16, 4, 128, [(300, 300)]),
    ("f32", "head", 64, 4, 2, 64, [(257, 700)]),
    ("f16", "head", 16, 16, 4, 128, [(130, 513), (1, 900), (1, 1), (33, 47), (8, 8)]),
    ("f32", "head", 24, 12, 4, 128, [(130, 413), (1, 900), (1, 1), (33, 47), (8, 8)]),
]


def _inputs(pkg, r, kv, order, page, H, KVH, hd, seqs, std=1.0, **kw):
    batch = Batch(r, seqs, page, **kw)
    pool = Pool(pkg, r, kv, order, batch.num_pages, page, KVH, hd, pad=8 if order == "outer" else 0, fill=np.nan)
    used = np.zeros(pool.k.shape, dtype=bool)
    for s, (_, L) in enumerate(seqs):
        for j in range(L):
            p = batch.place(s, j)
            for h in range(KVH if p else 0):
                used[pool.at(p[0], h, p[1])] = True
    for x in (pool.k, pool.v):                         # every slot that no sequence holds stays NaN
        x[used] = r.normal(size=int(used.sum())).astype(x.dtype)
    q = (std * r.normal(size=(batch.rows, H, hd))).astype(np.float32)
    return batch, pool, q


def _run(ctx, pkg, d, pool, batch, q, H, max_new=0, stream=0, times=1):
    hd = pool.hd
    kv, b = pool.put(d), batch.put(pkg, d, max_new)
    dq, out = d.put(q), d.put(np.full(q.shape, 77.0, dtype=np.float32))
    aid = ctx.paged_attn_prepare(batch.rows, len(batch.seqs), H, pool.KVH, hd)
    res = []
    for _ in range(times):
        ctx.paged_attn_run(aid, kv, b, dq, out, stream=stream)
        ctx.synchronize()
        res.append(d.get(out, q.shape, np.float32))
    ctx.paged_attn_release(aid)
    return res if times > 1 else res[0]


def _check(got, batch, ref, tol):
    assert np.all(np.isfinite(got[:batch.used]))
    off = np.abs(got[:batch.used].astype(np.float64) - ref) - tol
    w = np.unravel_index(np.argmax(off), off.shape) if off.size else None
    assert w is None or off[w] <= 0, (w, float(off[w]), got[w], ref[w])
    assert np.all(got[batch.used:] == 77.0)            # rows of nobody


@pytest.mark.parametrize("kv,order,page,H,KVH,hd,seqs", CASES)
def test_attention_matches_definition(ctx, pkg, kv, order, page, H, KVH, hd, seqs):
    r = rng(page + 3 * hd + H + len(seqs))
    batch, pool, q = _inputs(pkg, r, kv, order, page, H, KVH, hd, seqs, pad_rows=2)
    ref, tol = attention64(pool, batch, q, H)
    with device(ctx) as d:
        a, b = _run(ctx, pkg, d, pool, batch, q, H, times=2)
    _check(a, batch, ref, tol)
    assert np.array_equal(a, b)                        # the same bits each time


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("max_new", [1, 4, 40])
def test_attention_by_the_most_rows(ctx, pkg, kv, max_new):
    """max_new bounds the rows of a sequence: what is asked for is the same with it, further rows stay."""
    r = rng(5)
    seqs = [(1, 9), (1, 700), (min(4, max_new), 81), (max_new, max_new), (max_new + 2, 300)]
    batch, pool, q = _inputs(pkg, r, kv, "head", 16, 16, 4, 128, seqs)
    ref, tol = attention64(pool, batch, q, 16)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 16, max_new=max_new)
    last = batch.used - 2
    assert np.all(got[last:] == 77.0)
    assert np.all(np.abs(got[:last] - ref[:last]) <= tol[:last])


def test_many_sequences(ctx, pkg):
    """More sequences than the plan looks at in one go, short and long ones, some with no rows."""
    r = rng(20)
    seqs = [(int(r.integers(0, 3)), int(r.integers(1, 40))) for _ in range(1100)]
    seqs[700] = (1, 2500)
    seqs[1099] = (20, 300)
    batch, pool, q = _inputs(pkg, r, "f16", "slot", 8, 4, 2, 64, seqs, pad_rows=1)
    ref, tol = attention64(pool, batch, q, 4)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 4)
    _check(got, batch, ref, tol)


@pytest.mark.parametrize("rows,keys", [(1, 43 * 128), (20, 43 * 64)])
def test_every_tile_split(ctx, pkg, rows, keys):
    """As many split tiles as there can be: equal sequences, a few fewer than the work is cut into (two items for
    each of 256 CUs), so that each has a little more than an item's share; they read the same pages."""
    r = rng(24)
    page, n = 256, 500
    batch = Batch(r, [(rows, keys)] * n, page)
    batch.num_pages = batch.max_pages = -(-keys // page)
    batch.pages = np.tile(r.permutation(batch.num_pages).astype(np.int32), (n, 1))
    pool = Pool(pkg, r, "f16", "head", batch.num_pages, page, 1, 64, fill=0.0)
    k, v = np.zeros((2, keys, 64))
    for j in range(keys):
        p, slot = batch.place(0, j)
        for x, plain in ((pool.k, k), (pool.v, v)):
            x[pool.at(p, 0, slot)] = r.normal(size=64).astype(np.float16)
            plain[j] = x[pool.at(p, 0, slot)]
    q = r.normal(size=(batch.rows, 1, 64)).astype(np.float32)
    sc = (q[:, 0].astype(np.float64) @ k.T / 8).reshape(n, rows, keys)
    sc[:, np.arange(keys) > keys - rows + np.arange(rows)[:, None]] = -np.inf
    e = np.exp(sc - sc.max(-1, keepdims=True))
    ref = (e @ v / e.sum(-1, keepdims=True)).reshape(-1, 1, 64)
    S = (np.abs(q[:, 0]).astype(np.float64) @ np.abs(k).T / 8).max(-1)
    tol = EPS32 * (2 * (64 + 16) * S + keys + 64)[:, None, None] * np.abs(v).max()
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 1)
    _check(got, batch, ref, tol)


def test_pool_past_32_bits(ctx, pkg):
    """Pages whose element offsets pass 2^32 and whose bytes pass 2^33: append, then attend, single token and chunk."""
    r = rng(22)
    H, KVH, hd, page = 16, 4, 128, 16
    page_elems = KVH * page * hd
    num_pages = (9 << 30) // (2 * page_elems)               # 9 GiB of binary16 in each pool
    assert num_pages * page_elems > 2 ** 32
    seqs = [(1, 37), (40, 40)]
    ids = np.array([[num_pages - 1, 3, num_pages - 7], [num_pages - 2, num_pages // 2 + 1, num_pages - 5]], dtype=np.int32)
    batch = Batch(r, seqs, page)
    batch.pages, batch.num_pages, batch.max_pages = ids, num_pages, 3
    dk, dv = ctx.malloc(num_pages * page_elems * 2), ctx.malloc(num_pages * page_elems * 2)
    try:
        with device(ctx) as d:
            kv = pkg.PagedKV(dk, dv, 1, num_pages, page, KVH, hd, page_elems, page * hd, hd)
            # what the sequences cache, written through the append itself, 37 and 40 rows
            full = Batch(r, [(37, 37), (40, 40)], page)
            full.pages, full.num_pages, full.max_pages = ids, num_pages, 3
            x = r.normal(size=(77, (H + 2 * KVH) * hd)).astype(np.float32)
            p = d.put(x)
            ctx.paged_append(kv, full.put(pkg, d), H, p, p + 4 * H * hd, p + 4 * (H + KVH) * hd, x.shape[1], p, q_out_stride=x.shape[1])
            # a small pool with the same rows, for the definition
            pool = Pool(pkg, r, "f16", "head", 6, page, KVH, hd, fill=0.0)
            small = {int(i): n for n, i in enumerate(ids.reshape(-1))}
            for row, s, pos in full.row_places():
                at = small[int(ids[s, pos // page])]
                for h in range(KVH):
                    pool.k[pool.at(at, h, pos % page)] = x[row].reshape(-1, hd)[H + h]
                    pool.v[pool.at(at, h, pos % page)] = x[row].reshape(-1, hd)[H + KVH + h]
            ref_batch = Batch(r, seqs, page)
            ref_batch.pages = np.vectorize(small.get)(ids).astype(np.int32)
            ref_batch.num_pages, ref_batch.max_pages = 6, 3
            q = r.normal(size=(41, H, hd)).astype(np.float32)
            ref, tol = attention64(pool, ref_batch, q, H)
            aid = ctx.paged_attn_prepare(41, 2, H, KVH, hd)
            out = d.put(np.full(q.shape, 77.0, np.float32))
            ctx.paged_attn_run(aid, kv, batch.put(pkg, d), d.put(q), out)
            ctx.synchronize()
            _check(d.get(out, q.shape, np.float32), batch, ref, tol)
            ctx.paged_attn_release(aid)
    finally:
        ctx.free(dk)
        ctx.free(dv)


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_rows_that_see_nothing_are_zero(ctx, pkg, kv):
    """Lengths shorter than the new rows, lengths of 0 and below, and pages that are all outside the pool."""
    r = rng(6)
    # (the last two: tiles of 128 rows that see nothing, in front of work that follows)
    seqs = [(3, 0), (4, 2), (1, -7), (2, 5), (1, 3), (20, 11), (40, 0), (90, 17)]
    batch, pool, q = _inputs(pkg, r, kv, "head", 4, 8, 2, 64, seqs, bad={(3, 0): -1, (3, 1): 10 ** 7, (4, 0): -2 ** 31})
    ref, tol = attention64(pool, batch, q, 8)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 8)
    _check(got, batch, ref, tol)
    for row, s, pos in batch.row_places():
        if pos < 0 or s in (3, 4):
            assert not np.any(got[row])


@pytest.mark.parametrize("kv,H,KVH,hd", [("f16", 16, 4, 128), ("f32", 16, 4, 128), ("f16", 4, 2, 64), ("f32", 8, 8, 64)])
def test_pages_outside_the_pool_are_not_there(ctx, pkg, kv, H, KVH, hd):
    r = rng(7)
    seqs = [(1, 200), (30, 150), (2, 90)]
    bad = {(0, 3): -1, (0, 12): 2 ** 31 - 1, (1, 0): -5, (1, 9): 10 ** 6, (2, 5): -1}
    batch, pool, q = _inputs(pkg, r, kv, "head", 16, H, KVH, hd, seqs, bad=bad)
    ref, tol = attention64(pool, batch, q, H)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, H)
    _check(got, batch, ref, tol)


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, "largest"])
@pytest.mark.parametrize("kv,H,KVH,hd", [("f16", 16, 4, 128), ("f32", 12, 4, 128), ("f32", 4, 2, 64), ("f16", 3, 1, 40)])
def test_later_rows_do_not_reach_earlier_ones(ctx, pkg, kv, H, KVH, hd, what):
    """A chunk whose later tokens' keys and values are not finite, or of the type's largest
    size: the rows before them are the same as without."""
    r = rng(8)
    seqs = [(70, 200), (3, 50), (1, 130), (9, 9)]
    batch, pool, q = _inputs(pkg, r, kv, "head", 16, H, KVH, hd, seqs)
    ref, tol = attention64(pool, batch, q, H)
    if what == "largest":
        what = float(np.finfo(pool.dtype).max) * (1 if kv == "f16" else 0.25)
    first = {0: 200 - 31, 1: 48, 3: 4}                 # positions from here on are spoilt
    for s, at in first.items():
        for j in range(at, seqs[s][1]):
            p = batch.place(s, j)
            for h in range(KVH):
                pool.k[pool.at(p[0], h, p[1])] = what
                pool.v[pool.at(p[0], h, p[1])] = what
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, H)
    seen = 0
    for row, s, pos in batch.row_places():
        if pos < first.get(s, 10 ** 9):
            assert np.all(np.abs(got[row] - ref[row]) <= tol[row]), (row, s, pos)
            seen += 1
    assert seen == 70 - 31 + 1 + 1 + 4


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("scale", [1e-4, 3e3])
def test_values_and_keys_of_other_sizes(ctx, pkg, kv, scale):
    """Small and large values; keys that make one weight take nearly all."""
    r = rng(9)
    seqs = [(1, 600), (20, 300)]
    batch, pool, q = _inputs(pkg, r, kv, "head", 16, 16, 4, 128, seqs, std=4.0)
    for s, (_, L) in enumerate(seqs):                  # sizes that differ from position to position
        for j in range(L):
            p = batch.place(s, j)
            for h in range(4):
                at = pool.at(p[0], h, p[1])
                pool.v[at] = (pool.v[at].astype(np.float64) * scale * 2.0 ** -(j % 7)).astype(pool.dtype)
    ref, tol = attention64(pool, batch, q, 16)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 16)
    _check(got, batch, ref, tol)


def test_f32_cache_beyond_binary16(ctx, pkg):
    """Keys and values far outside binary16's range keep float32's precision."""
    r = rng(10)
    seqs = [(1, 200), (40, 90)]
    batch, pool, q = _inputs(pkg, r, "f32", "head", 16, 8, 2, 64, seqs)
    for s, (_, L) in enumerate(seqs):
        for j in range(L):
            p = batch.place(s, j)
            for h in range(2):
                at = pool.at(p[0], h, p[1])
                pool.k[at] *= np.float32(1e12)
                pool.v[at] *= np.float32([1e20, 1e-20, 1.0][s if s else j % 2 * 2])
    q *= np.float32(1e-12)
    ref, tol = attention64(pool, batch, q, 8)
    with device(ctx) as d:
        got = _run(ctx, pkg, d, pool, batch, q, 8)
    _check(got, batch, ref, tol)


def test_other_streams_strides_and_in_place(ctx, pkg):
    r = rng(16)
    H, KVH, hd = 8, 2, 64
    batch, pool, q = _inputs(pkg, r, "f16", "slot", 16, H, KVH, hd, [(1, 900), (30, 64), (2, 2)])
    ref, tol = attention64(pool, batch, q, H)
    wide = np.full((batch.rows, H * hd + 36), 77.0, dtype=np.float32)
    wide[:, :H * hd] = q.reshape(batch.rows, -1)
    other = pkg.HipContext(0)
    try:
        with device(ctx) as d:
            kv, b = pool.put(d), batch.put(pkg, d)
            aid = ctx.paged_attn_prepare(batch.rows, 3, H, KVH, hd)
            dq = d.put(wide)
            # over q itself, rows further apart than the heads, on a stream that is not the context's
            ctx.paged_attn_run(aid, kv, b, dq, dq, q_stride=wide.shape[1], out_stride=wide.shape[1], stream=other.stream)
            other.synchronize()
            got = d.get(dq, wide.shape, np.float32)
            assert np.all(got[:, H * hd:] == 77.0)
            _check(np.ascontiguousarray(got[:, :H * hd]).reshape(q.shape), batch, ref, tol)
            # an id for each stream: two calls that may run at once
            aid2 = ctx.paged_attn_prepare(batch.rows, 3, H, KVH, hd)
            dq = d.put(q)
            o1, o2 = d.empty(q.nbytes), d.empty(q.nbytes)
            for _ in range(4):
                ctx.paged_attn_run(aid, kv, b, dq, o1)
                ctx.paged_attn_run(aid2, kv, b, dq, o2, stream=other.stream)
            ctx.synchronize()
            other.synchronize()
            for o in (o1, o2):
                _check(d.get(o, q.shape, np.float32), batch, ref, tol)
            ctx.paged_attn_release(aid)
            ctx.paged_attn_release(aid2)
    finally:
        other.close()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_replays_take_the_arrays_of_the_moment(ctx, pkg, kv):
    """One captured call, replayed as the sequences grow and change places, eager calls of
    the same id between the replays."""
    r = rng(17)
    H, KVH, hd, page = 16, 4, 128, 16
    batch, pool, q = _inputs(pkg, r, kv, "head", page, H, KVH, hd, [(1, 1500), (3, 700), (40, 90)])
    steps = [[(1, 1500), (3, 700), (40, 90)], [(1, 17), (3, 3), (40, 40)], [(2, 1200), (40, 600), (2, 1)],
             [(0, 0), (44, 650), (0, 90)]]
    with device(ctx) as d:
        kvd, b = pool.put(d), batch.put(pkg, d)
        dq, out = d.put(q), d.put(np.full(q.shape, 77.0, np.float32))
        aid = ctx.paged_attn_prepare(batch.rows, 3, H, KVH, hd)
        ctx.synchronize()
        ctx.capture_begin()
        ctx.paged_attn_run(aid, kvd, b, dq, out)
        g = ctx.capture_end()
        for seqs in steps + steps[:1]:
            batch.seqs = seqs
            batch.row_start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
            batch.kv_len = np.array([L for _, L in seqs], dtype=np.int32)
            ctx.h2d(batch.d[0], batch.row_start)
            ctx.h2d(batch.d[1], batch.kv_len)
            ref, tol = attention64(pool, batch, q, H)
            got = []
            for eager in (False, True, False):
                ctx.h2d(out, np.full(q.shape, 77.0, np.float32))
                if eager:
                    ctx.paged_attn_run(aid, kvd, b, dq, out)
                else:
                    ctx.graph_launch(g)
                ctx.synchronize()
                got.append(d.get(out, q.shape, np.float32))
                _check(got[-1], batch, ref, tol)
            assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
        ctx.graph_destroy(g)
        ctx.paged_attn_release(aid)


def test_row_offsets_that_are_none(ctx, pkg):
    """Offsets that do not ascend or leave the row arrays: nothing outside the arrays is touched,
    and the next call with the id is right."""
    r = rng(18)
    H, KVH, hd = 8, 2, 64
    batch, pool, q = _inputs(pkg, r, "f16", "head", 16, H, KVH, hd, [(1, 900), (30, 64), (2, 2)])
    good = batch.row_start.copy()
    ref, tol = attention64(pool, batch, q, H)
    with device(ctx) as d:
        kv, b = pool.put(d), batch.put(pkg, d)
        dq, out = d.put(q), d.put(np.full(q.shape, 77.0, np.float32))
        aid = ctx.paged_attn_prepare(batch.rows, 3, H, KVH, hd)
        for starts in ([0, 10 ** 6, 3, 5], [-4, -3, -2, -1], [33, 20, 10, 0], [2 ** 31 - 1] * 4, [0, 33, 0, 33]):
            ctx.h2d(batch.d[0], np.array(starts, dtype=np.int32))
            ctx.paged_attn_run(aid, kv, b, dq, out)
            ctx.synchronize()
        ctx.h2d(batch.d[0], good)
        ctx.h2d(out, np.full(q.shape, 77.0, np.float32))
        ctx.paged_attn_run(aid, kv, b, dq, out)
        ctx.synchronize()
        _check(d.get(out, q.shape, np.float32), batch, ref, tol)
        ctx.paged_attn_release(aid)


def test_row_offsets_that_are_none_of_many(ctx, pkg):
    """The same with more sequences than one wave plans, which ask for more items than there are workgroups."""
    r = rng(25)
    H, KVH, hd, n = 8, 2, 64, 200
    batch, pool, q = _inputs(pkg, r, "f16", "head", 16, H, KVH, hd, [(1, 40 + 30 * (i % 7)) for i in range(n)], pad_rows=1)
    good = batch.row_start.copy()
    ref, tol = attention64(pool, batch, q, H)
    at = np.arange(n + 1)
    with device(ctx) as d:
        kv, b = pool.put(d), batch.put(pkg, d)
        dq, out = d.put(q), d.put(np.full(q.shape, 77.0, np.float32))
        aid = ctx.paged_attn_prepare(batch.rows, n, H, KVH, hd)
        for starts in (at % 2 * n, n - at, at * 10 ** 6, at - n, np.full(n + 1, -2 ** 31), np.where(at < 150, at, at % 2 * n)):
            ctx.h2d(batch.d[0], starts.astype(np.int32))
            ctx.paged_attn_run(aid, kv, b, dq, out)
            ctx.synchronize()
            assert np.all(d.get(out, q.shape, np.float32)[n:] == 77.0)      # a row of nobody
        ctx.h2d(batch.d[0], good)
        for _ in range(2):
            ctx.h2d(out, np.full(q.shape, 77.0, np.float32))
            ctx.paged_attn_run(aid, kv, b, dq, out)
            ctx.synchronize()
            _check(d.get(out, q.shape, np.float32), batch, ref, tol)
        ctx.paged_attn_release(aid)


def test_attention_refusals(ctx, pkg):
    r = rng(19)
    H, KVH, hd = 8, 2, 64
    batch, pool, q = _inputs(pkg, r, "f16", "head", 16, H, KVH, hd, [(2, 20)])
    inv = pkg.QORA_HIP_E_INVALID
    aid = ctypes.c_uint32()
    for a in [(0, 1, 8, 2, 64), (1, 0, 8, 2, 64), (1, 70000, 8, 2, 64), (1, 1, 8, 3, 64), (1, 1, 0, 2, 64),
              (1, 1, 8, 0, 64), (1, 1, 8, 2, 0), (1, 1, 8, 2, 136), (1, 1, 8, 2, 60), (2 ** 31, 1, 8, 2, 64)]:
        assert ctx.lib.qora_hip_paged_attn_prepare(ctx.h, *a, ctypes.byref(aid)) == inv, a
    assert ctx.lib.qora_hip_paged_attn_prepare(ctx.h, 1, 1, 8, 2, 64, None) == inv
    with device(ctx) as d:
        kv, b = pool.put(d), batch.put(pkg, d)
        dq, out = d.put(q), d.empty(q.nbytes + 64)
        aid = ctx.paged_attn_prepare(2, 1, H, KVH, hd)

        def call(i=aid, kv=kv, b=b, q=dq, qs=H * hd, o=out, os=H * hd):
            return ctx.lib.qora_hip_paged_attn_run(ctx.h, i, ctypes.byref(kv) if kv else None,
                                                   ctypes.byref(b) if b else None, q, qs, o, os, None)

        def pool_like(**ch):
            x = pkg.PagedKV.from_buffer_copy(kv)
            for n, v in ch.items():
                setattr(x, n, v)
            return x

        def batch_like(**ch):
            x = pkg.PagedBatch.from_buffer_copy(b)
            for n, v in ch.items():
                setattr(x, n, v)
            return x

        assert call() == pkg.QORA_HIP_OK
        for ch in [dict(i=aid + 1000), dict(kv=None), dict(b=None), dict(q=None), dict(o=None), dict(qs=H * hd - 4),
                   dict(os=H * hd + 2), dict(q=dq + 4), dict(o=dq + 16),
                   dict(kv=pool_like(head_dim=32)), dict(kv=pool_like(num_kv_heads=1)), dict(kv=pool_like(page_size=0)),
                   dict(kv=pool_like(slot_stride=56)), dict(kv=pool_like(slot_stride=68)), dict(kv=pool_like(kv_f16=2)),
                   dict(kv=pool_like(k=kv.k + 8)), dict(kv=pool_like(v=kv.k)), dict(b=batch_like(rows=3)),
                   dict(b=batch_like(num_seqs=2)), dict(b=batch_like(max_pages=0)), dict(b=batch_like(kv_len=0)),
                   dict(b=batch_like(max_pages=2 ** 31 - 1))]:
            assert call(**ch) == inv, ch
        assert call(b=batch_like(rows=0), q=None, o=None) == pkg.QORA_HIP_OK
        ctx.synchronize()
        # neither in a capture
        ctx.capture_begin()
        st = pkg.QORA_HIP_E_STATE
        x = ctypes.c_uint32()
        assert ctx.lib.qora_hip_paged_attn_prepare(ctx.h, 1, 1, 8, 2, 64, ctypes.byref(x)) == st
        assert ctx.lib.qora_hip_paged_attn_release(ctx.h, aid) == st
        ctx.graph_destroy(ctx.capture_end())
        ctx.paged_attn_release(aid)
        assert call() == inv and ctx.lib.qora_hip_paged_attn_release(ctx.h, aid) == inv
