"""qora_hip_paged_append against the rotation and the cache rows in float64:
layouts, page sizes, lengths from none to long, partial and no rotation, rows
without a place, what must stay as it was, and the argument checks."""
import ctypes

import numpy as np
import pytest

from helpers import device, rng
from paged_util import EPS16, EPS32, Batch, Pool, rotate64

pytestmark = pytest.mark.gpu

RAGGED = [(1, 1), (5, 5), (0, 7), (0, 0), (3, 40), (1, 33), (17, 17), (2, 300)]
CASES = [
    # kv, order, page, H, KVH, hd, half, seqs
    ("f16", "head", 16, 16, 4, 128, 64, RAGGED),
    ("f32", "slot", 24, 16, 4, 128, 64, RAGGED),
    ("f32", "outer", 1, 4, 2, 64, 32, RAGGED),
    ("f16", "slot", 100, 8, 8, 64, 16, RAGGED),       # a quarter of the dims rotated
    ("f16", "head", 7, 3, 1, 40, 0, RAGGED),          # not rotated
    ("f32", "head", 16, 5, 5, 8, 3, RAGGED),          # pairs that are no 16-byte units
    ("f16", "head", 16, 6, 2, 72, 33, RAGGED),
    ("f16", "head", 16, 16, 4, 128, 64, [(1, 1 + 5 * i) for i in range(70)]),      # more than a wave of sequences
    ("f32", "head", 16, 4, 2, 64, 32, [((1 if i % 3 else 0), 2 + i % 9) for i in range(200)]),
    ("f16", "head", 64, 4, 2, 64, 32, [(1500, 1500)]),
    ("f16", "head", 16, 4, 2, 64, 32, [(1, 1)]),
]


def _tables(pkg, positions, half):
    c, s = pkg.rope_tables(positions, max(half, 1), 5e6)
    return c.reshape(positions, -1), s.reshape(positions, -1)


def _expect(batch, pool, qkv, H, half, cos, sin, positions):
    """(q_out, k pool, v pool) in float64 and which q_out rows are written."""
    KVH, hd = pool.KVH, pool.hd
    q_out = np.full((batch.rows, H, hd), np.nan)
    k, v = pool.k.astype(np.float64), pool.v.astype(np.float64)
    for row, s, pos in batch.row_places():
        place = batch.place(s, pos)
        if place is None or (half and pos >= positions):
            continue
        x = qkv[row].reshape(H + 2 * KVH, hd).astype(np.float64)
        if half:
            x[:H + KVH] = rotate64(x[:H + KVH], cos[pos].astype(np.float64), sin[pos].astype(np.float64), half)
        q_out[row] = x[:H]
        for h in range(KVH):
            k[pool.at(place[0], h, place[1])] = x[H + h]
            v[pool.at(place[0], h, place[1])] = x[H + KVH + h]
    return q_out, k, v


def _call(ctx, pkg, d, pool, batch, qkv, H, half, cos, sin, positions, in_place=False, stream=0):
    KVH, hd = pool.KVH, pool.hd
    kv, b = pool.put(d), batch.put(pkg, d)
    p, ld = d.put(qkv), qkv.shape[1]
    out = p if in_place else d.put(np.full((batch.rows, H * hd), np.nan, dtype=np.float32))
    ctx.paged_append(kv, b, H, p, p + 4 * H * hd, p + 4 * (H + KVH) * hd, ld, out, d.put(cos), d.put(sin), half,
                     positions, q_out_stride=ld if in_place else 0, stream=stream)
    return out, kv, b


def _close(a, ref, eps, mag):
    """Two products and a sum in float32: three half steps of the terms' size, then the
    rounding of the store; equal where the reference says nothing was written (NaN)."""
    assert np.array_equal(np.isnan(a), np.isnan(ref))
    ok = ~np.isnan(ref)
    assert np.all(np.abs(a[ok] - ref[ok]) <= (3 * EPS32 + eps) * mag), float(np.abs(a[ok] - ref[ok]).max())


@pytest.mark.parametrize("kv,order,page,H,KVH,hd,half,seqs", CASES)
def test_append_matches_definition(ctx, pkg, kv, order, page, H, KVH, hd, half, seqs):
    r = rng(page * 100 + hd + len(seqs))
    batch = Batch(r, seqs, page, pad_rows=3)
    pool = Pool(pkg, r, kv, order, batch.num_pages, page, KVH, hd, pad=8 if order == "outer" else 0)
    positions = max(int(batch.kv_len.max()), 1)
    cos, sin = _tables(pkg, positions, half)
    qkv = r.normal(size=(batch.rows, (H + 2 * KVH) * hd)).astype(np.float32)
    q64, k64, v64 = _expect(batch, pool, qkv, H, half, cos, sin, positions)
    with device(ctx) as d:
        out, _, _ = _call(ctx, pkg, d, pool, batch, qkv, H, half, cos, sin, positions)
        got = d.get(out, (batch.rows, H, hd), np.float32)
        k, v = d.get(pool.dk, pool.k.shape, pool.dtype), d.get(pool.dv, pool.v.shape, pool.dtype)
    mag = 2 * float(np.abs(qkv).max())
    _close(got.astype(np.float64), q64, 0.0, mag)
    _close(k.astype(np.float64), k64, EPS16 if kv == "f16" else 0.0, mag)
    # v is stored, not computed
    assert np.array_equal(v, v64.astype(pool.dtype))


def test_append_in_place_and_keys_only(ctx, pkg):
    r = rng(11)
    H, KVH, hd, half = 4, 2, 64, 32
    batch = Batch(r, [(3, 9), (6, 6)], 4)
    cos, sin = _tables(pkg, 16, half)
    qkv = r.normal(size=(batch.rows, (H + 2 * KVH) * hd)).astype(np.float32)
    pool = Pool(pkg, r, "f32", "head", batch.num_pages, 4, KVH, hd)
    q64, k64, v64 = _expect(batch, pool, qkv, H, half, cos, sin, 16)
    mag = 2 * float(np.abs(qkv).max())
    with device(ctx) as d:
        out, kv, b = _call(ctx, pkg, d, pool, batch, qkv, H, half, cos, sin, 16, in_place=True)
        got = d.get(out, qkv.shape, np.float32)
        _close(got[:, :H * hd].reshape(-1, H, hd).astype(np.float64), q64, 0.0, mag)
        assert np.array_equal(got[:, H * hd:], qkv[:, H * hd:])       # the k and v parts of the rows stay
        _close(d.get(pool.dk, pool.k.shape, np.float32).astype(np.float64), k64, 0.0, mag)
        # keys and values only, from arrays of their own
        kv2 = pool.put(d)
        kin, vin = (d.put(np.ascontiguousarray(x)) for x in (qkv[:, H * hd:(H + KVH) * hd], qkv[:, (H + KVH) * hd:]))
        ctx.paged_append(kv2, b, 0, 0, kin, vin, KVH * hd, 0, d.put(cos), d.put(sin), half, 16)
        _close(d.get(pool.dk, pool.k.shape, np.float32).astype(np.float64), k64, 0.0, mag)
        assert np.array_equal(d.get(pool.dv, pool.v.shape, np.float32), v64.astype(np.float32))


def test_append_skips_rows_without_a_place(ctx, pkg):
    """Bad page ids, positions past the rotation tables or before 0, rows of nobody."""
    r = rng(12)
    H, KVH, hd, half, page = 4, 2, 64, 32, 4
    seqs = [(3, 9), (2, 6), (4, 2), (3, 21)]          # the third has rows at positions -2 and -1
    batch = Batch(r, seqs, page, pad_rows=2, bad={(0, 2): -1, (1, 1): 10 ** 6, (3, 5): -2 ** 31})
    pool = Pool(pkg, r, "f16", "head", batch.num_pages, page, KVH, hd)
    cos, sin = _tables(pkg, 20, half)                 # position 20 of the last is past them (and on a bad page)
    qkv = r.normal(size=(batch.rows, (H + 2 * KVH) * hd)).astype(np.float32)
    q64, k64, v64 = _expect(batch, pool, qkv, H, half, cos, sin, 20)
    with device(ctx) as d:
        out, _, _ = _call(ctx, pkg, d, pool, batch, qkv, H, half, cos, sin, 20)
        mag = 2 * float(np.abs(qkv).max())
        _close(d.get(out, q64.shape, np.float32).astype(np.float64), q64, 0.0, mag)
        _close(d.get(pool.dk, pool.k.shape, np.float16).astype(np.float64), k64, EPS16, mag)
        assert np.array_equal(d.get(pool.dv, pool.v.shape, np.float16), v64.astype(np.float16))


def test_append_row_offsets_that_are_none(ctx, pkg):
    """Offsets that do not ascend, or leave the row arrays, touch nothing."""
    r = rng(13)
    H, KVH, hd, page = 4, 2, 64, 4
    batch = Batch(r, [(2, 4), (2, 4)], page)
    pool = Pool(pkg, r, "f32", "head", batch.num_pages, page, KVH, hd)
    qkv = r.normal(size=(batch.rows, (H + 2 * KVH) * hd)).astype(np.float32)
    z = np.zeros((1, 1), np.float32)
    for starts in ([-5, -3, -1], [0, 100, 200], [4, 2, 0], [2 ** 31 - 1, 2 ** 31 - 1, 2 ** 31 - 1]):
        batch.row_start = np.array(starts, dtype=np.int32)
        with device(ctx) as d:
            out, _, _ = _call(ctx, pkg, d, pool, batch, qkv, H, 0, z, z, 1)
            assert np.all(np.isnan(d.get(out, (batch.rows, H * hd), np.float32)))
            assert np.array_equal(d.get(pool.dk, pool.k.shape, np.float32), pool.k)
            assert np.array_equal(d.get(pool.dv, pool.v.shape, np.float32), pool.v)


def test_append_replays_take_the_arrays_of_the_moment(ctx, pkg):
    """One captured append, replayed for three steps of a growing sequence."""
    r = rng(14)
    H, KVH, hd, half, page = 4, 2, 64, 32, 4
    batch = Batch(r, [(1, 12), (1, 12)], page)
    pool = Pool(pkg, r, "f32", "head", batch.num_pages, page, KVH, hd)
    cos, sin = _tables(pkg, 16, half)
    qkv = r.normal(size=(2, (H + 2 * KVH) * hd)).astype(np.float32)
    with device(ctx) as d:
        ctx.synchronize()
        bufs = pool.put(d), batch.put(pkg, d), d.put(qkv), d.put(np.zeros((2, H * hd), np.float32)), d.put(cos), d.put(sin)
        kv, b, p, out, dc, ds = bufs
        ctx.capture_begin()
        ctx.paged_append(kv, b, H, p, p + 4 * H * hd, p + 4 * (H + KVH) * hd, qkv.shape[1], out, dc, ds, half, 16)
        g = ctx.capture_end()
        k = pool.k.astype(np.float64)
        for step in range(3):
            lens = np.array([5 + step, 9 - step], dtype=np.int32)
            x = r.normal(size=qkv.shape).astype(np.float32)
            ctx.h2d(batch.d[1], lens)
            ctx.h2d(p, x)
            ctx.graph_launch(g)
            ctx.synchronize()
            batch.seqs = [(1, int(lens[0])), (1, int(lens[1]))]
            pool.k = k.astype(np.float32)
            _, k, _ = _expect(batch, pool, x, H, half, cos, sin, 16)
            _close(d.get(pool.dk, pool.k.shape, np.float32).astype(np.float64), k, 0.0, 2 * float(np.abs(x).max()))
            k = d.get(pool.dk, pool.k.shape, np.float32).astype(np.float64)
        ctx.graph_destroy(g)


def test_append_refusals(ctx, pkg):
    r = rng(15)
    H, KVH, hd, page = 4, 2, 64, 4
    batch = Batch(r, [(2, 4)], page)
    pool = Pool(pkg, r, "f32", "head", batch.num_pages, page, KVH, hd)
    row = (H + 2 * KVH) * hd
    with device(ctx) as d:
        kv, b = pool.put(d), batch.put(pkg, d)
        p, o = d.put(np.zeros((2, row), np.float32)), d.put(np.zeros((2, H * hd), np.float32))
        t = d.put(np.ones((8, 32), np.float32))
        ok = dict(kv=kv, b=b, H=H, q=p, qs=row, k=p + 4 * H * hd, ks=row, v=p + 4 * (H + KVH) * hd, vs=row, o=o,
                  os=H * hd, c=t, s=t, half=32, n=8)

        def call(**ch):
            a = dict(ok, **ch)
            return ctx.lib.qora_hip_paged_append(
                ctx.h, ctypes.byref(a["kv"]) if a["kv"] else None, ctypes.byref(a["b"]) if a["b"] else None, a["H"],
                a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["o"], a["os"], a["c"], a["s"], a["half"], a["n"],
                None)

        assert call() == pkg.QORA_HIP_OK
        bad = [dict(kv=None), dict(b=None), dict(q=None), dict(o=None), dict(k=None), dict(v=None), dict(c=None),
               dict(s=None), dict(half=33), dict(n=0), dict(H=0), dict(qs=H * hd - 4), dict(ks=KVH * hd - 4),
               dict(qs=row + 1), dict(q=p + 4), dict(o=p + 16, os=row), dict(os=H * hd - 4),
               dict(o=p + 4 * H * hd, os=row), dict(o=p + 4 * row - 16 * hd, os=row), dict(qs=2 ** 30)]
        for ch in bad:
            assert call(**ch) == pkg.QORA_HIP_E_INVALID, ch
        # nothing to do is no error, whatever the row arrays are
        empty = pkg.PagedBatch(0, 0, 0, 0, 0, 0, 0)
        assert call(b=empty, q=None, o=None, k=None, v=None) == pkg.QORA_HIP_OK
        ctx.synchronize()
