"""qora_hip_gemm_lora against x W + scale (x A) B in float64: ranks, adapters a
row, rows from one to many, both weight formats, in place, replays, refusals."""
import ctypes

import numpy as np
import pytest

from helpers import dequant_np, device, random_q4, rng

pytestmark = pytest.mark.gpu
EPS32 = 2.0 ** -24


def _weight(pkg, r, fmt, k, n):
    if fmt == "q4":
        packed, scales = random_q4(r, k, n)
        return pkg.Weight(k, n, packed=packed, scales=scales), dequant_np(packed, scales, k, n)
    w = r.normal(0, 0.02, size=(k, n)).astype(np.float16)
    return pkg.Weight(k, n, data=w.view(np.uint16).reshape(-1)), w.astype(np.float64)


def _adapters(pkg, r, ranks, k, n):
    return [pkg.LoraAdapter(r.normal(0, k ** -0.5, size=(k, x)).astype(np.float16),
                            r.normal(0, 0.05, size=(x, n)).astype(np.float16), float(np.float32(2.0 / x))) for x in ranks]


def _truth(x, w, ads, rows):
    """(y, tolerance): the product's and the adapters' terms in float64. Each sum of products
    in float32 of operands held to 22 bits is off by (terms + 16) half steps of the sum of
    its terms' sizes; u's error passes through B, and the two parts' sum rounds once more."""
    x = x.astype(np.float64)
    y, mag = x @ w, np.abs(x) @ np.abs(w)
    tol = (x.shape[1] + 16) * EPS32 * mag
    for e, a in enumerate(ads):
        at = np.nonzero(rows == e)[0]
        if at.size == 0:
            continue
        A, B = a.a.astype(np.float64), a.b.astype(np.float64)
        u, um = x[at] @ A, np.abs(x[at]) @ np.abs(A)
        y[at] += a.scale * (u @ B)
        tol[at] += abs(a.scale) * EPS32 * ((x.shape[1] + B.shape[0] + 48) * (um @ np.abs(B)))
    return y, tol + 4 * EPS32 * np.abs(y)


def _rows(r, T, count, run):
    out = []
    while len(out) < T:
        out += [int(r.integers(-1, count))] * int(r.integers(1, run + 1))
    return np.array(out[:T], dtype=np.int32)


CASES = [
    # fmt, k, n, ranks, rows, longest run of rows of one adapter
    ("q4", 2048, 2048, [16] * 12, 32, 1),
    ("q4", 2048, 512, [8], 1, 1),
    ("f16", 2048, 512, [8, 64, 3], 1, 1),
    ("q4", 256, 704, [1, 5, 16, 17, 33, 64], 50, 3),
    ("f16", 96, 32, [13, 200, 256], 7, 2),
    ("f16", 32, 96, [4], 3, 1),
    ("q4", 704, 256, [16, 8, 32], 200, 60),
    ("f16", 512, 384, [24, 64], 300, 130),
    ("q4", 11008, 2048, [64, 16], 5, 2),
    ("q4", 1056, 1088, [16, 32, 100], 17, 17),
    ("q4", 2048, 11008, [64] * 4, 130, 40),
    ("q4", 2048, 512, [16] * 20, 65, 1),               # many tokens, several K slices of x A
    ("f16", 4096, 256, [64, 16, 100], 96, 2),
    ("q4", 5024, 256, [33, 1, 256], 257, 40),
    ("f16", 2080, 160, [17, 40, 8], 1100, 300),
    ("f16", 608, 2080, [5, 48] * 9, 1031, 3),          # many columns and rows, many adapters a block
    ("q4", 1024, 4224, [32] * 5, 400, 2),
]


def _run(ctx, d, wid, lid, x, n, rows, y=0, stream=0):
    dx = d.put(x)
    y = y or d.put(np.full((x.shape[0], n), np.nan, np.float32))
    ctx.gemm_lora(wid, lid, dx, y, x.shape[0], d.put(rows), stream=stream)
    return y


@pytest.mark.parametrize("fmt,k,n,ranks,T,run", CASES)
def test_gemm_lora_matches_definition(ctx, pkg, fmt, k, n, ranks, T, run):
    r = rng(k + n + T)
    weight, w = _weight(pkg, r, fmt, k, n)
    ads = _adapters(pkg, r, ranks, k, n)
    x, rows = r.normal(size=(T, k)).astype(np.float32), _rows(r, T, len(ranks), run)
    rows[0] = len(ranks) - 1
    wid, lid = ctx.upload(weight), ctx.lora_upload(ads, T + 3)
    with device(ctx) as d:
        y1 = d.get(_run(ctx, d, wid, lid, x, n, rows), (T, n), np.float32)
        y2 = d.get(_run(ctx, d, wid, lid, x, n, rows), (T, n), np.float32)
    ctx.lora_release(lid)
    ctx.check(ctx.lib.qora_hip_release_weight(ctx.h, wid))
    ref, tol = _truth(x, w, ads, rows)
    off = np.abs(y1 - ref) - tol
    assert np.all(off <= 0), (float(off.max()), np.unravel_index(np.argmax(off), off.shape))
    assert np.array_equal(y1, y2)


def test_rows_without_an_adapter_are_the_plain_product(ctx, pkg):
    r = rng(2)
    k, n, T = 256, 320, 40
    weight, _ = _weight(pkg, r, "q4", k, n)
    x = r.normal(size=(T, k)).astype(np.float32)
    rows = np.array([-1, 5, 2 ** 31 - 1, -2 ** 31, 3] * 8, dtype=np.int32)     # 3 adapters: ids 0, 1, 2
    wid, lid = ctx.upload(weight), ctx.lora_upload(_adapters(pkg, r, [4, 16, 40], k, n), T)
    with device(ctx) as d:
        y = d.get(_run(ctx, d, wid, lid, x, n, rows), (T, n), np.float32)
        plain = d.empty(y.nbytes)
        ctx.check(ctx.lib.qora_hip_gemm(ctx.h, wid, d.put(x), plain, T, None))
        assert np.array_equal(y, d.get(plain, (T, n), np.float32))
    ctx.lora_release(lid)


@pytest.mark.parametrize("fmt,k,n,T", [("q4", 2048, 512, 130), ("q4", 2048, 8192, 200), ("q4", 640, 96, 100),
                                       ("f16", 2048, 512, 130), ("f16", 512, 4096, 90), ("f16", 4096, 4096, 300),
                                       ("f16", 512, 2080, 30), ("q4", 4096, 256, 9)])
def test_no_adapter_changes_no_bit(ctx, pkg, fmt, k, n, T):
    """Every form of the product: rows without an adapter are qora_hip_gemm's, beside rows that have one."""
    r = rng(k + T)
    weight, w = _weight(pkg, r, fmt, k, n)
    ads = _adapters(pkg, r, [16, 40], k, n)
    x = r.normal(size=(T, k)).astype(np.float32)
    wid, lid = ctx.upload(weight), ctx.lora_upload(ads, T)
    with device(ctx) as d:
        plain = d.empty(T * n * 4)
        ctx.check(ctx.lib.qora_hip_gemm(ctx.h, wid, d.put(x), plain, T, None))
        plain = d.get(plain, (T, n), np.float32)
        for rows in (np.full(T, -1, np.int32), (np.arange(T) % 5 - 3).astype(np.int32)):
            y = d.get(_run(ctx, d, wid, lid, x, n, rows), (T, n), np.float32)
            assert np.array_equal(y[rows < 0], plain[rows < 0])
            ref, tol = _truth(x, w, ads, rows)
            assert np.all(np.abs(y - ref) <= tol)
    ctx.lora_release(lid)
    ctx.check(ctx.lib.qora_hip_release_weight(ctx.h, wid))


def test_rows_of_very_different_size(ctx, pkg):
    """A row's own scale: tiny and huge rows side by side, and one that is not finite."""
    r = rng(3)
    k, n, T = 256, 128, 20
    weight, w = _weight(pkg, r, "f16", k, n)
    ads = _adapters(pkg, r, [16, 8], k, n)
    x = (r.normal(size=(T, k)) * 10.0 ** r.integers(-18, 18, size=(T, 1))).astype(np.float32)
    x[3] = 0
    rows = (np.arange(T) % 3 - 1).astype(np.int32)
    ref, tol = _truth(x, w, ads, rows)
    x[7, 5] = np.nan
    wid, lid = ctx.upload(weight), ctx.lora_upload(ads, T)
    with device(ctx) as d:
        y = d.get(_run(ctx, d, wid, lid, x, n, rows), (T, n), np.float32)
    ctx.lora_release(lid)
    keep = np.arange(T) != 7
    assert np.all(np.abs(y - ref)[keep] <= tol[keep])
    assert not np.any(y[3]) and np.all(np.isnan(y[7]))


def test_in_place_other_stream_and_replays(ctx, pkg):
    r = rng(4)
    k = n = 512
    for T in (3, 40, 150):
        weight, w = _weight(pkg, r, "q4", k, n)
        ads = _adapters(pkg, r, [16, 24], k, n)
        wid, lid = ctx.upload(weight), ctx.lora_upload(ads, T)
        x, rows = r.normal(size=(T, k)).astype(np.float32), _rows(r, T, 2, 9)
        ref, tol = _truth(x, w, ads, rows)
        with device(ctx) as d:
            dx = d.put(x)
            ctx.gemm_lora(wid, lid, dx, dx, T, d.put(rows))
            assert np.all(np.abs(d.get(dx, (T, n), np.float32) - ref) <= tol)
            other = pkg.HipContext(0)
            y = _run(ctx, d, wid, lid, x, n, rows, stream=other.stream)
            other.synchronize()
            assert np.all(np.abs(d.get(y, (T, n), np.float32) - ref) <= tol)
            other.close()
            dx, dr = d.put(x), d.put(rows)
            ctx.capture_begin()
            ctx.gemm_lora(wid, lid, dx, y, T, dr)
            g = ctx.capture_end()
            for i in range(3):
                rows = _rows(r, T, 3, 5) if i else rows
                x = r.normal(size=(T, k)).astype(np.float32) if i == 2 else x
                ctx.h2d(dx, x)
                ctx.h2d(dr, rows)
                ref, tol = _truth(x, w, ads, rows)
                ctx.graph_launch(g)
                ctx.synchronize()
                a = d.get(y, (T, n), np.float32)
                assert np.all(np.abs(a - ref) <= tol)
                ctx.gemm_lora(wid, lid, dx, y, T, dr)
                ctx.synchronize()
                assert np.all(np.abs(d.get(y, (T, n), np.float32) - ref) <= tol)
            ctx.graph_destroy(g)
        ctx.lora_release(lid)


def test_lora_refusals(ctx, pkg):
    r = rng(5)
    weight, _ = _weight(pkg, r, "f16", 64, 96)
    wid, inv = ctx.upload(weight), pkg.QORA_HIP_E_INVALID
    ads = _adapters(pkg, r, [4], 64, 96)
    lid = ctx.lora_upload(ads, 8)
    x = ctypes.c_uint32()

    def desc(a=True, b=True, rank=4):
        return (pkg.LoraAdapterDesc * 1)(pkg.LoraAdapterDesc(ads[0].a.ctypes.data if a else None,
                                                             ads[0].b.ctypes.data if b else None, rank, 1.0))

    for d, cnt, k, n, m in [(None, 1, 64, 96, 8), (desc(a=False), 1, 64, 96, 8), (desc(b=False), 1, 64, 96, 8),
                            (desc(rank=0), 1, 64, 96, 8), (desc(rank=257), 1, 64, 96, 8), (desc(), 0, 64, 96, 8),
                            (desc(), 1, 60, 96, 8), (desc(), 1, 64, 90, 8), (desc(), 1, 64, 96, 0), (desc(), 1, 0, 96, 8)]:
        assert ctx.lib.qora_hip_lora_upload(ctx.h, d, cnt, k, n, m, ctypes.byref(x)) == inv
    with pytest.raises(ValueError):
        ctx.lora_upload([pkg.LoraAdapter(np.zeros((64, 4)), np.zeros((5, 96)))], 8)
    wide = ctx.upload(_weight(pkg, r, "f16", 64, 128)[0])
    with device(ctx) as d:
        dx, y, rows = d.put(np.ones((9, 64), np.float32)), d.empty(9 * 96 * 4), d.put(np.zeros(9, np.int32))

        def call(w=wid, i=lid, x=dx, y=y, T=8, rows=rows):
            return ctx.lib.qora_hip_gemm_lora(ctx.h, w, i, x, y, T, rows, None)

        assert call() == pkg.QORA_HIP_OK
        for ch in [dict(w=10 ** 6), dict(i=10 ** 6), dict(x=None), dict(y=None), dict(rows=None), dict(T=0), dict(T=9),
                   dict(w=wide)]:
            assert call(**ch) == inv, ch
        ctx.synchronize()
        ctx.capture_begin()
        assert ctx.lib.qora_hip_lora_upload(ctx.h, desc(), 1, 64, 96, 8, ctypes.byref(x)) == pkg.QORA_HIP_E_STATE
        assert ctx.lib.qora_hip_lora_release(ctx.h, lid) == pkg.QORA_HIP_E_STATE
        ctx.graph_destroy(ctx.capture_end())
        ctx.lora_release(lid)
        assert call() == inv and ctx.lib.qora_hip_lora_release(ctx.h, lid) == inv
