"""The many-request calls together, as a server's attention block uses them:
q, k and v with each request's adapter, append, attention, the o projection.
Prompts of different length first, then single tokens, eagerly and from one
captured graph; every stage against float64 on the stage's own inputs."""
import numpy as np
import pytest

from helpers import dequant_np, device, random_q4, rng
from paged_util import EPS32, Batch, Pool, attention64, rotate64
from test_gpu_lora import _adapters, _truth

pytestmark = pytest.mark.gpu

HID, H, KVH, HD, PAGE, HALF = 256, 4, 2, 64, 16, 32
POSITIONS = 400


class Layer:
    def __init__(self, ctx, pkg, r, max_rows):
        self.ctx, self.pkg = ctx, pkg
        self.w, self.ad, self.wid, self.lid = {}, {}, {}, {}
        for name, k, n in (("q", HID, H * HD), ("k", HID, KVH * HD), ("v", HID, KVH * HD), ("o", H * HD, HID)):
            packed, scales = random_q4(r, k, n)
            self.w[name] = dequant_np(packed, scales, k, n)
            self.ad[name] = _adapters(pkg, r, [8, 16, 5], k, n)
            self.wid[name] = ctx.upload(pkg.Weight(k, n, packed=packed, scales=scales))
            self.lid[name] = ctx.lora_upload(self.ad[name], max_rows)
        c, s = pkg.rope_tables(POSITIONS, HALF, 5e6)
        self.cos, self.sin = c.reshape(POSITIONS, HALF), s.reshape(POSITIONS, HALF)
        self.attn = ctx.paged_attn_prepare(max_rows, 4, H, KVH, HD)

    def buffers(self, d, rows):
        self.dcos, self.dsin = d.put(self.cos), d.put(self.sin)
        self.b = {n: d.empty(rows * c * 4) for n, c in (("x", HID), ("q", H * HD), ("k", KVH * HD), ("v", KVH * HD),
                                                        ("qr", H * HD), ("a", H * HD), ("y", HID))}
        self.drows = d.put(np.zeros(rows, np.int32))

    def run(self, kv, batch, rows):
        c, b = self.ctx, self.b
        for n in "qkv":
            c.gemm_lora(self.wid[n], self.lid[n], b["x"], b[n], rows, self.drows)
        c.paged_append(kv, batch, H, b["q"], b["k"], b["v"], H * HD, b["qr"], self.dcos, self.dsin, HALF, POSITIONS,
                       k_stride=KVH * HD, v_stride=KVH * HD)
        c.paged_attn_run(self.attn, kv, batch, b["qr"], b["a"])
        c.gemm_lora(self.wid["o"], self.lid["o"], b["a"], b["y"], rows, self.drows)

    def close(self):
        for lid in self.lid.values():
            self.ctx.lora_release(lid)
        self.ctx.paged_attn_release(self.attn)


def _check_step(layer, d, pool, batch, x, adapters, rows):
    """Each stage's output against float64 on what the stage before left on the device."""
    get = {n: d.get(layer.b[n], (rows, c), np.float32) for n, c in (("q", H * HD), ("k", KVH * HD), ("v", KVH * HD),
                                                                    ("qr", H * HD), ("a", H * HD), ("y", HID))}
    for n in "qkv":
        ref, tol = _truth(x, layer.w[n], layer.ad[n], adapters)
        assert np.all(np.abs(get[n] - ref) <= tol), n
    pool.k, pool.v = d.get(pool.dk, pool.k.shape, np.float32), d.get(pool.dv, pool.v.shape, np.float32)
    for row, s, pos in batch.row_places():
        cos, sin = layer.cos[pos].astype(np.float64), layer.sin[pos].astype(np.float64)
        mag = 2 * np.abs(get["q"][row]).max()
        assert np.all(np.abs(get["qr"][row].reshape(H, HD) - rotate64(get["q"][row].reshape(H, HD), cos, sin, HALF))
                      <= 3 * EPS32 * mag)
        page, slot = batch.place(s, pos)
        for h in range(KVH):
            kr = rotate64(get["k"][row].reshape(KVH, HD)[h], cos, sin, HALF)
            assert np.all(np.abs(pool.k[pool.at(page, h, slot)] - kr) <= 6 * EPS32 * np.abs(get["k"][row]).max())
            assert np.array_equal(pool.v[pool.at(page, h, slot)], get["v"][row].reshape(KVH, HD)[h])
    ref, tol = attention64(pool, batch, get["qr"].reshape(rows, H, HD), H)
    assert np.all(np.abs(get["a"].reshape(rows, H, HD) - ref) <= tol)
    ref, tol = _truth(get["a"], layer.w["o"], layer.ad["o"], adapters)
    assert np.all(np.abs(get["y"] - ref) <= tol)
    return get["y"]


def _set(ctx, batch, seqs):
    batch.seqs = seqs
    batch.row_start = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
    batch.kv_len = np.array([L for _, L in seqs], dtype=np.int32)
    ctx.h2d(batch.d[0], batch.row_start)
    ctx.h2d(batch.d[1], batch.kv_len)


def test_block_of_a_layer_prompts_then_tokens(ctx, pkg):
    r = rng(21)
    prompts = [(5, 5), (130, 130), (1, 1), (33, 33)]
    grow = [(1, n + 6) for n, _ in prompts]                # pages for the tokens to come
    batch = Batch(r, grow, PAGE)
    layer = Layer(ctx, pkg, r, 169)
    pool = Pool(pkg, r, "f32", "head", batch.num_pages, PAGE, KVH, HD, fill=np.nan)
    of_request = np.array([0, 2, -1, 1], dtype=np.int32)
    with device(ctx) as d:
        kv = pool.put(d)
        batch.rows = 169
        cb = batch.put(pkg, d)
        layer.buffers(d, 169)

        def step(seqs, graph=None):
            _set(ctx, batch, seqs)
            rows = int(batch.row_start[-1])
            batch.used = cb.rows = rows
            x = r.normal(size=(rows, HID)).astype(np.float32)
            adapters = np.repeat(of_request, [n for n, _ in seqs])
            ctx.h2d(layer.b["x"], x)
            ctx.h2d(layer.drows, adapters)
            if graph is None:
                layer.run(kv, cb, rows)
            else:
                ctx.graph_launch(graph)
            ctx.synchronize()
            return _check_step(layer, d, pool, batch, x, adapters, rows)

        step(prompts)
        for i in range(2):
            step([(1, n + 1 + i) for n, _ in prompts])
        # the same single-token step from a graph: its replays follow the arrays
        ctx.capture_begin()
        layer.run(kv, cb, 4)
        g = ctx.capture_end()
        for i in range(2, 5):
            step([(1, n + 1 + i) for n, _ in prompts], graph=g)
        y = step([(1, n + 6) for n, _ in prompts], graph=g)
        # and an eager step in between the replays leaves nothing behind
        _set(ctx, batch, [(1, n + 6) for n, _ in prompts])
        layer.run(kv, cb, 4)
        ctx.synchronize()
        assert np.array_equal(y, d.get(layer.b["y"], (4, HID), np.float32))
        ctx.graph_launch(g)
        ctx.synchronize()
        assert np.array_equal(y, d.get(layer.b["y"], (4, HID), np.float32))
        ctx.graph_destroy(g)
    layer.close()
