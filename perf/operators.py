"""Performance cases of the many-request serving operators on one GPU.

Three operators of a server that runs many sequences through one model:
appending a batch's new keys and values to a paged cache with the position
rotation on the way, causal attention of the new rows (one token or a chunk of
a prompt, mixed freely in a batch) over that cache, and a projection shared by
all rows with a low-rank adapter of each row's own request beside it.

Head counts and matrix sizes are SmolLM3-3B's (16 query heads over 4 KV heads
of 128; 2048 and 11008 wide) and those of the smaller test models. `run` either
computes the operators in plain 32-bit tensor operations or, where `own` is
true, calls the library.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

DEV = "cuda:0"
THETA = 5e6
HEADS = dict(heads=16, kv_heads=4, head_dim=128)


def listed():
    return [
        # One decode step of 32 requests: a row each, rotated and appended.
        # Launch latency is everything.
        dict(HEADS, name="append_decode", op="append", kv="f16", page=16, order="head", seqs=32, new=1, ctx=1000,
             mix="decode", half=64, ragged=1),
        # Prompts admitted together: ragged chunks of up to 2048 tokens into
        # the f32 cache.
        dict(HEADS, name="append_prompts", op="append", kv="f32", page=64, order="head", seqs=4, new=2048, ctx=300,
             mix="chunk", half=64, ragged=2),
        # A layer without rotation and the slot-major page layout, with a page
        # size that is no power of two; q is passed on unrotated.
        dict(name="append_nope", op="append", kv="f16", page=24, order="slot", seqs=7, new=333, ctx=700, mix="chunk",
             heads=12, kv_heads=4, head_dim=128, half=0, ragged=3),
        # One user's next token: the smallest attention call.
        dict(HEADS, name="attn_one", op="attn", kv="f16", page=16, order="head", seqs=1, new=1, ctx=2000,
             mix="decode", ragged=4),
        # The decode step of a busy server: 32 requests of very different age.
        dict(HEADS, name="attn_decode", op="attn", kv="f16", page=16, order="head", seqs=32, new=1, ctx=8192,
             mix="decode", ragged=5),
        # The same with the reference's f32 cache and as many KV heads as
        # query heads, of 64.
        dict(name="attn_decode_f32", op="attn", kv="f32", page=32, order="slot", seqs=16, new=1, ctx=4096,
             mix="decode", heads=8, kv_heads=8, head_dim=64, ragged=6),
        # Two requests at the end of the position table: few rows, long keys.
        dict(HEADS, name="attn_long", op="attn", kv="f16", page=256, order="head", seqs=2, new=1, ctx=65535,
             mix="decode", ragged=7),
        # A chunk of a long prompt behind what is cached of it.
        dict(HEADS, name="attn_chunk", op="attn", kv="f16", page=64, order="head", seqs=1, new=512, ctx=7680,
             mix="chunk", ragged=8),
        # Ragged chunks over the f32 cache, three query heads a KV head.
        dict(name="attn_chunk_f32", op="attn", kv="f32", page=24, order="head", seqs=3, new=300, ctx=1500,
             mix="chunk", heads=12, kv_heads=4, head_dim=128, ragged=9),
        # Continuous batching: one request's prompt chunk beside the single
        # tokens of sixteen others.
        dict(HEADS, name="attn_mixed", op="attn", kv="f16", page=16, order="head", seqs=17, new=509, ctx=4096,
             mix="mixed", ragged=10),
        # The o projection of one decode step: 32 requests over 12 adapters,
        # some rows without one.
        dict(name="lora_decode", op="lora", fmt="q4", tokens=32, k=2048, n=2048, adapters=12, rank=16, run=1,
             ragged=11),
        # The gate projection of a prompt block: four requests' rows in turn.
        dict(name="lora_prompt", op="lora", fmt="q4", tokens=512, k=2048, n=11008, adapters=4, rank=64, run=130,
             ragged=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "attn", "lora"])
    ragged = rng.randint(100, 1 << 20)
    if op == "lora":
        # (weights of at most the gate projection's size)
        k, n = 32 * _log_int(rng, 8, 344), 32 * _log_int(rng, 8, 344)
        n = max(256, min(n, 2048 * 11008 // k // 32 * 32))
        return dict(op=op, fmt=rng.choice(["q4", "q4", "f16"]), tokens=_log_int(rng, 1, 512), k=k, n=n,
                    adapters=_log_int(rng, 1, 32), rank=rng.choice([1, 4, 8, 13, 16, 32, 64]),
                    run=_log_int(rng, 1, 200), ragged=ragged)
    heads, kv_heads, head_dim = rng.choice([(16, 4, 128), (16, 4, 128), (4, 2, 64), (8, 8, 64), (12, 4, 128)])
    c = dict(op=op, kv=rng.choice(["f16", "f16", "f32"]), page=rng.choice([16, 16, 24, 32, 64, 256]),
             order=rng.choice(["head", "slot"]), mix=rng.choice(["decode", "chunk", "mixed"]), heads=heads,
             kv_heads=kv_heads, head_dim=head_dim, ragged=ragged)
    if op == "append":
        return dict(c, seqs=_log_int(rng, 1, 32), new=1 if c["mix"] == "decode" else _log_int(rng, 2, 512),
                    ctx=_log_int(rng, 1, 1000), half=rng.choice([0, head_dim // 2, head_dim // 2, head_dim // 4]))
    c.update(seqs=_log_int(rng, 1, 32), new=1 if c["mix"] == "decode" else _log_int(rng, 2, 512),
             ctx=_log_int(rng, 1, 32768))
    # no more work, and no larger a padded score matrix, than the listed cases have
    while c["ctx"] > 1:
        w = work(c)
        if (w["flops"] < 3e10 and w["bytes"] < 3e8
                and c["seqs"] * c["new"] * (c["ctx"] + c["new"]) * c["heads"] < 6e8):
            break
        c["ctx"] = c["ctx"] * 2 // 3
        c["seqs"] = max(1, c["seqs"] * 4 // 5)
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFFFFFFFFFF)
    return g


def _normal(seed, stream, *shape, std=1.0):
    return torch.randn(*shape, generator=_gen(seed, stream), device=DEV, dtype=torch.float32) * std


def _lengths(c):
    """(new rows, positions cached with them) of each sequence: a matter of the case, not of the seed."""
    r = random.Random(c["ragged"])
    new, kv = [], []
    for i in range(c["seqs"]):
        n = c["new"] if i == 0 else (1 if c["mix"] == "mixed" else c["new"])
        if c["mix"] == "chunk" and i > 0:
            n = r.randint(1, c["new"])
        old = c["ctx"] if i == 0 else r.randint(0, c["ctx"])
        new.append(n)
        kv.append(old + n)
    return new, kv


def _batch(c, seed):
    """The batch as a server holds it: row offsets, lengths, page tables; pages are handed out in random order."""
    new, kv = _lengths(c)
    need = [-(-x // c["page"]) for x in kv]
    perm = torch.randperm(sum(need), generator=_gen(seed, 1), device=DEV).to(torch.int32)
    pages = torch.zeros(c["seqs"], max(need), dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        pages[i, :n] = perm[at:at + n]
        at += n
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(pages=pages, num_pages=at, rows=start[-1],
                row_start=torch.tensor(start, dtype=torch.int32, device=DEV),
                kv_len=torch.tensor(kv, dtype=torch.int32, device=DEV))


def _pool_shape(c, num_pages):
    inner = (c["kv_heads"], c["page"]) if c["order"] == "head" else (c["page"], c["kv_heads"])
    return (num_pages, *inner, c["head_dim"])


def _cache(c, seed, num_pages):
    dt = torch.float16 if c["kv"] == "f16" else torch.float32
    return tuple(_normal(seed, i, *_pool_shape(c, num_pages)).to(dt) for i in (2, 3))


def _rope(positions, half):
    f = THETA ** (-torch.arange(half, device=DEV, dtype=torch.float64) / max(half, 1))
    a = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _weight(c, seed):
    """The shared weight's stored values: (bytes [k][n/2], f16 scales [k][n/32]) or f16 [k][n]."""
    k, n = c["k"], c["n"]
    if c["fmt"] == "f16":
        return (_normal(seed, 2, k, n, std=0.02).half(),)
    b = torch.randint(0, 225, (k, n // 2), generator=_gen(seed, 2), device=DEV, dtype=torch.uint8)
    packed = (b % 15 + 1) | ((torch.div(b, 15, rounding_mode="floor") + 1) << 4)
    return packed, (torch.randn(k, n // 32, generator=_gen(seed, 3), device=DEV).abs() * (0.02 / 7)).half()


def _ranks(c):
    r = random.Random(c["ragged"])
    return [c["rank"]] + [r.randint(1, c["rank"]) for _ in range(c["adapters"] - 1)]


def _row_adapters(c):
    """Each row's adapter: runs of rows of one request, about one in eight of them without an adapter."""
    r = random.Random(c["ragged"] + 1)
    out = []
    while len(out) < c["tokens"]:
        a = -1 if out and r.random() < 0.125 else r.randrange(c["adapters"])
        out += [a] * (r.randint(1, c["run"]) if c["run"] > 1 else 1)
    return out[: c["tokens"]]


def _adapters(c, seed):
    """a [adapters][k][rank] and b [adapters][rank][n] in binary16, zero past an adapter's own rank."""
    a = _normal(seed, 4, c["adapters"], c["k"], c["rank"], std=1.0 / math.sqrt(c["k"]))
    b = _normal(seed, 5, c["adapters"], c["rank"], c["n"], std=0.05)
    for i, r in enumerate(_ranks(c)):
        a[i, :, r:] = 0
        b[i, r:] = 0
    return a.half(), b.half()


def _scales(c):
    return [2.0 / r for r in _ranks(c)]


def prepare(case, seed):
    c = case
    s = dict(case=c)
    if c["op"] == "lora":
        s.update(x=_normal(seed, 1, c["tokens"], c["k"]), w=_weight(c, seed), y=torch.zeros(c["tokens"], c["n"], device=DEV),
                 row_adapter=torch.tensor(_row_adapters(c), dtype=torch.int32, device=DEV),
                 scale=torch.tensor(_scales(c), device=DEV))
        s["a"], s["b"] = _adapters(c, seed)
    else:
        H, KVH, hd = c["heads"], c["kv_heads"], c["head_dim"]
        s["b"] = b = _batch(c, seed)
        s["k"], s["v"] = _cache(c, seed, b["num_pages"])
        if c["op"] == "append":
            # the rows of the fused q|k|v projection
            s["qkv"] = _normal(seed, 4, b["rows"], (H + 2 * KVH) * hd)
            s["q_out"] = torch.zeros(b["rows"], H * hd, device=DEV)
            s["cos"], s["sin"] = _rope(max(_lengths(c)[1]), c["half"])
        else:
            s["q"] = _normal(seed, 4, b["rows"], H * hd, std=1.5)
            s["out"] = torch.zeros(b["rows"], H * hd, device=DEV)
    if own:
        _prepare_own(s)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------

def _prepare_own(s):
    pkg = importlib.import_module("qora-llm_amd")
    c = s["case"]
    s["ctx"] = ctx = pkg.HipContext(0)
    if c["op"] == "lora":
        w = [t.cpu().numpy() for t in s["w"]]
        if c["fmt"] == "q4":
            weight = pkg.Weight(c["k"], c["n"], packed=w[0].reshape(-1), scales=w[1].view("uint16").reshape(-1))
        else:
            weight = pkg.Weight(c["k"], c["n"], data=w[0].view("uint16").reshape(-1))
        s["wid"] = ctx.upload(weight)
        a, b = s["a"].cpu().numpy(), s["b"].cpu().numpy()
        s["lora"] = ctx.lora_upload([pkg.LoraAdapter(a[i, :, :r], b[i, :r], scale)
                                     for i, (r, scale) in enumerate(zip(_ranks(c), _scales(c)))], c["tokens"])
        return
    H, KVH, hd, page, b = c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["b"]
    head, slot = (page * hd, hd) if c["order"] == "head" else (hd, KVH * hd)
    s["kv"] = pkg.PagedKV(s["k"].data_ptr(), s["v"].data_ptr(), pkg.KV_F16 if c["kv"] == "f16" else pkg.KV_F32,
                          b["num_pages"], page, KVH, hd, KVH * page * hd, head, slot)
    s["batch"] = pkg.PagedBatch(b["row_start"].data_ptr(), b["kv_len"].data_ptr(), b["pages"].data_ptr(), c["seqs"],
                                b["pages"].shape[1], b["rows"], c["new"])
    if c["op"] == "attn":
        s["attn"] = ctx.paged_attn_prepare(b["rows"], c["seqs"], H, KVH, hd)


def _run_own(s):
    c, ctx = s["case"], s["ctx"]
    H, KVH, hd = c["heads"], c["kv_heads"], c["head_dim"]
    if c["op"] == "append":
        p, ld = s["qkv"].data_ptr(), (H + 2 * KVH) * hd
        ctx.paged_append(s["kv"], s["batch"], H, p, p + 4 * H * hd, p + 4 * (H + KVH) * hd, ld, s["q_out"].data_ptr(),
                         s["cos"].data_ptr(), s["sin"].data_ptr(), c["half"], s["cos"].shape[0])
        return s["q_out"], s["k"], s["v"]
    ctx.paged_attn_run(s["attn"], s["kv"], s["batch"], s["q"].data_ptr(), s["out"].data_ptr())
    return s["out"]


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def _slots(c, b, pos, seq):
    """Page and slot of position pos (a tensor) of sequence seq."""
    return b["pages"][seq, pos // c["page"]].long(), pos % c["page"]


def _row_places(c, b):
    """Sequence and position of each row."""
    row = torch.arange(b["rows"], device=DEV)
    seq = torch.searchsorted(b["row_start"][1:].long(), row, right=True)
    return seq, b["kv_len"].long()[seq] - (b["row_start"].long()[seq + 1] - row)


def _rotate(x, cos, sin, half):
    if half == 0:
        return x
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), -1)


def _append_plain(s):
    c, b = s["case"], s["b"]
    H, KVH, hd, half = c["heads"], c["kv_heads"], c["head_dim"], c["half"]
    seq, pos = _row_places(c, b)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    qkv = s["qkv"].view(b["rows"], H + 2 * KVH, hd)
    s["q_out"].copy_(_rotate(qkv[:, :H], cos, sin, half).reshape(b["rows"], H * hd))
    k, v = _rotate(qkv[:, H:H + KVH], cos, sin, half), qkv[:, H + KVH:]
    page, slot = _slots(c, b, pos, seq)
    for pool, new in ((s["k"], k), (s["v"], v)):
        rows = pool.transpose(1, 2) if c["order"] == "head" else pool     # [page][slot][kv head][dim]
        rows[page, slot] = new.to(pool.dtype)
    return s["q_out"], s["k"], s["v"]


def _attn_plain(s):
    c, b = s["case"], s["b"]
    H, KVH, hd, S = c["heads"], c["kv_heads"], c["head_dim"], c["seqs"]
    G, nmax, lmax = H // KVH, c["new"], max(_lengths(c)[1])
    # keys and values of every sequence, padded to the longest: [S][kv head][lmax][dim]
    key = torch.arange(lmax, device=DEV)
    held = key < b["kv_len"][:, None]
    page, slot = _slots(c, b, torch.where(held, key, 0), torch.arange(S, device=DEV)[:, None])
    kv = []
    for pool in (s["k"], s["v"]):
        rows = pool.transpose(1, 2) if c["order"] == "head" else pool
        kv.append(rows[page, slot].float().permute(0, 2, 1, 3).contiguous())
    # the queries, padded to the most rows: [S][kv head][nmax * G][dim]
    seq, pos = _row_places(c, b)
    at = torch.arange(b["rows"], device=DEV) - b["row_start"].long()[seq]
    q = torch.zeros(S, nmax, H, hd, device=DEV)
    q[seq, at] = s["q"].view(-1, H, hd)
    qpos = (b["kv_len"].long() - (b["row_start"][1:] - b["row_start"][:-1]))[:, None] + torch.arange(nmax, device=DEV)
    q = q.view(S, nmax, KVH, G, hd).permute(0, 2, 1, 3, 4).reshape(S, KVH, nmax * G, hd)
    sc = torch.matmul(q, kv[0].transpose(2, 3)).view(S, KVH, nmax, G, lmax) / math.sqrt(hd)
    see = (key <= qpos[..., None]) & held[:, None]
    sc = sc.masked_fill(~see[:, None, :, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    o = torch.matmul(p.view(S, KVH, nmax * G, lmax), kv[1]).view(S, KVH, nmax, G, hd)
    o = o / p.sum(-1, keepdim=True)
    s["out"].copy_(o.permute(0, 2, 1, 3, 4).reshape(S, nmax, H * hd)[seq, at])
    return s["out"]


def _dequant(c, w, dt):
    if c["fmt"] == "f16":
        return w[0].to(dt)
    q = torch.stack((w[0] & 15, w[0] >> 4), dim=-1).reshape(c["k"], c["n"]).to(dt) - 8.0
    return (q.reshape(c["k"], c["n"] // 32, 32) * w[1].to(dt).unsqueeze(-1)).reshape(c["k"], c["n"])


def _lora_plain(s):
    c, x = s["case"], s["x"]
    E, R = c["adapters"], c["rank"]
    # every row through every adapter, and only its own kept
    u = torch.matmul(x, s["a"].float().permute(1, 0, 2).reshape(c["k"], E * R)).view(-1, E, R)
    mine = s["row_adapter"][:, None] == torch.arange(E, device=DEV)
    u = u * (mine * s["scale"])[..., None]
    s["y"].copy_(torch.matmul(x, _dequant(c, s["w"], torch.float32))
                 + torch.matmul(u.view(-1, E * R), s["b"].float().view(E * R, c["n"])))
    return s["y"]


def run(state):
    op = state["case"]["op"]
    if op == "lora":
        if own:
            state["ctx"].gemm_lora(state["wid"], state["lora"], state["x"].data_ptr(), state["y"].data_ptr(),
                                   state["case"]["tokens"], state["row_adapter"].data_ptr())
            return state["y"]
        return _lora_plain(state)
    if own:
        return _run_own(state)
    return _append_plain(state) if op == "append" else _attn_plain(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "lora":
        rows, used = _row_adapters(c), 0
        for a in sorted(set(rows) - {-1}):
            used += _ranks(c)[a] * (c["k"] + c["n"])
        kn = c["k"] * c["n"]
        wb = 2 * kn if c["fmt"] == "f16" else kn // 2 + kn // 16
        low = sum(_ranks(c)[a] for a in rows if a >= 0) * (c["k"] + c["n"])
        return {"bytes": wb + 2 * used + 4 * c["tokens"] * (c["k"] + c["n"] + 1),
                "flops": 2 * c["tokens"] * kn + 2 * low}
    new, kv = _lengths(c)
    es, H, KVH, hd = 2 if c["kv"] == "f16" else 4, c["heads"], c["kv_heads"], c["head_dim"]
    rows = sum(new)
    if c["op"] == "append":
        return {"bytes": rows * hd * (8 * H + KVH * 2 * (4 + es) + (8 * c["half"] // hd)),
                "flops": 6 * rows * (H + KVH) * c["half"]}
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, kv))
    return {"bytes": sum(kv) * KVH * hd * 2 * es + 8 * rows * H * hd + 4 * sum(-(-L // c["page"]) for L in kv),
            "flops": 4 * seen * H * hd}


def exact(case, seed):
    c = case
    if c["op"] == "lora":
        x, y = _normal(seed, 1, c["tokens"], c["k"]).double(), None
        y = x @ _dequant(c, _weight(c, seed), torch.float64)
        a, b = _adapters(c, seed)
        rows, scale = _row_adapters(c), torch.tensor(_scales(c)).tolist()
        for i in range(c["adapters"]):
            at = [t for t, r in enumerate(rows) if r == i]
            if at:
                y[at] += scale[i] * (x[at] @ a[i].double()) @ b[i].double()
        return y
    H, KVH, hd = c["heads"], c["kv_heads"], c["head_dim"]
    new, kv = _lengths(c)
    b = _batch(c, seed)
    pools = _cache(c, seed, b["num_pages"])
    starts, pages = b["row_start"].tolist(), b["pages"]
    if c["op"] == "append":
        qkv = _normal(seed, 4, b["rows"], (H + 2 * KVH) * hd).double().view(b["rows"], H + 2 * KVH, hd)
        cos, sin = (t.double() for t in _rope(max(kv), c["half"]))
        dt, half = pools[0].dtype, c["half"]
        k, v = (p.double() for p in pools)
        q_out = torch.empty(b["rows"], H * hd, device=DEV, dtype=torch.float64)
        for i in range(c["seqs"]):
            x = qkv[starts[i]:starts[i + 1]].clone()
            pos = torch.arange(kv[i] - new[i], kv[i], device=DEV)
            cs, sn = cos[pos][:, None], sin[pos][:, None]
            lo, hi = x[:, :H + KVH, :half].clone(), x[:, :H + KVH, half:2 * half].clone()
            x[:, :H + KVH, :half] = lo * cs - hi * sn
            x[:, :H + KVH, half:2 * half] = hi * cs + lo * sn
            q_out[starts[i]:starts[i + 1]] = x[:, :H].reshape(-1, H * hd)
            page, slot = pages[i, pos // c["page"]].long(), pos % c["page"]
            for pool, rows in ((k, x[:, H:H + KVH]), (v, x[:, H + KVH:])):
                if c["order"] == "head":
                    pool[page, :, slot] = rows
                else:
                    pool[page, slot] = rows
        return q_out, k, v
    q = _normal(seed, 4, b["rows"], H * hd, std=1.5).double().view(-1, H, hd)
    out = torch.empty(b["rows"], H * hd, device=DEV, dtype=torch.float64).view(-1, H, hd)
    for i in range(c["seqs"]):
        own_pages = pages[i, : -(-kv[i] // c["page"])].long()
        k, v = ((p[own_pages] if c["order"] == "slot" else p[own_pages].transpose(1, 2)).double()
                .reshape(-1, KVH, hd)[: kv[i]] for p in pools)
        rows = slice(starts[i], starts[i + 1])
        hidden = torch.arange(kv[i], device=DEV) > torch.arange(kv[i] - new[i], kv[i], device=DEV)[:, None]
        for h in range(H):
            kh, vh = k[:, h // (H // KVH)], v[:, h // (H // KVH)]
            out[rows, h] = torch.softmax((q[rows, h] @ kh.t() / math.sqrt(hd)).masked_fill(hidden, -math.inf), -1) @ vh
    return out.reshape(-1, H * hd)
