"""Timed cases of the paged cache's operators: the producer that rotates new
rows into pages, attention over a page table, and copies of pages.

A case is a dict of plain values: "op" names the operator, the rest its sizes.
listed() holds the representative ones, draw() gives others of the same ranges,
prepare() makes what a program has in hand before the call, run() is one pass
(in plain torch operations, or with `own` through toklet_amd.ops), exact() is
the same result in 64-bit floating point, and work() what a pass cannot do
without.
"""

from __future__ import annotations

import functools
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ES = {"f32": 4, "f16": 2, "bf16": 2}
# Query heads / KV heads / head_dim: those the session path serves, and a
# multi-head and a single-KV-head layout.
_SHAPES = ((14, 2, 64), (16, 8, 128), (32, 8, 128), (8, 4, 256))
_MORE = _SHAPES + ((12, 12, 64), (8, 1, 128))


def _case(name, op, heads, dtype, page, **more):
    hq, hkv, d = heads
    return dict(name=name, op=op, hq=hq, hkv=hkv, d=d, dtype=dtype, page=page, **more)


def _rotary(d, layout="half", rotated=0, theta=1e6, scaling="none", factor=1.0, low=1.0, high=4.0, original=8192,
            magnitude=1.0):
    return dict(layout=layout, rotated=rotated or d, theta=theta, scaling=scaling, factor=factor, low=low, high=high,
                original=original, magnitude=magnitude)


def listed():
    return [
        # The producer of one token of a short chat: launch and latency.
        _case("produce_step", "produce", (16, 8, 128), "bf16", 16, batch=1, tokens=1, ragged=False, shortest=301,
              longest=301, norm=True, fused=False, proj="f32", **_rotary(128)),
        # One token of each of 64 sessions, positions scaled by frequency bands,
        # Q, K and V slices of one 16-bit projection.
        _case("produce_batch", "produce", (32, 8, 128), "f16", 64, batch=64, tokens=1, ragged=False, shortest=512,
              longest=4096, norm=False, fused=True, proj="f16", **_rotary(128, theta=5e5, scaling="bands", factor=8.0)),
        # Prompts of a batch, 6000 tokens in all: interleaved pairs in half of
        # each head, bands with a magnitude, per-head norms.
        _case("produce_prompts", "produce", (8, 4, 256), "bf16", 32, batch=8, tokens=750, ragged=True, shortest=1500,
              longest=20000, norm=True, fused=False, proj="f32",
              **_rotary(256, "interleaved", 128, 1e4, "bands", 4.0, 1.0, 32.0, 8192, 0.1 * math.log(4.0) + 1.0)),
        # One decode step of a short chat over its pages.
        _case("attend_step", "attend", (16, 8, 128), "bf16", 16, batch=1, tokens=1, ragged=False, shortest=301,
              longest=301, window=0, softcap=0.0),
        # A serving batch: 64 sessions of mixed lengths, one new token each.
        _case("attend_batch", "attend", (16, 8, 128), "f16", 16, batch=64, tokens=1, ragged=False, shortest=512,
              longest=8192, window=0, softcap=0.0),
        # Four sessions with long contexts, one new token each.
        _case("attend_long", "attend", (32, 8, 128), "bf16", 64, batch=4, tokens=1, ragged=False, shortest=100001,
              longest=131072, window=0, softcap=0.0),
        # A chunk of each of 32 sessions after about 4096 cached tokens.
        _case("attend_chunks", "attend", (32, 8, 128), "bf16", 64, batch=32, tokens=128, ragged=False, shortest=4224,
              longest=4224, window=0, softcap=0.0),
        # A mixed batch on a sliding layer with a score softcap: some sessions
        # decode, others bring up to 200 tokens, one has nothing to do.
        _case("attend_mixed", "attend", (8, 4, 256), "bf16", 32, batch=24, tokens=200, ragged=True, shortest=203,
              longest=4096, window=1024, softcap=50.0),
        # Chunks over an FP32 cache.
        _case("attend_f32", "attend", (14, 2, 64), "f32", 16, batch=4, tokens=128, ragged=False, shortest=1000,
              longest=2048, window=0, softcap=0.0),
        # A whole prompt of 8192 tokens.
        _case("attend_prompt", "attend", (32, 8, 128), "bf16", 64, batch=1, tokens=8192, ragged=False, shortest=8192,
              longest=8192, window=0, softcap=0.0),
        # The partly filled last pages of 24 forked sessions, in 28 layers' K and V.
        _case("copy_fork", "copy", (16, 8, 128), "bf16", 16, planes=56, pages=256, moved=24),
        # Compaction of a large cache: 1024 pages of six layers move down.
        _case("copy_compact", "copy", (8, 4, 256), "bf16", 32, planes=12, pages=2100, moved=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("produce", "attend", "attend", "attend", "copy"))
    hq, hkv, d = heads = rng.choice(_MORE)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    page = rng.choice((16, 32, 64, 128))
    if op == "copy":
        plane = hkv * page * d * _ES[dtype]
        planes = 2 * _log(rng, 1, 32)
        moved = _log(rng, 1, max(2, min(2000, (700 << 20) // (plane * planes))))
        c = _case("", op, heads, dtype, page, planes=planes, pages=2 * moved + _log(rng, 1, 64), moved=moved)
    elif op == "produce":
        batch = _log(rng, 1, 64)
        tokens = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, 6000 // batch))
        longest = tokens + _log(rng, 1, min(30000, (1 << 29) // (hkv * d * _ES[dtype] * batch)))
        scaling = rng.choice(("none", "linear", "bands"))
        c = _case("", op, heads, dtype, page, batch=batch, tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7,
                  shortest=max(tokens, longest // rng.choice((1, 4, 16))), longest=longest, norm=rng.random() < 0.5,
                  fused=rng.random() < 0.5, proj=rng.choice(("f32", dtype)),
                  **_rotary(d, rng.choice(("half", "interleaved")), rng.choice((d, d // 2, d // 4)),
                            rng.choice((1e4, 5e5, 1e6)), scaling, 1.0 if scaling == "none" else rng.choice((2.0, 8.0)), 1.0,
                            rng.choice((4.0, 32.0)), rng.choice((4096, 8192)), rng.choice((1.0, 1.2))))
    else:
        batch = _log(rng, 1, 64)
        tokens = 1 if rng.random() < 0.45 else _log(rng, 2, 512)
        # At most 1 GiB of keys and values and 100 GFLOP, as the larger listed cases have.
        most = (1 << 30) // (2 * hkv * d * _ES[dtype] * batch)
        if tokens > 1:
            most = min(most, int(1e11) // (4 * d * hq * tokens * batch), (1 << 31) // (4 * hq * tokens * batch))
        most = max(tokens + 1, min(65536, most))
        longest = tokens + _log(rng, 1, most)
        c = _case("", op, heads, dtype, page, batch=batch, tokens=tokens, ragged=tokens > 1 and rng.random() < 0.7,
                  shortest=max(tokens, longest // rng.choice((1, 4, 16))), longest=longest,
                  window=rng.choice((0, 0, _log(rng, 16, 4096))), softcap=rng.choice((0.0, 0.0, 30.0, 50.0)))
    del c["name"]
    return c


# ---- inputs: N(0, 1) activations, as the path's own tests and benchmark draw them

def _lengths(case, seed):
    """Keys and new tokens of every session (host integers): the case's own
    lengths, in an order that the seed gives."""
    fixed, g = torch.Generator().manual_seed(0), torch.Generator().manual_seed(seed)
    b = case["batch"]
    keys = torch.randint(case["shortest"], case["longest"] + 1, (b,), generator=fixed)
    new = torch.full((b,), case["tokens"])
    if case["ragged"]:
        new = torch.randint(1, case["tokens"] + 1, (b,), generator=fixed)
        new[torch.rand(b, generator=fixed) < 0.25] = 1
        new[b // 2] = case["tokens"]
        if b > 3:
            new[1] = 0  # a session with nothing to do in this pass
    return keys[torch.randperm(b, generator=g)], new[torch.randperm(b, generator=g)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, d, hq, hkv, page = _DT[case["dtype"]], case["d"], case["hq"], case["hkv"], case["page"]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    s = dict(case=dict(case))
    if case["op"] == "copy":
        cpu = torch.Generator().manual_seed(seed)
        s["pool"] = torch.empty(case["planes"], case["pages"], hkv, page, d, dtype=dt, device="cuda")
        for plane in s["pool"]:
            plane.copy_(randn(case["pages"], hkv, page, d))
        order = torch.randperm(case["pages"], generator=cpu)
        s["src"], s["dst"] = order[:case["moved"]].clone(), order[case["moved"]:2 * case["moved"]].clone()
        s["src_dev"], s["dst_dev"] = s["src"].cuda(), s["dst"].cuda()
        return s
    keys, new = _lengths(case, seed)
    b, total = case["batch"], int(new.sum())
    used = (keys + page - 1) // page
    pages, columns = int(used.sum()) + 3, -(-case["longest"] // page)
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))
    table = torch.zeros(b, columns, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used.tolist()):
        table[i, :n] = perm[at:at + n]
        at += n
    s.update(total=total, page_table=table.cuda(), key_lens=keys.int().cuda(),
             query_start=torch.cat((torch.zeros(1, dtype=torch.int64), new.cumsum(0))).int().cuda())
    s["k_pages"], s["v_pages"] = (randn(pages, hkv, page, d, dtype=dt) for _ in range(2))
    if case["op"] == "produce":
        pt = _DT[case["proj"]]
        if case["fused"]:
            rows = randn(total, hq + 2 * hkv, d, dtype=pt)
            s["q_proj"], s["k_proj"], s["v_proj"] = rows[:, :hq], rows[:, hq:hq + hkv], rows[:, hq + hkv:]
        else:
            s["q_proj"], s["k_proj"], s["v_proj"] = (randn(total, h, d, dtype=pt) for h in (hq, hkv, hkv))
        s["q_norm"] = s["k_norm"] = None
        if case["norm"]:
            s["q_norm"], s["k_norm"] = 1.0 + 0.02 * randn(d), 1.0 + 0.02 * randn(d)
        s["q_out"] = torch.zeros(total, hq, d, dtype=dt, device="cuda")
    else:
        s["q"] = randn(total, hq, d, dtype=dt)
        s["context"] = torch.zeros(total, hq, d, dtype=dt, device="cuda")
    return s


# ---- the framework's calls

@functools.lru_cache(None)
def _context():
    from toklet_amd import ops

    return ops.Context(torch.cuda.current_device(), synchronous=False)


def _own(s):
    from toklet_amd import ops

    c, ctx = s["case"], _context()
    if c["op"] == "copy":
        ops.copy_pages(ctx, s["pool"], s["src"], s["dst"])
        return s["pool"]
    batch = ops.PagedBatch(page_table=s["page_table"], key_lens=s["key_lens"], query_start=s["query_start"],
                           total_queries=s["total"], max_queries=c["tokens"], max_keys=c["longest"])
    if c["op"] == "attend":
        ops.paged_attention(ctx, batch, s["q"], s["k_pages"], s["v_pages"], s["context"], scale=c["d"] ** -0.5,
                            window=c["window"] or None, softcap=c["softcap"])
        return s["context"]
    rotary = ops.RotaryPositions(layout=c["layout"], rotated_dims=c["rotated"], theta=c["theta"], scaling=c["scaling"],
                                 factor=c["factor"], low_freq_factor=c["low"], high_freq_factor=c["high"],
                                 original_max_positions=c["original"], magnitude=c["magnitude"])
    ops.paged_produce(ctx, batch, rotary, s["q_proj"], s["k_proj"], s["v_proj"], s["q_norm"], s["k_norm"], s["q_out"],
                      s["k_pages"], s["v_pages"])
    return s["q_out"], s["k_pages"], s["v_pages"]


# ---- the plain form

def _inverse_frequencies(c):
    """FP64 [rotated / 2]: theta^(-2j/rotated); divided by the factor (linear), or
    by wavelength band: kept where `high` or more rotations fit the original
    length, divided where `low` or fewer do, blended in between."""
    j = torch.arange(c["rotated"] // 2, dtype=torch.float64, device="cuda")
    f = c["theta"] ** (-2.0 * j / c["rotated"])
    if c["scaling"] == "linear":
        return f / c["factor"]
    if c["scaling"] == "bands":
        keep = ((c["original"] * f / (2.0 * math.pi) - c["low"]) / (c["high"] - c["low"])).clamp(0.0, 1.0)
        return f * (keep + (1.0 - keep) / c["factor"])
    return f


def _positions(s):
    """Session and position of every new token."""
    start = s["query_start"].long()
    t = torch.arange(s["total"], device="cuda")
    b = torch.searchsorted(start[1:], t, right=True)
    return b, s["key_lens"].long()[b] - start[b + 1] + t


def _plain_produce(s):
    c = s["case"]
    b, pos = _positions(s)
    angle = pos.double()[:, None] * _inverse_frequencies(c)
    cos, sin = ((f(angle) * c["magnitude"]).float()[:, None, :] for f in (torch.cos, torch.sin))

    def rotated(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
        r = c["rotated"]
        if c["layout"] == "half":
            a, e = x[..., :r // 2], x[..., r // 2:r]
            turned = torch.cat((a * cos - e * sin, e * cos + a * sin), -1)
        else:
            a, e = x[..., 0:r:2], x[..., 1:r:2]
            turned = torch.stack((a * cos - e * sin, e * cos + a * sin), -1).flatten(-2)
        return torch.cat((turned, x[..., r:]), -1)

    dt = s["q_out"].dtype
    page, at = s["page_table"].long()[b, pos // c["page"]], pos % c["page"]
    s["q_out"].copy_(rotated(s["q_proj"], s["q_norm"]))
    s["k_pages"][page, :, at] = rotated(s["k_proj"], s["k_norm"]).to(dt)
    s["v_pages"][page, :, at] = s["v_proj"].to(dt)
    return s["q_out"], s["k_pages"], s["v_pages"]


def _plain_attend(s):
    c = s["case"]
    nb, hkv, d, tokens = c["batch"], c["hkv"], c["d"], c["tokens"]
    group = c["hq"] // hkv
    start, lens = s["query_start"].long(), s["key_lens"].long()
    new = start[1:] - start[:-1]
    table = s["page_table"].long()
    keys = table.shape[1] * c["page"]
    # [batch, KV head, key, feature]
    k, v = (x[table].permute(0, 2, 1, 3, 4).reshape(nb, hkv, keys, d).float() for x in (s["k_pages"], s["v_pages"]))
    i = torch.arange(tokens, device="cuda")
    real = i < new[:, None]
    row = torch.where(real, start[:-1, None] + i, s["total"])
    q = torch.cat((s["q"], torch.zeros_like(s["q"][:1])))[row].float()
    q = q.view(nb, tokens, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(nb, hkv, group * tokens, d)
    pos = (lens - new)[:, None] + i
    key = torch.arange(keys, device="cuda")
    seen = (key <= pos[..., None]) & (key < lens[:, None, None]) & real[..., None]
    if c["window"]:
        seen &= pos[..., None] - key < c["window"]
    scores = (q @ k.transpose(2, 3).contiguous()).mul_(d ** -0.5)
    if c["softcap"]:
        scores = scores.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    scores = scores.view(nb, hkv, group, tokens, keys).masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    mass = p.sum(-1, keepdim=True)
    out = (p.view(nb, hkv, group * tokens, keys) @ v).view(nb, hkv, group, tokens, d)
    out = torch.where(mass > 0, out / mass, 0.0).permute(0, 3, 1, 2, 4).reshape(nb * tokens, c["hq"], d)
    whole = torch.zeros(s["total"] + 1, c["hq"], d, device="cuda").index_copy_(0, row.flatten(), out)
    s["context"].copy_(whole[:-1])
    return s["context"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "copy":
        state["pool"][:, state["dst_dev"]] = state["pool"][:, state["src_dev"]]
        return state["pool"]
    return _plain_attend(state) if op == "attend" else _plain_produce(state)


# ---- 64 bits, session by session

def _exact_produce(s, keys, new):
    c = s["case"]
    q_out, k_pages, v_pages = (s[n].double() for n in ("q_out", "k_pages", "v_pages"))
    r, page = c["rotated"], c["page"]
    freq = []
    for j in range(r // 2):
        f = c["theta"] ** (-2.0 * j / r)
        turns = c["original"] * f / (2.0 * math.pi)  # rotations over the original length
        if c["scaling"] == "linear" or (c["scaling"] == "bands" and turns <= c["low"]):
            f /= c["factor"]
        elif c["scaling"] == "bands" and turns < c["high"]:
            w = (turns - c["low"]) / (c["high"] - c["low"])
            f = (1.0 - w) * f / c["factor"] + w * f
        freq.append(f)
    freq = torch.tensor(freq, dtype=torch.float64, device="cuda")
    first = torch.arange(r // 2, device="cuda") * (1 if c["layout"] == "half" else 2)
    second = first + (r // 2 if c["layout"] == "half" else 1)
    at = 0
    for b, n in enumerate(new):
        pos = torch.arange(keys[b] - n, keys[b], device="cuda")
        turn = torch.polar(torch.full((n, 1, r // 2), c["magnitude"], dtype=torch.float64, device="cuda"),
                           (pos.double()[:, None] * freq)[:, None])
        rows = {}
        for name in ("q", "k"):
            x, w = s[name + "_proj"][at:at + n].double(), s[name + "_norm"]
            if w is not None:
                x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
            z = torch.complex(x[..., first], x[..., second]) * turn
            x = x.clone()
            x[..., first], x[..., second] = z.real, z.imag
            rows[name] = x
        where = s["page_table"][b].long()[pos // page]
        q_out[at:at + n] = rows["q"]
        k_pages[where, :, pos % page] = rows["k"]
        v_pages[where, :, pos % page] = s["v_proj"][at:at + n].double()
        at += n
    return q_out, k_pages, v_pages


def _exact_attend(s, keys, new):
    c = s["case"]
    group, page = c["hq"] // c["hkv"], c["page"]
    out = torch.zeros(s["total"], c["hq"], c["d"], dtype=torch.float64, device="cuda")
    at = 0
    for b, n in enumerate(new):
        if n == 0:
            continue
        length = keys[b]
        where = s["page_table"][b, :-(-length // page)].long()
        pos = torch.arange(length - n, length, device="cuda")[:, None]
        key = torch.arange(length, device="cuda")
        hidden = key > pos
        if c["window"]:
            hidden |= key <= pos - c["window"]
        for h in range(c["hkv"]):
            k, v = (x[where, h].reshape(-1, c["d"])[:length].double() for x in (s["k_pages"], s["v_pages"]))
            for j in range(h * group, (h + 1) * group):
                x = s["q"][at:at + n, j].double() @ k.t() / math.sqrt(c["d"])
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                out[at:at + n, j] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v
        at += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        pool = s["pool"].double()
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[:, b].copy_(s["pool"][:, a])
        return pool
    keys, new = (x.tolist() for x in _lengths(case, seed))
    return (_exact_attend if case["op"] == "attend" else _exact_produce)(s, keys, new)


# ---- what a pass cannot do without

def work(case):
    c, es = case, _ES[case["dtype"]]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    if c["op"] == "copy":
        return {"bytes": 2 * c["planes"] * c["moved"] * hkv * c["page"] * d * es, "flops": 0}
    keys, new = (x.tolist() for x in _lengths(case, 0))
    total = sum(new)
    entries = sum(-(-n // c["page"]) for n in keys) * 4
    if c["op"] == "produce":
        values = total * (hq + 2 * hkv) * d
        return {"bytes": values * (_ES[c["proj"]] + es) + total * 4, "flops": total * (hq + hkv) * (3 * c["rotated"] + 4 * d * c["norm"])}
    window = c["window"] or max(keys) + 1
    read = pairs = 0
    for n, t in zip(keys, new):
        if t:
            read += min(n, window + t - 1)
            full = max(0, min(t, window - 1 - (n - t)))  # rows that the window does not cut
            pairs += full * (n - t) + full * (full + 1) // 2 + (t - full) * window
    return {"bytes": 2 * read * hkv * d * es + 2 * total * hq * d * es + entries, "flops": 4 * pairs * hq * d}
