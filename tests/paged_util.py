"""Builders, 64-bit references and error bounds of the paged cache's tests."""

from __future__ import annotations

import math

import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # a rounding, relative to the value


class Paged:
    """Random pages, tables and queries.  `spans`: (keys, new tokens) per sequence.  Every
    row that no key occupies is NaN, and so is every page of no sequence; table entries past
    the last key name no page."""

    def __init__(self, spans, heads, dtype, page, seed=0, slots=False, token_major=False, spare=0, scale_v=1.0):
        self.spans, self.dtype, self.page = spans, dtype, page
        self.hq, self.hkv, self.d = heads
        g = torch.Generator().manual_seed(seed)
        dt = DT[dtype]
        b = len(spans)
        used = [-(-n // page) for n, _ in spans]
        self.pages = sum(used) + 3
        perm = torch.randperm(self.pages, generator=g).tolist()
        self.rows = list(range(b))
        total_rows = b
        if slots:
            total_rows = b + 2
            self.rows = torch.randperm(total_rows, generator=g)[:b].tolist()
        columns = max(used) + 1
        table = torch.full((total_rows, columns), 2 ** 31 - 1, dtype=torch.int32)
        lens = torch.full((total_rows,), -5, dtype=torch.int32)
        shape = (self.pages, page, self.hkv, self.d) if token_major else (self.pages, self.hkv, page, self.d)
        self.k_cpu, self.v_cpu = (torch.full(shape, math.nan, dtype=dt) for _ in range(2))
        if token_major:
            self.k_cpu, self.v_cpu = self.k_cpu.transpose(1, 2), self.v_cpu.transpose(1, 2)
        self.table_of = []
        for i, (n, _) in enumerate(spans):
            mine = [perm.pop() for _ in range(used[i])]
            self.table_of.append(mine)
            table[self.rows[i], :used[i]] = torch.tensor(mine, dtype=torch.int32)
            lens[self.rows[i]] = n
            k, v = (torch.randn(self.hkv, used[i] * page, self.d, generator=g).to(dt) for _ in range(2))
            v = (v.float() * scale_v).to(dt)
            k[:, n:], v[:, n:] = math.nan, math.nan
            for j, gpage in enumerate(mine):
                self.k_cpu[gpage] = k[:, j * page:(j + 1) * page]
                self.v_cpu[gpage] = v[:, j * page:(j + 1) * page]
        self.new = [t for _, t in spans]
        self.total = sum(self.new) + spare
        start = [0]
        for t in self.new:
            start.append(start[-1] + t)
        self.start = start
        self.q_cpu = torch.randn(self.total, self.hq, self.d, generator=g).to(dt)
        self.k, self.v, self.q = self._cuda(self.k_cpu), self._cuda(self.v_cpu), self.q_cpu.cuda()
        self.table, self.lens = table.cuda(), lens.cuda()
        self.query_start = torch.tensor(start, dtype=torch.int32).cuda()
        self.slots = torch.tensor(self.rows, dtype=torch.int32).cuda() if slots else None

    @staticmethod
    def _cuda(t):
        if t.is_contiguous():
            return t.cuda()
        return t.transpose(1, 2).contiguous().cuda().transpose(1, 2)

    def batch(self, **bounds):
        from toklet_amd import ops

        args = dict(page_table=self.table, key_lens=self.lens, total_queries=self.total,
                    max_queries=max(1, max(self.new)), max_keys=max(1, max(n for n, _ in self.spans)),
                    query_start=self.query_start, slots=self.slots)
        args.update(bounds)
        return ops.PagedBatch(**args)

    def sequence(self, i):
        """K and V of sequence i in FP64: [kv_heads, keys, head_dim]."""
        n = self.spans[i][0]
        out = []
        for pages in (self.k, self.v):
            x = pages[torch.tensor(self.table_of[i], dtype=torch.int64, device="cuda")] if n else pages[:0]
            out.append(x.permute(1, 0, 2, 3).reshape(self.hkv, -1, self.d)[:, :n].double())
        return out


def attention(p: Paged, scale, window=None, softcap=0.0):
    """The context in FP64 and, per element, how far a kernel may be off: with u = 2^-24,
    h the storage's half step, A = sum_j p_j |v_j| and n visible keys,
      h |o|                      the context's rounding,
      2 h A                      weights rounded to 16 bits (numerator and mass),
      2 ds A                     scores: D FP32 products and sums, (D + 4) u of their
                                 magnitudes, and FP32 tanh, 2^-21 of the cap,
      (2 n + 16) u A             FP32 sums over the keys, exponentials, the division,
      n 2^-25 max|v|             f16 weights below 2^-14 lose up to 2^-25 of the largest."""
    u, h = 2.0 ** -24, HALF_STEP[p.dtype]
    out = torch.zeros(p.total, p.hq, p.d, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    group = p.hq // p.hkv
    for i, (n, t) in enumerate(p.spans):
        if t == 0 or n == 0:
            continue
        k, v = p.sequence(i)
        pos = torch.arange(n - t, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = key <= pos
        if window:
            seen &= key > pos - window
        rows = slice(p.start[i], p.start[i] + t)
        for head in range(p.hq):
            kh, vh, q = k[head // group], v[head // group], p.q[rows, head].double()
            x = q @ kh.t() * scale
            size = (q.abs() @ kh.abs().t() * scale).masked_fill(~seen, 0.0)
            ds = (p.d + 4) * u * size
            if softcap:
                x = softcap * torch.tanh(x / softcap)
                ds = ds + softcap * 2.0 ** -21
            w = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
            w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
            o, a = w @ vh, w @ vh.abs()
            count = seen.sum(-1, keepdim=True).double()
            e = h * o.abs() + (2 * ds.amax(-1, keepdim=True) + (2 * count + 16) * u) * a
            if p.dtype != "f32":
                e = e + 2 * h * a
            if p.dtype == "f16":
                e = e + count * 2.0 ** -25 * vh.abs().amax()
            out[rows, head], tol[rows, head] = o, e
    return out, tol


def frequencies(r, theta, scaling="none", factor=1.0, low=1.0, high=4.0, original=8192):
    out = []
    for j in range(r // 2):
        f = theta ** (-2.0 * j / r)
        turns = original * f / (2 * math.pi)
        if scaling == "linear" or (scaling == "bands" and turns <= low):
            f /= factor
        elif scaling == "bands" and turns < high:
            w = (turns - low) / (high - low)
            f = (1 - w) * f / factor + w * f
        out.append(f)
    return torch.tensor(out, dtype=torch.float64)


def produce(x, pos, w, layout, r, freq, magnitude=1.0, eps=1e-6):
    """One projection's rows [tokens, heads, D] at positions `pos` in FP64, and the size of
    what each element is formed of."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    if layout == "none":
        return x, x.abs()
    freq = freq.to(x.device)
    a = pos.double()[:, None, None] * freq
    c, s = torch.cos(a) * magnitude, torch.sin(a) * magnitude
    first = torch.arange(r // 2, device=x.device) * (1 if layout == "half" else 2)
    second = first + (r // 2 if layout == "half" else 1)
    y, size = x.clone(), x.abs().clone()
    u, v = x[..., first], x[..., second]
    y[..., first], y[..., second] = u * c - v * s, v * c + u * s
    size[..., first] = size[..., second] = (u.abs() + v.abs()) * magnitude
    return y, size
