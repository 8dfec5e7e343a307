"""The paged cache's operators against plain 64-bit implementations: attention over page
tables, the producer that writes pages, page copies, and a run of them together."""

import math

import pytest

from gpu_util import log

pytestmark = pytest.mark.gpu

HEADS = {64: (14, 2, 64), 128: (16, 8, 128), 256: (8, 4, 256)}


@pytest.fixture(scope="module")
def ctx():
    from toklet_amd import ops

    return ops.Context(0)


def check(name, got, want, tol):
    import torch

    assert torch.isfinite(got).all(), name
    off = (got.double() - want).abs()
    worst = (off / tol.clamp_min(1e-300)).amax() if off.numel() else torch.tensor(0.0)
    log(f"{name}: largest error {off.max().item() if off.numel() else 0:.3e}, {worst.item():.3f} of its bound")
    assert (off <= tol).all(), f"{name}: {worst.item()} times the bound"


def attend(ctx, p, window=None, softcap=0.0, scale=None, **bounds):
    import torch

    from paged_util import attention
    from toklet_amd import ops

    scale = scale or p.d ** -0.5
    out = torch.full_like(p.q, 7.0)
    ops.paged_attention(ctx, p.batch(**bounds), p.q, p.k, p.v, out, scale=scale, window=window, softcap=softcap)
    want, tol = attention(p, scale, window, softcap)
    real = p.start[-1]
    assert (out[real:] == 7.0).all(), "rows behind the last sequence are left as they were"
    return out[:real], want[:real], tol[:real]


def span_sets():
    return {
        "one": [(1, 1)],
        "two": [(2, 1), (1, 1)],
        "page_ends": [(15, 1), (16, 1), (17, 1), (31, 2), (32, 3), (33, 4), (64, 1)],
        "decode": [(301, 1), (1, 1), (77, 1), (1000, 1), (4096, 1)],
        "short_chunks": [(5, 5), (40, 3), (100, 2), (333, 8), (17, 4)],
        "chunks": [(130, 130), (257, 64), (300, 33), (64, 16), (1025, 127)],
        "mixed": [(513, 1), (200, 200), (0, 0), (90, 1), (1500, 37), (65, 0), (33, 33)],
        "long_prompt": [(700, 700)],
    }


@pytest.mark.parametrize("spans", list(span_sets()))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_lengths(ctx, dtype, d, spans):
    from paged_util import Paged

    p = Paged(span_sets()[spans], HEADS[d], dtype, page=16, seed=d)
    log(f"lengths {spans} {dtype} {d}")
    check(f"{spans} {dtype} {d}", *attend(ctx, p))


@pytest.mark.parametrize("heads", [(1, 1, 64), (12, 12, 64), (8, 1, 128), (16, 1, 128), (20, 4, 128), (24, 2, 64),
                                   (32, 1, 64), (3, 1, 256), (40, 2, 256)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_head_layouts(ctx, dtype, heads):
    from paged_util import Paged

    for name, spans in (("decode", [(200, 1), (33, 1)]), ("chunk", [(150, 70), (40, 40), (260, 5)])):
        p = Paged(spans, heads, dtype, page=32, seed=3)
        log(f"heads {heads} {dtype} {name}")
        check(f"{heads} {dtype} {name}", *attend(ctx, p))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("token_major", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_pages(ctx, dtype, token_major, page):
    """Page sizes, page layouts, slots in any order, padded rows behind the batch."""
    from paged_util import Paged

    for name, spans in (("decode", [(700, 1), (1500, 1), (3, 1)]), ("chunk", [(700, 90), (1100, 40), (9, 9)])):
        p = Paged(spans, HEADS[128], dtype, page=page, seed=page, slots=True, token_major=token_major, spare=5)
        log(f"pages {page} {token_major} {dtype} {name}")
        check(f"{page} {token_major} {dtype} {name}", *attend(ctx, p, max_queries=96))


@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (17, 50.0), (100, 30.0), (1000, 0.0), (None, 5.0)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_masks(ctx, dtype, d, window, softcap):
    """Windows that start inside a page, and capped scores; the keys before every row's
    window hold NaN, as freed pages may."""
    from paged_util import Paged

    for name, spans in (("decode", [(300, 1), (5, 1), (1290, 1)]), ("chunk", [(300, 60), (5, 5), (1290, 130)])):
        p = Paged(spans, HEADS[d], dtype, page=16, seed=5)
        want = attend_with_freed_pages(p, window)
        log(f"mask {window} {softcap} {dtype} {d} {name}")
        got, ref, tol = attend(ctx, p, window, softcap, scale=0.25 if softcap else None)
        assert want
        check(f"{window} {softcap} {dtype} {d} {name}", got, ref, tol)


def attend_with_freed_pages(p, window):
    """NaN into every key that no new token's window reaches."""
    if window:
        for i, (n, t) in enumerate(p.spans):
            for j in range(max(0, n - t - window + 1)):
                page, row = p.table_of[i][j // p.page], j % p.page
                p.k[page, :, row], p.v[page, :, row] = math.nan, math.nan
    # The reference reads them as weights of zero: give it zeros there.
    original = p.sequence

    def sequence(i):
        k, v = original(i)
        return k.nan_to_num(0.0), v.nan_to_num(0.0)

    p.sequence = sequence
    return True


def test_attention_rows_without_keys(ctx):
    """More new tokens than keys: the first rows have positions below 0 and see nothing."""
    import torch

    from paged_util import Paged, attention
    from toklet_amd import ops

    for dtype in ("bf16", "f32"):
        p = Paged([(40, 40), (0, 0), (130, 64)], HEADS[128], dtype, page=16, seed=9)
        want, tol = attention(p, 0.1)
        # Ten keys fewer in sequence 0 for the same rows: rows 0..9 see nothing.
        p.lens[0] = 30
        p.spans[0] = (30, 30)
        short, short_tol = attention_shifted(p, 10)
        out = torch.full_like(p.q, 7.0)
        ops.paged_attention(ctx, p.batch(), p.q, p.k, p.v, out, scale=0.1)
        assert (out[:10] == 0).all()
        check(f"rows without keys {dtype}", out[10:40], short, short_tol)
        check(f"other sequences {dtype}", out[40:], want[40:], tol[40:])


def attention_shifted(p, skip):
    import copy

    from paged_util import attention

    r = copy.copy(p)
    r.spans, r.total, r.start = [p.spans[0]], p.spans[0][1], [0, p.spans[0][1]]
    r.q = p.q[skip:skip + r.total]
    r.table_of = [p.table_of[0][:-(-p.spans[0][0] // p.page)]]
    want, tol = attention(r, 0.1)
    return want, tol


def tuned(monkeypatch, stream=None, synchronous=True, **env):
    """A context whose launches split as the settings say."""
    from toklet_amd import ops

    for name, value in env.items():
        monkeypatch.setenv("TKH_PAGED_" + name, str(value))
    ctx = ops.Context(0, stream=stream, synchronous=synchronous)
    for name in env:
        monkeypatch.delenv("TKH_PAGED_" + name)
    return ctx


FINEST = dict(DECODE_BLOCKS=1, DECODE_GROUPS=4096, CHUNK_TILES=1, CHUNK_GROUPS=4096)


@pytest.mark.parametrize("window,softcap", [(None, 0.0), (500, 20.0)])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_many_splits(monkeypatch, dtype, d, window, softcap):
    """As many splits as there are key blocks, of which the last to arrive joins all in one
    order: equal results from call to call, and counters left as they were."""
    import torch

    from paged_util import Paged

    ctx = tuned(monkeypatch, **FINEST)
    for name, spans in (("decode", [(3000, 1), (129, 1), (1, 1), (0, 0), (2000, 1)]),
                        ("chunk", [(2100, 70), (300, 33), (64, 64), (1500, 1), (20, 20)])):
        p = Paged(spans, HEADS[d], dtype, page=16, seed=d + 1)
        log(f"splits {name} {dtype} {d}")
        got, want, tol = attend(ctx, p, window, softcap)
        check(f"{name} {dtype} {d}", got, want, tol)
        for _ in range(3):
            assert torch.equal(attend(ctx, p, window, softcap)[0], got)
    ctx.close()


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("window,softcap", [(None, 0.0), (100, 0.0), (33, 30.0)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attention_wide_rows(monkeypatch, dtype, d, window, softcap, split):
    """Workgroups of 256 rows, which large batches have, at sizes that end inside them."""
    from paged_util import Paged

    ctx = tuned(monkeypatch, WIDE_GROUPS=1, **(FINEST if split else {}))
    for spans in ([(900, 300), (64, 64), (257, 257), (700, 5), (90, 1)], [(128, 128), (0, 0), (1060, 65)]):
        p = Paged(spans, (8, 2, d), dtype, page=32, seed=d)
        want = attend_with_freed_pages(p, window)
        log(f"wide {dtype} {d} {window} {split}")
        got, ref, tol = attend(ctx, p, window, softcap)
        assert want
        check(f"wide {dtype} {d} {window} {split}", got, ref, tol)
    ctx.close()


@pytest.mark.parametrize("sequences", [63, 64, 65, 130, 1030, 2100])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_many_sequences(ctx, dtype, sequences):
    """More sequences than a wave has lanes, than one launch lists; short ones among long ones."""
    from paged_util import Paged

    spans = [(i % 37, min(i % 37, i % 4)) for i in range(sequences)]
    spans[sequences // 2], spans[-1], spans[3] = (3000, 1), (700, 40), (1500, 33)
    p = Paged(spans, (4, 2, 64), dtype, page=16, seed=sequences, slots=sequences % 2 == 0)
    log(f"sequences {sequences} {dtype}")
    check(f"{sequences} {dtype}", *attend(ctx, p))


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("heads", [(8, 4, 256), (12, 3, 128), (7, 7, 64), (16, 8, 128), (9, 1, 128)])
def test_attention_chunks_of_many(monkeypatch, heads, split):
    """Chunks of many sequences, some of them none and some single tokens: every row block of
    every head is worked on once, however the list is dealt out."""
    from paged_util import Paged

    ctx = tuned(monkeypatch, **(FINEST if split else {}))
    for count in (9, 33, 61):
        spans = [(40 + 23 * i % 300, (0, 1, 17, 40, 3)[i % 5] if i % 7 else 40) for i in range(count)]
        p = Paged(spans, heads, "bf16", page=16, seed=count)
        log(f"many chunks {heads} {split} {count}")
        check(f"many chunks {heads} {split} {count}", *attend(ctx, p))
    ctx.close()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_far_pages(ctx, dtype):
    """Pages further apart than 32 bits of bytes, and of elements, reach."""
    import torch

    from paged_util import Paged

    for spans in ([(90, 1), (60, 1)], [(90, 40), (60, 60)]):
        p = Paged(spans, HEADS[64], dtype, page=16, seed=8)
        apart = 1 << 29  # elements; 13 pages
        store = torch.empty(2 * (p.pages - 1) * apart + 2 * 16 * 64 * 2, dtype=p.k.dtype, device="cuda")
        k, v = (torch.as_strided(store, p.k.shape, (2 * apart, 16 * 64, 64, 1), i * 16 * 64 * 2) for i in range(2))
        k.copy_(p.k)
        v.copy_(p.v)
        p.k, p.v = k, v
        assert (p.pages - 1) * 2 * apart > 1 << 32
        log(f"far {dtype} {spans}")
        check(f"far {dtype}", *attend(ctx, p))
        del k, v, store, p


def test_attention_two_streams(monkeypatch):
    """Two contexts on streams of their own, at work at the same time, give what each gives alone."""
    import torch

    from paged_util import Paged
    from toklet_amd import ops

    work = []
    for i in range(2):
        ctx = tuned(monkeypatch, stream=torch.cuda.Stream(), **FINEST)
        p = Paged([(2500 - 900 * i, 1), (900, 40 + i), (33, 33)], HEADS[128], "bf16", page=16, seed=i)
        torch.cuda.synchronize()
        alone, out = torch.empty_like(p.q), torch.empty_like(p.q)
        ops.paged_attention(ctx, p.batch(), p.q, p.k, p.v, alone, scale=0.1)
        ctx.close()
        work.append((tuned(monkeypatch, stream=torch.cuda.Stream(), synchronous=False, **FINEST), p, p.batch(), alone, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, p, batch, _, out in work:
            ops.paged_attention(ctx, batch, p.q, p.k, p.v, out, scale=0.1)
    for ctx, _, _, alone, out in work:
        ctx.synchronize()
        assert torch.equal(out, alone)
        ctx.close()


def test_attention_large_scores(ctx):
    """Scores of hundreds, one key far above the others, and equal scores."""
    import torch

    from paged_util import Paged

    for dtype in ("bf16", "f16", "f32"):
        for spans in ([(400, 1), (70, 1)], [(400, 100), (90, 90)]):
            p = Paged(spans, HEADS[128], dtype, page=16, seed=11)
            check(f"large {dtype} {len(spans)}", *attend(ctx, p, scale=4.0))
            hot = p.table_of[0][7]
            p.k[hot, :, 3] = (p.k[hot, :, 3].float() * 8).to(p.k.dtype)
            check(f"peaky {dtype}", *attend(ctx, p))
            p.k.copy_(torch.where(p.k.isnan(), p.k, torch.zeros_like(p.k)))
            check(f"equal {dtype}", *attend(ctx, p))


def test_attention_uniform_rows(ctx):
    """query_start None: max_queries rows each; a broadcast-free strided table."""
    import torch

    from paged_util import Paged, attention
    from toklet_amd import ops

    p = Paged([(50, 3), (90, 3), (3, 3)], HEADS[128], "bf16", page=16, seed=2)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, :p.table.shape[1]] = p.table
    out = torch.empty_like(p.q)
    ops.paged_attention(ctx, p.batch(query_start=None, page_table=wide[:, :10], max_keys=160), p.q, p.k, p.v, out, scale=0.1)
    want, tol = attention(p, 0.1)
    check("uniform", out, want, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_nonfinite(ctx, dtype):
    """A visible NaN or infinity is reported; the context keeps no trace for the next call."""
    import torch

    from paged_util import Paged
    from toklet_amd import _lib, ops

    for spans in ([(100, 1), (50, 1)], [(100, 60), (50, 30)]):
        for where in ("k", "v", "q"):
            for value in (math.nan, math.inf, -math.inf):
                p = Paged(spans, HEADS[128], dtype, page=16, seed=4)
                if where == "q":
                    p.q[0, 3, 5] = value
                else:
                    getattr(p, where)[p.table_of[0][1], 2, 3, 9] = value
                out = torch.empty_like(p.q)
                log(f"nonfinite {dtype} {where} {value}")
                with pytest.raises(ops.TkhError) as e:
                    ops.paged_attention(ctx, p.batch(), p.q, p.k, p.v, out, scale=0.1)
                assert e.value.code == _lib.NON_FINITE
        p = Paged(spans, HEADS[128], dtype, page=16, seed=4)
        check(f"after {dtype}", *attend(ctx, p))


def test_bad_metadata(ctx):
    """Slots, row ranges, lengths and page numbers out of range: reported, nothing touched outside."""
    import torch

    from paged_util import Paged
    from toklet_amd import _lib, ops

    def broken(spans):
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "page", p, lambda: p.table[p.rows[0]].fill_(p.pages)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "negative page", p, lambda: p.table[p.rows[1]].fill_(-1)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "slot", p, lambda: p.slots[1:2].fill_(99)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "negative slot", p, lambda: p.slots[0:1].fill_(-1)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "length", p, lambda: p.lens[p.rows[0]:p.rows[0] + 1].fill_(10 ** 6)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "negative length", p, lambda: p.lens[p.rows[0]:p.rows[0] + 1].fill_(-1)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "rows", p, lambda: p.query_start[2:].fill_(10 ** 6)
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6, slots=True)
        yield "decreasing rows", p, lambda: p.query_start[1:2].fill_(-3)

    for spans in ([(40, 1), (100, 1)], [(80, 50), (100, 30)]):
        for name, p, breaks in broken(spans):
            breaks()
            out = torch.empty_like(p.q)
            log(f"bad {name} {spans}")
            with pytest.raises(ops.TkhError) as e:
                ops.paged_attention(ctx, p.batch(), p.q, p.k, p.v, out, scale=0.1)
            assert e.value.code == _lib.INVALID_CONFIG, name
            x = torch.randn(p.total, 32, 128, device="cuda")
            before = p.k.clone(), p.v.clone()
            with pytest.raises(ops.TkhError) as e:
                ops.paged_produce(ctx, p.batch(), ops.RotaryPositions(), x[:, :16], x[:, 16:24], x[:, 24:], None, None, out,
                                  p.k, p.v)
            assert e.value.code == _lib.INVALID_CONFIG, name
            if name in ("slot", "negative slot", "length", "negative length"):
                kept = set(range(p.pages)) - set(p.table_of[0]) - set(p.table_of[1])
                for a, b in zip(before, (p.k, p.v)):
                    for g in kept:
                        assert torch.equal(a[g].nan_to_num(3.0), b[g].nan_to_num(3.0))
        p = Paged(spans, HEADS[128], "bf16", page=16, seed=6)
        check("after", *attend(ctx, p))


# ---- the producer

def produced(ctx, p, rot, norm, fused, proj, eps=1e-6):
    import torch

    from paged_util import DT, frequencies, produce
    from toklet_amd import ops

    g = torch.Generator().manual_seed(1)
    pt = DT[proj]
    n = p.hq + 2 * p.hkv
    rows = torch.randn(p.total, n, p.d, generator=g).to(pt).cuda()
    xs = [rows[:, :p.hq], rows[:, p.hq:p.hq + p.hkv], rows[:, p.hq + p.hkv:]]
    if not fused:
        xs = [x.contiguous() for x in xs]
    wq, wk = (1 + 0.1 * torch.randn(2, p.d, generator=g)).cuda() if norm else (None, None)
    q = torch.full_like(p.q, 7.0)
    k0, v0 = p.k.clone(), p.v.clone()
    ops.paged_produce(ctx, p.batch(), rot, *xs, wq, wk, q, p.k, p.v, eps)
    r = rot.rotated_dims or p.d
    freq = frequencies(r, rot.theta, rot.scaling, rot.factor, rot.low_freq_factor, rot.high_freq_factor,
                       rot.original_max_positions)
    from paged_util import HALF_STEP

    # One rounding of the result, FP32 arithmetic of a few steps on what forms it (2^-21).
    def near(name, got, want, size):
        check(name, got, want, HALF_STEP[p.dtype] * want.abs() + 2.0 ** -21 * size + 2.0 ** -25)

    real = p.start[-1]
    assert (q[real:] == 7.0).all()
    for i, (n, t) in enumerate(p.spans):
        if not t:
            continue
        at = slice(p.start[i], p.start[i] + t)
        pos = torch.arange(n - t, n, device="cuda")
        want, size = produce(xs[0][at], pos, wq, rot.layout, r, freq, rot.magnitude, eps)
        near(f"q {i}", q[at], want, size)
        want, size = produce(xs[1][at], pos, wk, rot.layout, r, freq, rot.magnitude, eps)
        page = torch.tensor(p.table_of[i], device="cuda")[pos // p.page]
        near(f"k {i}", p.k[page, :, pos % p.page], want, size)
        assert torch.equal(p.v[page, :, pos % p.page], xs[2][at].to(p.v.dtype)), f"v {i}"
        k0[page, :, pos % p.page] = p.k[page, :, pos % p.page]
        v0[page, :, pos % p.page] = p.v[page, :, pos % p.page]
    # Nothing else was written.
    assert torch.equal(k0.nan_to_num(3.0), p.k.nan_to_num(3.0)) and torch.equal(v0.nan_to_num(3.0), p.v.nan_to_num(3.0))


@pytest.mark.parametrize("layout,scaling", [("none", "none"), ("half", "none"), ("half", "linear"), ("half", "bands"),
                                            ("interleaved", "none"), ("interleaved", "linear"), ("interleaved", "bands")])
@pytest.mark.parametrize("dtype,proj", [("bf16", "f32"), ("f16", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16")])
def test_produce(ctx, layout, scaling, dtype, proj):
    from paged_util import Paged
    from toklet_amd import ops

    for d, r in ((64, 0), (64, 8), (128, 0), (128, 64), (128, 120), (256, 0), (256, 40)):
        p = Paged([(1, 1), (0, 0), (49, 33), (2000, 1), (17, 16)], HEADS[d], dtype, page=16, seed=d + r, slots=r == 64,
                  token_major=r == 8, spare=2)
        rot = ops.RotaryPositions(layout=layout, rotated_dims=r, theta=1e4 if r else 1e6, scaling=scaling, factor=8.0,
                                  low_freq_factor=1.0, high_freq_factor=32.0, original_max_positions=512,
                                  magnitude=1.25 if r == 40 else 1.0)
        log(f"produce {layout} {scaling} {dtype} {proj} {d} {r}")
        produced(ctx, p, rot, norm=r != 0, fused=d != 256, proj=proj)


def test_produce_far_positions(ctx):
    """Angles at positions near 2^20 keep their precision."""
    import torch

    from paged_util import Paged
    from toklet_amd import ops

    p = Paged([(16, 16), (40, 5)], HEADS[128], "f32", page=1024, seed=1)
    # The same pages again and again before the last one, as the table may say.
    far = 1 << 20
    columns = far // 1024
    table = p.table[:, :1].expand(2, columns).contiguous()
    p.table, p.lens = table, torch.tensor([far, far - 1000], dtype=torch.int32, device="cuda")
    rows = torch.randn(p.total, 32, 128, device="cuda")
    q = torch.empty_like(p.q)
    from paged_util import frequencies, produce

    rot = ops.RotaryPositions(theta=1e4)
    ops.paged_produce(ctx, p.batch(max_keys=far), rot, rows[:, :16], rows[:, 16:24], rows[:, 24:], None, None, q, p.k, p.v)
    for i, (n, t) in enumerate(((far, 16), (far - 1000, 5))):
        at = slice(p.start[i], p.start[i] + t)
        want, size = produce(rows[at, :16], torch.arange(n - t, n, device="cuda"), None, "half", 128, frequencies(128, 1e4))
        check(f"far {n}", q[at], want, 2.0 ** -24 * want.abs() + 2.0 ** -21 * size)


def test_produce_nonfinite(ctx):
    import torch

    from paged_util import Paged
    from toklet_amd import _lib, ops

    for at in ((0, 2, 5), (1, 17, 100), (2, 31, 0)):
        p = Paged([(20, 3)], HEADS[128], "bf16", page=16)
        rows = torch.randn(3, 32, 128, device="cuda")
        rows[at] = math.inf
        with pytest.raises(ops.TkhError) as e:
            ops.paged_produce(ctx, p.batch(), ops.RotaryPositions(), rows[:, :16], rows[:, 16:24], rows[:, 24:], None, None,
                              torch.empty_like(p.q), p.k, p.v)
        assert e.value.code == _lib.NON_FINITE


# ---- page copies

@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 16, 64), (4, 9, 2, 16, 64), (3, 700, 1, 16, 64), (12, 40, 4, 32, 256), (2, 5, 3, 7, 9)])
def test_copy_pages(ctx, dtype, shape):
    import torch

    from paged_util import DT
    from toklet_amd import ops

    g = torch.Generator().manual_seed(shape[1])
    pool = torch.randn(shape, generator=g).to(DT[dtype]).cuda()
    n = shape[1]
    lists = [([], []), ([0], [n - 1]), (list(range(n // 2)), list(range(n - n // 2, n)))]
    # Chains, repeated pages, copies onto themselves and back: one after the other.
    order = torch.randint(0, n, (2, 1500), generator=g).tolist()
    lists += [tuple(order), (list(range(n - 1)), list(range(1, n))), (list(range(1, n)), list(range(n - 1)))]
    for src, dst in lists:
        want = pool.clone()
        for a, b in zip(src, dst):
            want[:, b] = want[:, a].clone()
        log(f"copy {dtype} {shape} {len(src)}")
        ops.copy_pages(ctx, pool, src, dst)
        assert torch.equal(pool, want)
    # Planes and pages of other strides.
    wide = torch.randn(shape[0] * 2, n, *shape[2:], generator=g).to(DT[dtype]).cuda()
    view, keep = wide[::2], wide[1::2].clone()
    want = view.clone()
    want[:, n - 1] = want[:, 0]
    ops.copy_pages(ctx, view, torch.tensor([0]), torch.tensor([n - 1]))
    assert torch.equal(wide[::2], want) and torch.equal(wide[1::2], keep)
    turned = torch.randn(n, shape[0], *shape[2:], generator=g).to(DT[dtype]).cuda().transpose(0, 1)
    want = turned.clone()
    want[:, 0] = want[:, n // 2].clone()
    ops.copy_pages(ctx, turned, [n // 2], [0])
    assert torch.equal(turned, want)


# ---- together

def test_sessions_together():
    """Prompts, forks, decode steps, compaction and truncation of sessions on one owner, two layers,
    against full attention over each session's own rows."""
    import torch

    from paged_util import HALF_STEP, frequencies, produce
    from toklet_amd import ops, paged

    ctx = ops.Context(0, synchronous=False)
    hq, hkv, d, layers = 8, 2, 64, 2
    kv = paged.PagedKv(ctx, layers, hkv, d, page_tokens=16, pages=40, sequences=6, sequence_pages=12, storage=torch.bfloat16)
    rot = ops.RotaryPositions(layout="interleaved", theta=1e4)
    freq = frequencies(d, 1e4)
    g = torch.Generator(device="cuda").manual_seed(0)
    rows = {}  # (sequence, layer) -> projected K and V rows so far

    def step(seqs, new):
        kv.extend(seqs, new)
        b = kv.batch(seqs, new)
        total = sum(new)
        for layer in range(layers):
            x = torch.randn(total, hq + 2 * hkv, d, generator=g, device="cuda")
            q, out = (torch.empty(total, hq, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv.append(layer, b, rot, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q)
            kv.attend(layer, b, q, out, scale=d ** -0.5)
            ctx.synchronize()
            at = 0
            for s, n in zip(seqs, new):
                k_old, v_old = rows.get((s, layer), (x[:0, :hkv].double(), x[:0, :hkv].double()))
                have = k_old.shape[0]
                pos = torch.arange(have, have + n, device="cuda")
                k_new = produce(x[at:at + n, hq:hq + hkv], pos, None, "interleaved", d, freq)[0].bfloat16().double()
                k_all = torch.cat((k_old, k_new))
                v_all = torch.cat((v_old, x[at:at + n, hq + hkv:].bfloat16().double()))
                rows[s, layer] = (k_all, v_all)
                for h in range(hq):
                    kh, vh = k_all[:, h * hkv // hq], v_all[:, h * hkv // hq]
                    sc = q[at:at + n, h].double() @ kh.t() * d ** -0.5
                    sc = sc.masked_fill(torch.arange(have + n, device="cuda") > pos[:, None], -math.inf)
                    w = torch.softmax(sc, -1)
                    # A K element that rounds the other way (FP32 against FP64 rotation) moves a
                    # score by at most a step of one product: its probability by the same share.
                    ds = (q[at:at + n, h].double().abs() @ kh.abs().t()).amax() * d ** -0.5 * 2 * HALF_STEP["bf16"] * 2.0 ** -5
                    tol = 4 * HALF_STEP["bf16"] * (w @ vh.abs()) + 2 * ds * (w @ vh.abs())
                    off = (out[at:at + n, h].double() - w @ vh).abs()
                    assert (off <= tol).all(), (s, layer, h, (off / tol).max().item())
                at += n

    a, b = kv.open(), kv.open()
    step([a, b], [37, 50])
    step([b, a], [1, 1])
    c = kv.fork(a)
    for layer in range(layers):
        rows[c, layer] = rows[a, layer]
    step([a, c, b], [1, 3, 1])
    e = kv.fork(b)
    for layer in range(layers):
        rows[e, layer] = rows[b, layer]
    kv.close_sequence(a)
    for layer in range(layers):
        del rows[a, layer]
    assert kv.compact() >= 0
    used = [p for s in (b, c, e) for p in kv.pages(s)]
    assert max(used) < len(set(used))
    step([c, b, e], [20, 1, 1])
    kv.truncate(e, 33)
    for layer in range(layers):
        rows[e, layer] = tuple(x[:33] for x in rows[e, layer])
    step([e, b], [70, 2])
    a = kv.open()
    step([a, e], [5, 1])
    assert kv.key_lens[torch.tensor([a, b, c, e], device="cuda")].tolist() == [kv.length(s) for s in (a, b, c, e)]
    for s in (a, b, c, e):
        kv.close_sequence(s)
    assert kv.free_pages == 40
    kv.close()


def test_captured_steps():
    """A captured decode step replayed while its sessions grow, eager work of the same context in between."""
    import torch

    from toklet_amd import ops, paged

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = ops.Context(0, stream=stream, synchronous=False)
        hq, hkv, d = 16, 8, 128
        kv = paged.PagedKv(ctx, 1, hkv, d, page_tokens=16, pages=300, sequences=4, sequence_pages=70, storage=torch.bfloat16)
        kv.pool.copy_(torch.randn_like(kv.pool, dtype=torch.float32))
        seqs = [kv.open() for _ in range(3)]
        kv.extend(seqs, [1000, 30, 333])
        b = kv.batch(seqs, [1, 1, 1], max_keys=70 * 16)
        x = torch.randn(3, hq + 2 * hkv, d, device="cuda")
        q, out, eager = (torch.empty(3, hq, d, dtype=torch.bfloat16, device="cuda") for _ in range(3))
        rot = ops.RotaryPositions()

        def step(to):
            kv.append(0, b, rot, x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:], q)
            kv.attend(0, b, q, to, scale=d ** -0.5)

        step(out)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            with pytest.raises(ops.TkhError):
                kv.extend(seqs, [1, 1, 1])
            with pytest.raises(ops.TkhError):  # its clearing would be recorded
                paged.PagedKv(ctx, 1, hkv, d, 16, 8, 2, 4, torch.bfloat16)
            step(out)
        for i in range(6):
            kv.extend(seqs, [1, 1, 17 if i == 2 else 1])
            x.copy_(torch.randn_like(x))
            graph.replay()
            step(eager)
            ctx.synchronize()
            assert torch.equal(out, eager), i
    kv.close()
    ctx.close()


def test_captured_chunks(monkeypatch):
    """A captured pass of chunks and single tokens with split keys, replayed with eager passes in between."""
    import torch

    from paged_util import Paged
    from toklet_amd import ops

    stream = torch.cuda.Stream()
    ctx = tuned(monkeypatch, stream=stream, synchronous=False, **FINEST)
    p = Paged([(1400, 40), (700, 1), (0, 0), (200, 200)], HEADS[128], "bf16", page=16, seed=3)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        out, eager = torch.empty_like(p.q), torch.empty_like(p.q)
        batch = p.batch()

        def step(to):
            ops.paged_attention(ctx, batch, p.q, p.k, p.v, to, scale=0.1)

        step(eager)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(out)
        for i in range(6):
            p.q.copy_(torch.randn_like(p.q))
            if i == 3:  # lengths that the replay reads anew
                p.lens[p.rows[0]] = 1300
            out.fill_(0.0)
            graph.replay()
            step(eager)
            ctx.synchronize()
            assert torch.equal(out, eager), i
    ctx.close()
