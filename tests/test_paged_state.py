"""The paged cache's bookkeeping and the operators' refusals, without a GPU."""

import ctypes
import os
import random
import subprocess
import tempfile

import pytest
import torch

from toklet_amd import _lib, ops, paged

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def owner(pages=20, sequences=4, sequence_pages=8, page=16):
    return paged.PagedKv(None, 2, 2, 64, page, pages, sequences, sequence_pages, torch.bfloat16)


def code(f, *args):
    with pytest.raises(ops.TkhError) as e:
        f(*args)
    return e.value.code


def test_extend_truncate_close():
    kv = owner()
    a = kv.open()
    assert a == 0 and kv.length(a) == 0 and kv.pages(a) == []
    kv.extend([a], [1])
    assert kv.pages(a) == [0]
    kv.extend([a], [15])
    assert kv.pages(a) == [0] and kv.length(a) == 16
    b = kv.open()
    kv.extend([b, a], [33, 1])
    assert kv.pages(b) == [1, 2, 3] and kv.pages(a) == [0, 4] and kv.free_pages == 15
    kv.truncate(b, 16)
    assert kv.pages(b) == [1] and kv.free_pages == 17
    kv.extend([a], [0])
    kv.extend([a], [31])
    assert kv.pages(a) == [0, 4, 2]
    kv.close_sequence(a)
    assert kv.free_pages == 19 and kv.open() == 0
    with pytest.raises(ValueError):
        kv.length(3)


def test_refusals_leave_everything():
    kv = owner(pages=6)
    a, b = kv.open(), kv.open()
    kv.extend([a, b], [20, 20])
    before = kv.pages(a), kv.pages(b), kv.free_pages
    assert code(kv.extend, [a, b], [30, 30]) == _lib.CAPACITY
    assert code(kv.extend, [a], [16 * 8]) == _lib.CAPACITY
    assert code(kv.extend, [a, a], [1, 1]) == _lib.INVALID_PARAMETER
    assert code(kv.extend, [a, 3], [1, 1]) == _lib.INVALID_CONFIG
    assert code(kv.extend, [a, 77], [1, 1]) == _lib.INVALID_CONFIG
    assert code(kv.extend, [a, -1], [1, 1]) == _lib.INVALID_CONFIG
    assert code(kv.truncate, a, 21) == _lib.INVALID_PARAMETER
    assert code(kv.truncate, 2, 0) == _lib.INVALID_CONFIG
    assert code(kv.close_sequence, 2) == _lib.INVALID_CONFIG
    assert code(kv.fork, 2) == _lib.INVALID_CONFIG
    assert (kv.pages(a), kv.pages(b), kv.free_pages) == before
    kv.open(), kv.open()
    assert code(kv.open) == _lib.CAPACITY and code(kv.fork, a) == _lib.CAPACITY
    kv.extend([a, b], [12, 12])  # in their own pages
    assert kv.free_pages == 2


def test_fork_copies_the_shared_tail_on_write():
    kv = owner(sequences=5)
    a = kv.open()
    kv.extend([a], [40])  # pages 0, 1, 2; the last holds 8 keys
    b, c = kv.fork(a), kv.fork(a)
    assert kv.pages(b) == kv.pages(c) == [0, 1, 2] and kv.free_pages == 17
    # b and c write: both copy; then a holds its tail alone.
    kv.extend([b, c], [1, 1])
    assert kv.pages(b) == [0, 1, 3] and kv.pages(c) == [0, 1, 4]
    kv.extend([a], [9])
    assert kv.pages(a) == [0, 1, 2, 5]
    kv.close_sequence(a)
    assert kv.pages(b) == [0, 1, 3] and kv.free_pages == 20 - 4
    # All holders of one tail in one call: the last keeps it.
    d = kv.fork(b)
    kv.extend([b, d], [1, 1])
    assert kv.pages(b) == [0, 1, 2] and kv.pages(d) == [0, 1, 3]
    # A full last page is shared without a copy.
    kv.truncate(d, 32)
    e = kv.open()
    f = kv.fork(d)
    kv.extend([d, f], [1, 1])
    assert kv.pages(d)[:2] == kv.pages(f)[:2] == [0, 1] and kv.pages(d)[2] != kv.pages(f)[2]
    assert kv.length(e) == 0


def test_capacity_counts_copies():
    kv = owner(pages=4)
    a = kv.open()
    kv.extend([a], [40])
    b = kv.fork(a)
    kv.extend([a, b], [1, 1])  # one copy: the fourth page
    assert kv.free_pages == 0
    c = kv.fork(a)
    assert code(kv.extend, [c], [1]) == _lib.CAPACITY
    kv.close_sequence(b)
    kv.extend([c], [1])
    assert kv.free_pages == 0


def test_random_operations_keep_the_books():
    """Reference counts, free pages, sharing and the lowest-page rule over random histories; a model
    of each sequence's keys shows that no page is written while another sequence sees it."""
    rng = random.Random(7)
    for trial in range(30):
        kv = owner(pages=rng.randint(5, 40), sequences=5, sequence_pages=9)
        total = kv.free_pages
        lengths = {}
        for _ in range(120):
            op = rng.choice(("open", "fork", "extend", "extend", "truncate", "close", "compact"))
            try:
                if op == "open":
                    lengths[kv.open()] = 0
                elif op == "compact":
                    kv.compact()
                    used = {p for s in lengths for p in kv.pages(s)}
                    assert not used or max(used) == len(used) - 1
                elif not lengths:
                    continue
                elif op == "fork":
                    s = rng.choice(list(lengths))
                    lengths[kv.fork(s)] = lengths[s]
                elif op == "extend":
                    some = rng.sample(list(lengths), rng.randint(1, len(lengths)))
                    more = [rng.choice((0, 1, 3, 16, 40)) for _ in some]
                    kv.extend(some, more)
                    for s, n in zip(some, more):
                        if n:  # the page under the first new key is this sequence's alone
                            page = kv.pages(s)[lengths[s] // 16]
                            assert all(page not in kv.pages(o) for o in lengths if o != s)
                        lengths[s] += n
                elif op == "truncate":
                    s = rng.choice(list(lengths))
                    lengths[s] = rng.randint(0, lengths[s])
                    kv.truncate(s, lengths[s])
                else:
                    s = rng.choice(list(lengths))
                    kv.close_sequence(s)
                    del lengths[s]
            except ops.TkhError as e:
                assert e.code == _lib.CAPACITY
            assert {s: kv.length(s) for s in lengths} == lengths
            used = {p for s in lengths for p in kv.pages(s)}
            assert kv.free_pages == total - len(used)
            for s in lengths:
                assert len(set(kv.pages(s))) == len(kv.pages(s)) == -(-lengths[s] // 16)
        kv.close()


def test_create_refusals():
    def create(layers=1, kv_heads=1, head_dim=64, page_tokens=16, pages=4, sequences=1, sequence_pages=4,
               storage=torch.float32):
        return paged.PagedKv(None, layers, kv_heads, head_dim, page_tokens, pages, sequences, sequence_pages, storage)

    create().close()
    for name in ("layers", "kv_heads", "head_dim", "page_tokens", "pages", "sequences", "sequence_pages"):
        assert code(lambda: create(**{name: 0})) == _lib.ZERO_DIMENSION
    for args in (dict(head_dim=80), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=2048),
                 dict(pages=2 ** 40), dict(sequences=2 ** 20), dict(sequence_pages=2 ** 30)):
        assert code(lambda: create(**args)) in (_lib.UNSUPPORTED, _lib.SIZE_OVERFLOW)
    assert code(lambda: create(layers=2 ** 62)) == _lib.SIZE_OVERFLOW


def layout(**kw):
    d = dict(pages=4, page_tokens=16, kv_heads=2, head_dim=64, page_stride=2048, head_stride=1024, row_stride=64)
    d.update(kw)
    return _lib.PagedLayout(**d)


def batch(**kw):
    d = dict(sequences=2, total_queries=2, max_queries=1, max_keys=64, table_rows=2, table_stride=4,
             page_table=None, key_lens=None, query_start=None, slots=None)
    d.update(kw)
    return _lib.PagedBatch(**d)


def attention(b=None, lay=None, heads=4, dtype=_lib.BF16, q=None, kv=8192, scale=0.125, window=0, softcap=0.0):
    b, lay = b or batch(), lay or layout()
    err = _lib.Error()
    n = b.total_queries * heads * lay.head_dim if q is None else q
    rc = _lib.load().tkh_paged_attention(None, ctypes.byref(b), ctypes.byref(lay), heads, dtype, None, n, None, kv, None,
                                         kv, scale, window, softcap, None, n, ctypes.byref(err))
    return rc, err


def test_attention_refusals():
    rc, err = attention()
    assert rc == _lib.INVALID_PARAMETER and err.tensor == b"context"  # only the context is missing
    for kw in (dict(pages=0), dict(kv_heads=0), dict(head_dim=0), dict(page_tokens=0)):
        assert attention(lay=layout(**kw))[0] == _lib.ZERO_DIMENSION
    for kw in (dict(head_dim=96), dict(page_tokens=24), dict(page_tokens=8)):
        assert attention(lay=layout(**kw))[0] == _lib.UNSUPPORTED
    for kw in (dict(row_stride=60), dict(row_stride=56), dict(head_stride=32), dict(head_stride=512), dict(page_stride=1024),
               dict(page_stride=2052)):
        assert attention(lay=layout(**kw))[0] == _lib.INVALID_PARAMETER, kw
    # Heads outside rows, rows outside heads, and room between them.
    for kw in (dict(head_stride=64, row_stride=128), dict(page_stride=4096), dict(head_stride=1032, page_stride=2056)):
        rc, err = attention(lay=layout(**kw), kv=10 ** 6)
        assert rc == _lib.INVALID_PARAMETER and err.tensor == b"context", kw
    assert attention(lay=layout(page_stride=2 ** 62))[0] == _lib.SIZE_OVERFLOW
    # Strides whose bytes pass 32 bits, and more query rows than 2^30.
    for kw in (dict(page_stride=2 ** 30 + 8), dict(row_stride=2 ** 17 + 8, page_stride=2 ** 29)):
        assert attention(lay=layout(**kw))[0] == _lib.UNSUPPORTED, kw
    assert attention(lay=layout(pages=1, page_stride=2 ** 31))[1].tensor == b"context"
    assert attention(batch(total_queries=2 ** 24, query_start=64), heads=128)[0] == _lib.UNSUPPORTED
    for name in ("sequences", "max_queries", "max_keys", "table_rows", "table_stride"):
        assert attention(batch(**{name: 0}))[0] == _lib.ZERO_DIMENSION, name
    assert attention(batch(total_queries=3))[0] == _lib.LENGTH
    assert attention(batch(total_queries=3, query_start=64))[1].tensor == b"context"  # rows behind the batch
    assert attention(batch(total_queries=1))[0] == _lib.LENGTH
    assert attention(batch(table_rows=1))[0] == _lib.INVALID_PARAMETER
    assert attention(batch(max_keys=65))[0] == _lib.INVALID_PARAMETER
    assert attention(heads=3)[0] == _lib.INVALID_PARAMETER
    assert attention(heads=0, q=0)[0] == _lib.ZERO_DIMENSION
    assert attention(dtype=3)[0] == _lib.INVALID_PARAMETER
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attention(scale=scale)[0] == _lib.INVALID_PARAMETER
    for cap in (-1.0, float("nan"), float("inf")):
        assert attention(softcap=cap)[0] == _lib.INVALID_PARAMETER
    rc, err = attention(q=511)
    assert rc == _lib.LENGTH and err.tensor == b"q" and err.expected == 512
    rc, err = attention(kv=8191)
    assert rc == _lib.LENGTH and err.tensor == b"k pages" and err.expected == 8192


def produce(rope=None, stride=None, rows=None, norm=False, eps=1e-6, heads=4, dtype=_lib.BF16, src=_lib.F32, q=512):
    b, lay, err = batch(), layout(), _lib.Error()
    s = stride or [256, 128, 128]
    n = rows or [s[0] + 256, s[1] + 128, s[2] + 128]
    at = 16 if norm else None
    proj = _lib.PagedProjections(None, None, None, *s, *n, at, at, eps)
    r = _lib.Rope(1, 0, 0, 1e4, 1.0, 1.0, 4.0, 1.0, 8192)
    for k, v in (rope or {}).items():
        setattr(r, k, v)
    rc = _lib.load().tkh_paged_produce(None, ctypes.byref(b), ctypes.byref(lay), ctypes.byref(r), heads, src,
                                       ctypes.byref(proj), dtype, None, q, None, 8192, None, 8192, ctypes.byref(err))
    return rc, err


def test_produce_refusals():
    rc, err = produce()
    assert rc == _lib.INVALID_PARAMETER and err.tensor == b"context"
    nan, inf = float("nan"), float("inf")
    for rope in (dict(layout=3), dict(scaling=3), dict(theta=0.0), dict(theta=nan), dict(magnitude=0.0), dict(magnitude=inf),
                 dict(rotated_dims=72), dict(scaling=1, factor=0.5), dict(scaling=2, factor=nan),
                 dict(scaling=2, low_freq_factor=0.0), dict(scaling=2, high_freq_factor=1.0),
                 dict(scaling=2, original_max_positions=0)):
        rc, err = produce(rope)
        assert rc == _lib.INVALID_PARAMETER and err.tensor != b"context", rope
    assert produce(dict(rotated_dims=12))[0] == _lib.UNSUPPORTED
    assert produce(dict(layout=0, theta=nan))[1].tensor == b"context"  # unused without a rotation
    for stride in ([255, 128, 128], [256, 124, 128], [256, 128, 130]):
        assert produce(stride=stride)[0] == _lib.INVALID_PARAMETER and produce(stride=stride)[1].tensor != b"context"
    rc, err = produce(rows=[512, 255, 256])
    assert rc == _lib.LENGTH and err.tensor == b"k projection"
    assert produce(norm=True, eps=0.0)[1].tensor == b"norm epsilon"
    assert produce(q=500)[0] == _lib.LENGTH
    assert produce(dtype=7)[0] == produce(src=9)[0] == _lib.INVALID_PARAMETER


def test_copy_refusals():
    def copy(src, dst, pool_bytes=4096, planes=2, plane_stride=2048, pages=4, page_stride=512, page_bytes=512):
        err = _lib.Error()
        a, b = ops._u64s(src), ops._u64s(dst)
        rc = _lib.load().tkh_copy_pages(None, None, pool_bytes, planes, plane_stride, pages, page_stride, page_bytes, a, b,
                                        len(src), ctypes.byref(err))
        return rc, err

    rc, err = copy([0], [1])
    assert rc == _lib.INVALID_PARAMETER and err.tensor == b"context"
    rc, err = copy([0, 4], [1, 2])
    assert rc == _lib.INVALID_PARAMETER and err.tensor == b"page" and err.index == 1
    assert copy([0], [-1])[1].tensor == b"page"
    for kw in (dict(planes=0), dict(pages=0), dict(page_bytes=0)):
        assert copy([0], [0], **kw)[0] == _lib.ZERO_DIMENSION
    for kw in (dict(page_bytes=511, page_stride=511), dict(page_stride=256), dict(plane_stride=1024)):
        assert copy([0], [1], **kw)[0] == _lib.INVALID_PARAMETER
        assert copy([0], [1], **kw)[1].tensor != b"context"
    assert copy([0], [1], pool_bytes=4095)[0] == _lib.LENGTH
    assert copy([0], [1], planes=4, plane_stride=512, page_stride=2048, pool_bytes=8192)[1].tensor == b"context"
    assert copy([0], [1], page_stride=2 ** 63, plane_stride=2 ** 63)[0] == _lib.SIZE_OVERFLOW


def test_bindings_refuse_tensors():
    t = torch.zeros(2, 4, dtype=torch.int32)
    b = ops.PagedBatch(page_table=t, key_lens=t[0], total_queries=1, max_queries=1, max_keys=1)
    with pytest.raises(TypeError):
        b._c(0)  # not on the device
    b.page_table = t.long()
    with pytest.raises(TypeError):
        b._c(-1)
    b.page_table = t[:, ::2]
    with pytest.raises(ValueError):
        b._c(-1)
    b.page_table = t[:1].expand(2, 4)
    with pytest.raises(ValueError):
        b._c(-1)
    with pytest.raises(ValueError):
        ops.RotaryPositions(layout="spiral")._c()
    k = torch.zeros(3, 2, 16, 64)
    with pytest.raises(ValueError):
        ops._paged_layout(k, k[:2])
    with pytest.raises(ValueError):
        ops._paged_layout(k, k.transpose(2, 3))
    with pytest.raises(ValueError):
        ops._rows(torch.zeros(3, 4, 64), 3, 2, 64)
    with pytest.raises(ValueError):
        ops._rows(torch.zeros(3, 4, 128)[..., ::2], 3, 4, 64)
    assert ops._rows(torch.zeros(3, 6, 64)[:, :4], 3, 4, 64) == (384, 2 * 384 + 256)


def test_struct_layouts_match_header():
    names = {"tkh_paged_layout": _lib.PagedLayout, "tkh_paged_batch": _lib.PagedBatch, "tkh_rope": _lib.Rope,
             "tkh_paged_projections": _lib.PagedProjections, "tkh_paged_options": _lib.PagedOptions,
             "tkh_paged_info": _lib.PagedInfo}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "tokhip.h"\nint main(void){' + "".join(
        f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in c._fields_)
        for n, c in names.items()) + "return 0;}"
    with tempfile.TemporaryDirectory() as d:
        c, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        open(c, "w").write(src)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = [x for c in names.values() for x in [ctypes.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]]
    assert got == want
