"""The prompt and beam operators without a GPU: what the C ABI refuses before
any device call, workspace sizes, the torch schemas, fake kernels, and that no
CPU tensor is accepted."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import bc_capi as C
import branchcraft_torch as B

P = ctypes.c_void_p(1024)
ODD = ctypes.c_void_p(1026)
LIB = C.lib()


def shape(**kw):
    d = dict(batch=2, query_heads=8, kv_heads=2, dim=64, max_pages=4, physical_pages=10) | kw
    return C.make_shape(*d.values())


def test_append_plan_refusals():
    def call(batch=2, pool=10, width_in=4, width_out=4, max_tokens=5, out=ctypes.c_void_p(2048),
             pages=P, slots=P, scratch=P):
        return LIB.bc_append_plan(batch, pool, pages, width_in, P, P, P, P, P, P, P, P, out,
                                  width_out, P, max_tokens, P, slots, P, P, P, scratch, None)

    assert call(batch=0) == 1
    assert call(batch=4097) == 1
    assert call(pool=0) == 1
    assert call(pool=2 ** 27) == 1
    assert call(width_in=0) == 1
    assert call(width_out=2 ** 27) == 1
    assert call(max_tokens=-1) == 1
    assert call(out=P, width_out=5) == 1
    assert call(pages=None) == 1
    assert call(slots=None) == 1
    assert call(scratch=None) == 1


def test_append_kv_refusals():
    layout = C.KvLayout(2048, 128, 64)

    def call(s=None, tokens=3, k=P, stride=128, cache=P, lay=layout, clones=None, n=0, counts=None):
        return LIB.bc_append_kv(ctypes.byref(s or shape()), tokens, k, stride, P, 128, cache, P,
                                ctypes.byref(lay) if lay else None, P, clones, n, counts, None)

    assert call(s=shape(dim=96)) == 1
    assert call(s=shape(kv_heads=0)) == 1
    assert call(s=shape(physical_pages=0)) == 1
    assert call(tokens=-1) == 1
    assert call(k=None) == 1
    assert call(k=ODD) == 1
    assert call(stride=132) == 1
    assert call(stride=-128) == 1
    assert call(cache=ODD) == 1
    assert call(lay=None) == 1
    assert call(lay=C.KvLayout(2048, 124, 64)) == 1
    assert call(lay=C.KvLayout(2048, 0, 64)) == 1
    assert call(n=1) == 1
    assert call(clones=P, n=1) == 1
    assert call(n=-1) == 1


def test_chunk_refusals():
    layout = C.KvLayout(2048, 128, 64)

    def call(s=None, tokens=3, dtype=0, q=P, stride=512, lay=layout, ws=P, size=None, **o):
        s = s or shape()
        opt = C.ChunkOptions(*(dict(scale=0.125, softcap=0.0, window=0, alibi_slopes=None,
                                    prefix=None, key_start=None) | o).values())
        if size is None:
            size = C.chunk_workspace_bytes(s, max(tokens, 0))
        return LIB.bc_chunk_attention(ctypes.byref(s), tokens, dtype, q, stride, P, P,
                                      ctypes.byref(lay) if lay else None, P, P, P,
                                      ctypes.byref(opt), P, 0, ws, size, None)

    for s in (shape(dim=96), shape(query_heads=9), shape(query_heads=0), shape(batch=0),
              shape(max_pages=0), shape(physical_pages=0), shape(query_heads=258, kv_heads=2),
              shape(physical_pages=2 ** 27), shape(max_pages=2 ** 27)):
        assert call(s=s) == 1
    assert call(tokens=-1) == 1
    assert call(dtype=2) == 1
    assert call(dtype=-1) == 1
    assert call(q=None) == 1
    assert call(q=ODD) == 1
    assert call(stride=508) == 1
    assert call(stride=-512) == 1
    assert call(lay=None) == 1
    assert call(lay=C.KvLayout(2048, 128, 72)) == 1
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=bad) == 1
    for bad in (-1.0, float("nan"), float("inf")):
        assert call(softcap=bad) == 1
    assert call(window=-1) == 1
    if C.chunk_workspace_bytes(shape(), 3):
        assert call(ws=None) == 1
        assert call(size=C.chunk_workspace_bytes(shape(), 3) - 1) == 1


def test_beam_refusals():
    def call(batch=2, beams=3, vocab=50, k=4, dtype=2, logits=P, stride=50, ws=P, size=None):
        if size is None:
            size = LIB.bc_beam_workspace_bytes(batch, beams, vocab, k, dtype)
        return LIB.bc_beam_select(batch, beams, vocab, k, dtype, logits, stride, P, P, P, P, ws,
                                  size, None)

    for kw in (dict(batch=0), dict(beams=0), dict(beams=65), dict(vocab=0),
               dict(vocab=2 ** 20 + 1, stride=2 ** 21), dict(k=0), dict(k=65), dict(k=5, vocab=1),
               dict(dtype=3), dict(dtype=-1), dict(logits=None), dict(logits=ODD),
               dict(stride=49), dict(ws=None), dict(ws=ODD), dict(size=10)):
        assert call(**kw) == 1, kw
    assert C.beam_workspace_bytes(2, 3, 50, 65, torch.float32) == 0
    assert C.beam_workspace_bytes(2, 3, 50, 4, torch.float32) > 0


def test_reorder_refusals():
    def call(batch=2, beams=3, out=3, pool=10, width=4, po=ctypes.c_void_p(2048), ws=P, size=None):
        if size is None:
            size = C.reorder_workspace_bytes(batch, beams, width)
        return LIB.bc_beam_reorder(batch, beams, out, pool, P, width, P, P, P, P, P, P, P, P, po,
                                   ctypes.c_void_p(4096), ws, size, None)

    for kw in (dict(batch=0), dict(beams=0), dict(beams=65), dict(out=0), dict(out=65),
               dict(pool=0), dict(width=0), dict(po=P), dict(ws=None), dict(ws=ODD),
               dict(size=8), dict(batch=2 ** 25, width=64)):
        assert call(**kw) == 1, kw
    assert C.reorder_workspace_bytes(2, 65, 4) == 0


def test_fake_kernels():
    with FakeTensorMode():
        i = dict(dtype=torch.int32)
        pages, lengths = torch.empty(6, 9, **i), torch.empty(6, **i)
        state = torch.empty(50, **i), torch.empty(50, **i), torch.empty(1, **i)
        out = B.append_plan(pages, lengths, lengths, *state, 40, 12)
        assert [tuple(t.shape) for t in out] == [(6, 12), (6,), (50,), (50,), (1,), (7,), (40,),
                                                 (40,), (3, 6), (3,)]
        out = B.append_plan_(pages, lengths, lengths, *state, 40)
        assert [tuple(t.shape) for t in out] == [(7,), (40,), (40,), (3, 6), (3,)]
        q = torch.empty(40, 8, 64, dtype=torch.bfloat16)
        k = torch.empty(50, 16, 2, 64, dtype=torch.bfloat16)
        assert B.append_kv_(k, k, q[:, :2], q[:, :2], torch.empty(40, **i)) is None
        o = B.chunk_attention(q, k, k, pages, torch.empty(7, **i), lengths, softcap=3.0)
        assert o.shape == q.shape and o.dtype == q.dtype
        o32 = torch.empty(40, 8, 64)
        assert B.chunk_attention_out(q, k, k, pages, torch.empty(7, **i), lengths, o32) is o32
        s, t, p = B.beam_select(torch.empty(2, 3, 100), torch.empty(2, 3), 5)
        assert s.shape == t.shape == p.shape == (2, 5)
        assert s.dtype == torch.float32 and t.dtype == p.dtype == torch.int32
        rows = torch.empty(2, 3, 9, **i)
        out = B.beam_reorder(rows, torch.empty(2, 3, **i), torch.empty(2, 4, **i), *state)
        assert [tuple(t.shape) for t in out] == [(2, 4, 9), (2, 4), (50,), (50,), (1,)]
        out = B.beam_reorder_(rows, torch.empty(2, 3, **i), torch.empty(2, 4, **i), *state)
        assert [tuple(t.shape) for t in out] == [(2, 4, 9), (2, 4)]


def test_cpu_tensors_are_rejected():
    i = torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.float16)
    cache = torch.zeros(1, 16, 1, 64, dtype=torch.float16)
    for call in (lambda: B.append_plan(i[None], i, i, i, i, i, 1),
                 lambda: B.append_kv_(cache, cache, x, x, i),
                 lambda: B.chunk_attention(x, cache, cache, i[None], torch.zeros(2, dtype=torch.int32), i),
                 lambda: B.beam_select(torch.zeros(1, 1, 4), torch.zeros(1, 1), 1),
                 lambda: B.beam_reorder(i[None, None], i[None], i[None], i, i, i)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_chunk_limits_and_output_alignment():
    def call(s, output):
        layout = C.KvLayout(2048, 128, 64)
        opt = C.ChunkOptions(0.125, 0.0, 0, None, None, None)
        size = C.chunk_workspace_bytes(s, 3)
        return LIB.bc_chunk_attention(ctypes.byref(s), 3, 0, P, 512, P, P, ctypes.byref(layout), P,
                                      P, P, ctypes.byref(opt), output, 0, P, size, None)

    assert call(shape(batch=4097), P) == 1
    assert C.chunk_workspace_bytes(shape(batch=4097), 3) == 0
    assert call(shape(), ctypes.c_void_p(4096 + 16)) == 1
    assert call(shape(), ctypes.c_void_p(4096 + 2)) == 1


def test_append_refuses_rows_before_it_plans(monkeypatch):
    from branchcraft_torch import sequences

    def planned(*_):
        raise AssertionError("planned before the rows were checked")

    monkeypatch.setattr(sequences, "append_plan_", planned)
    seq = sequences.PagedSequences(2, 1, 4, 8, 2, 64, device="cpu")
    new = torch.ones(2, dtype=torch.int32)
    good = torch.zeros(2, 2, 64, dtype=torch.float16)
    wide = torch.zeros(2, 2, 68, dtype=torch.float16)
    for bad in (good[:1], good[:, :1], good[..., :32], good.float(), good[0],
                torch.zeros(2, 64, 2, dtype=torch.float16).transpose(1, 2), wide[..., :64],
                torch.zeros(257, dtype=torch.float16)[1:].view(2, 2, 64)):
        with pytest.raises(ValueError):
            seq.append(good, bad, new)
    with pytest.raises(AssertionError):
        seq.append(good, good, new)


def test_tanh_polynomial_error():
    """The coefficients and their error as the source states them."""
    import re
    from pathlib import Path

    import numpy as np

    text = (Path(C.__file__).parent / "csrc" / "branchcraft.cu").read_text()
    coef = [float(x) for x in re.search(r"kTanh\[5\] = \{([^}]*)\}", text)[1].split(",")]
    border = float(re.search(r"kTanhNear = ([\d.]+)", text)[1])
    stated = float(re.search(r"error of tanh there: (\S+) with these", text)[1])
    u = np.linspace(0, border, 200001)
    err = np.abs(u * sum(c * u ** (2 * i) for i, c in enumerate(coef)) - np.tanh(u)).max()
    assert 0.9 * stated < err <= 1.01 * stated


class Recorder:
    """Stands in for the library: keeps a call's arguments, reports success."""

    def __init__(self):
        self.args = None

    def __getattr__(self, name):
        def call(*args):
            self.args = args
            return 0
        return call


def test_capi_strides_of_views(monkeypatch):
    """What the ctypes wrappers take as the distance of rows, and the views they refuse."""
    rec = Recorder()
    monkeypatch.setattr(C, "_lib", rec)
    monkeypatch.setattr(C, "_stream", lambda s=None: None)
    wide = torch.zeros(3, 4, 50)
    out = torch.zeros(3, 2)

    def select(x):
        C.beam_select(x, torch.zeros(x.shape[:2]), 2, out, out.int(), out.int(), out)
        return rec.args[6]

    assert select(wide) == 50
    assert select(wide[:, :1]) == 200   # one beam of every request
    assert select(wide[1:2, :2]) == 50
    assert select(wide[:, :, :40]) == 50
    for bad in (wide[:, :2], wide[:, ::2][:, :1].expand(3, 2, 50), wide[..., ::2],
                wide.transpose(0, 1), torch.zeros(3, 50, 4).transpose(1, 2)):
        with pytest.raises(ValueError):
            select(bad)

    cache = torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    planes = torch.zeros(5, 2, 16, 2, 64, dtype=torch.float16)
    q = torch.zeros(3, 8, 64, dtype=torch.float16)
    i = torch.zeros(4, dtype=torch.int32)
    s = shape(physical_pages=5)

    def both(k, v, x=q):
        C.chunk_attention(s, x, k, v, i, i, i, q)
        chunk = rec.args[4]
        C.append_kv(s, x[:, :2], x[:, :2], k, v, i)
        assert rec.args[3] == rec.args[5] == chunk
        return chunk

    assert both(planes[:, 0], planes[:, 1]) == 512
    assert both(cache, cache, torch.zeros(3, 12, 64, dtype=torch.float16)[:, :8]) == 768
    for k, v in ((cache, planes[:, 1]), (planes[:, 0], cache), (cache, cache[:4]),
                 (cache[..., ::2], cache[..., ::2])):
        with pytest.raises(ValueError):
            both(k, v)
    for x in (torch.zeros(3, 8, 128, dtype=torch.float16)[..., :64],
              torch.zeros(8, 3, 64, dtype=torch.float16).transpose(0, 1)):
        with pytest.raises(ValueError):
            both(cache, cache, x)


def test_chunk_refuses_tables_whose_tiles_pass_an_int():
    """2^31 - 1 keys less a tile: the last key's tile still ends below 2^31."""
    assert C.chunk_workspace_bytes(shape(max_pages=134217719), 3) > 0
    assert C.chunk_workspace_bytes(shape(max_pages=134217720), 3) == 0
    layout = C.KvLayout(2048, 128, 64)
    opt = C.ChunkOptions(0.125, 0.0, 0, None, None, None)
    s = shape(max_pages=134217727)
    assert LIB.bc_chunk_attention(ctypes.byref(s), 3, 0, P, 512, P, P, ctypes.byref(layout), P, P, P,
                                  ctypes.byref(opt), P, 0, P, 2 ** 40, None) == 1
