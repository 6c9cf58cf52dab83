"""CPU: the scheduler-step entry points (step tables, multi-axis rotary,
ragged-chunk attention) refuse bad arguments with a status and a message
before any CUDA call, and their wrappers refuse host tensors."""

import ctypes

import pytest
import torch

ARG, UNSUPPORTED, WORKSPACE = 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    from kessie_b200 import _lib
    return _lib.load()


def _msg():
    from kessie_b200 import _lib
    return _lib.last_error()[1]


def _tables(lib, **kw):
    a = dict(ctx=16, new=16, R=2, table=16, stride=8, maxp=8, ps=16, pages=10, free=16, nfree=4, count=None, T=4,
             start=16, seq=16, pos=16, slots=16, used=16)
    a.update(kw)
    return lib.kessie_step_tables_v2(a["ctx"], a["new"], a["R"], a["table"], a["stride"], a["maxp"], a["ps"],
                                     a["pages"], a["free"], a["nfree"], a["count"], a["T"], a["start"], a["seq"],
                                     a["pos"], a["slots"], a["used"], None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(R=-1), ARG, "sizes"), (dict(ps=0), ARG, "sizes"), (dict(T=-3), ARG, "sizes"), (dict(nfree=-1), ARG, "sizes"),
    (dict(R=8193), UNSUPPORTED, "8193"), (dict(stride=7), ARG, "stride"), (dict(ctx=None), ARG, "null"),
    (dict(start=None), ARG, "null"), (dict(table=None), ARG, "null"), (dict(free=None), ARG, "null"),
    (dict(slots=None), ARG, "null"), (dict(used=None), ARG, "null")])
def test_step_tables_refuses(lib, kw, status, word):
    assert _tables(lib, **kw) == status
    assert word in _msg()


def _remap(lib, sections=(16, 24, 24), interleaved=0, dtype=1, T=4, H=2, D=128, k=16, theta=1e4, tgt=16):
    sec = (ctypes.c_int * max(len(sections), 1))(*sections)
    return lib.kessie_rope_axes_remap_v2(k, 256, 128, 16, 256, 128, dtype, T, H, D, None, 0, tgt, 4, sec,
                                         len(sections), interleaved, theta, None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(dtype=7), UNSUPPORTED, "dtype"), (dict(T=-1), ARG, "shape"), (dict(D=0), ARG, "shape"),
    (dict(k=None), ARG, "null"), (dict(tgt=None), ARG, "null"), (dict(sections=()), ARG, "axes"),
    (dict(sections=(1,) * 9), ARG, "axes"), (dict(sections=(16, -1)), ARG, "section"),
    (dict(sections=(0, 0)), UNSUPPORTED, "frequencies"), (dict(sections=(200, 57)), UNSUPPORTED, "frequencies"),
    (dict(sections=(40, 40)), ARG, "rotated"), (dict(sections=(16, 24, 24), interleaved=1), ARG, "interleave"),
    (dict(theta=0.0), ARG, "theta"), (dict(theta=float("nan")), ARG, "theta"), (dict(theta=float("inf")), ARG, "theta")])
def test_rope_axes_remap_refuses(lib, kw, status, word):
    assert _remap(lib, **kw) == status
    assert word in _msg()


def _insert(lib, dtype=1, T=4, Hq=4, Hkv=2, D=128, pages=3, ps=16, slots=16, q=16, kv=16):
    sec = (ctypes.c_int * 1)(64)
    return lib.kessie_rope_axes_insert_v2(q, 512, 128, 16, 512, 128, 16, 256, 128, 16, 256, 128, dtype, T, Hq, Hkv, D,
                                          16, 4, sec, 1, 0, 1e4, kv, 8192, 512, 256, 128, pages, ps, slots, None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(dtype=3), UNSUPPORTED, "dtype"), (dict(Hkv=0), ARG, "shape"), (dict(pages=0), ARG, "shape"),
    (dict(ps=0), ARG, "shape"), (dict(slots=None), ARG, "null"), (dict(q=None), ARG, "null"), (dict(kv=None), ARG, "null")])
def test_rope_axes_insert_refuses(lib, kw, status, word):
    assert _insert(lib, **kw) == status
    assert word in _msg()


def _chunks(lib, **kw):
    a = dict(q=16, k=16, v=16, qst=1024, qsh=128, page=4096, tok=256, head=128, pages=4, ps=16, table=16, start=16,
             seq=16, window=0, scale=0.1, B=2, T=5, Hq=8, Hkv=2, D=128, maxs=64, dt=1, out=16, ws=16, wsn=1 << 40)
    a.update(kw)
    return lib.kessie_paged_fog_chunks_v2(a["q"], a["qst"], a["qsh"], a["k"], a["v"], a["page"], a["tok"], a["head"],
                                          a["pages"], a["ps"], a["table"], 8, a["start"], a["seq"], None, 0.5,
                                          a["window"], 1, a["scale"], a["B"], a["T"], a["Hq"], a["Hkv"], a["D"],
                                          a["maxs"], a["dt"], None, a["out"], 1024, 128, a["ws"], a["wsn"], None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(dt=2), UNSUPPORTED, "dtype"), (dict(D=96), UNSUPPORTED, "head_dim"), (dict(ps=24), UNSUPPORTED, "page_size"),
    (dict(ps=0), UNSUPPORTED, "page_size"), (dict(Hq=7), ARG, "shape"), (dict(B=-1), ARG, "shape"),
    (dict(T=-1), ARG, "shape"), (dict(pages=0), ARG, "shape"), (dict(Hq=258, Hkv=2), UNSUPPORTED, "129"),
    (dict(scale=0.0), ARG, "sm_scale"), (dict(scale=-1.0), ARG, "sm_scale"), (dict(scale=float("inf")), ARG, "sm_scale"),
    (dict(q=None), ARG, "null"), (dict(start=None), ARG, "null"), (dict(out=None), ARG, "null"),
    (dict(q=24), ARG, "aligned"), (dict(tok=260), ARG, "aligned"), (dict(ws=None), WORKSPACE, "workspace"),
    (dict(wsn=0), WORKSPACE, "workspace")])
def test_paged_fog_chunks_refuses(lib, kw, status, word):
    assert _chunks(lib, **kw) == status
    assert word in _msg()


def test_nothing_to_do_is_ok(lib):
    assert _chunks(lib, T=0) == 0 and _chunks(lib, B=0) == 0
    assert _remap(lib, T=0) == 0 and _insert(lib, T=0) == 0


def test_wrappers_refuse_host_tensors():
    from kessie_b200 import ops
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.step_tables(i, i, torch.zeros(2, 4, dtype=torch.int32), 16, i, 4)
    x = torch.zeros(2, 4, 128)
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_axes_remap(x, None, torch.zeros(1, 2, dtype=torch.int32), [64])
    with pytest.raises(ValueError, match="CUDA"):
        ops.rope_axes_insert(x, x, x, torch.zeros(1, 2, dtype=torch.int32), [64], torch.zeros(1, 16, 2, 4, 128), i)
    c = torch.zeros(4, 16, 4, 128)
    with pytest.raises(ValueError, match="CUDA"):
        ops.paged_fog_chunks(x, c, c, torch.zeros(1, 4, dtype=torch.int32), i, i[:1])


def _buffers():
    return {n: ctypes.addressof(b) for n, b in _KEEP.items()}


_KEEP = {n: (ctypes.c_int64 * 64)() for n in ("ctx", "new", "table", "free", "count", "start", "seq", "pos", "slots",
                                             "used")}


@pytest.mark.parametrize("output,source", [("seq", "ctx"), ("seq", "new"), ("start", "ctx"), ("used", "count"),
                                           ("pos", "free"), ("slots", "new"), ("table", "free")])
def test_step_tables_refuses_outputs_in_its_inputs(lib, output, source):
    """The inputs are read by every block while another writes: last step's
    seq_lens cannot be the context lengths of a call that writes them."""
    at = _buffers()
    at[output] = at[source]
    assert _tables(lib, **at) == ARG and "shares memory" in _msg(), _msg()
    at[output] = at[source] + 4                                       # one element on
    if output not in ("used",):
        assert _tables(lib, **at) == ARG and "shares memory" in _msg(), _msg()


def test_outputs_whose_rows_share_memory_are_refused(lib):
    sec = (ctypes.c_int * 1)(64)
    for st, sh in ((0, 128), (256, 0)):
        assert lib.kessie_rope_axes_remap_v2(16, 256, 128, 16, st, sh, 1, 4, 2, 128, None, 0, 16, 4, sec, 1, 0, 1e4,
                                             None) == ARG
        assert "share memory" in _msg()
