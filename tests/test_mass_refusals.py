"""What the operators of a bounded cache refuse, on the host: nothing here reaches a device."""
import ctypes

import pytest
import torch

from kinetics_b200 import _lib, ops

ONE, NULL = 1 << 12, None               # an aligned dummy address, never dereferenced


def _shape(**kw):
    base = dict(batch=2, num_kv_heads=1, group_size=4, head_dim=128, page_size=16, dtype=1, num_pages=8)
    base.update(kw)
    return _lib.Shape(*[base[f] for f, _ in _lib.Shape._fields_])


def _mass(a=ONE, b=ONE, stride=64, rows=2):
    return _lib.Mass(a, b, stride, rows, 1.0)


def _decode(shape=None, mass=None, q=ONE, ws=ONE, bytes_=1 << 30, pages=5000, total=-1, view=None, **kw):
    return _lib.load().ktk_dense_decode_mass(q, ONE, ONE, ONE, ONE, view, pages, total, 0.1, mass or _mass(), ONE, ws, bytes_,
                                             shape or _shape(**kw), NULL, NULL)


def _prefill(shape=None, mass=None, total=5, new=3, pages=4, window=0, scale=0.1, ws=ONE, bytes_=1 << 30, q=ONE, **kw):
    return _lib.load().ktk_prefill_attention_mass(q, ONE, total, new, ONE, ONE, ONE, ONE, None, pages, -1, window, scale,
                                                  mass or _mass(), ONE, ws, bytes_, shape or _shape(**kw), NULL, NULL)


def _evict(shape=None, mass=None, pos=ONE, pos_out=ONE, pages=400, keep=2000, sink=0, recent=0, ws=ONE, bytes_=1 << 30, kv=ONE, **kw):
    return _lib.load().ktk_evict(kv, ONE, ONE, ONE, None, pages, mass or _mass(), pos, pos_out, ONE, ONE, keep, sink, recent, ws, bytes_,
                                 shape or _shape(**kw), NULL, NULL)


@pytest.mark.parametrize("call", [_decode, _prefill, _evict])
def test_sizes_and_pointers(call):
    text = _lib.load().ktk_last_error
    assert call(head_dim=64) == -2 and b"head_dim" in text()
    assert call(page_size=32) == -2
    assert call(group_size=3) == -2
    assert call(dtype=7) == -1
    assert call(batch=0) == 0                                                # nothing to do
    assert call(mass=_mass(a=None)) == -1 and b"mass" in text()
    assert call(mass=_mass(stride=0)) == -1 and call(mass=_mass(rows=0)) == -1
    # in place or apart, nothing in between: 2 rows of 64 places, one kv head
    assert call(mass=_mass(ONE, ONE + 4)) == -1 and b"overlap" in text()
    assert call(mass=_mass(ONE + 508, ONE)) == -1
    assert call(ws=None) == -3 and b"workspace" in text()
    assert call(bytes_=1) == -3
    assert call(ws=ONE + 8) == -1 and b"aligned" in text()


def test_each_ones_own():
    text = _lib.load().ktk_last_error
    assert _decode(q=None) == -1 and _prefill(q=ONE + 2) == -1 and _evict(kv=ONE + 2) == -1
    for scale in (0.0, -0.1, 1e-31, float("nan"), float("inf")):
        assert _prefill(scale=scale) == -1 and b"sm_scale" in text()
    assert _prefill(total=0) == 0
    assert _prefill(window=-1) == -1 and _prefill(new=0) == -1 and _prefill(pages=0) == -1
    assert _prefill(pages=1 << 40) == -5 and _decode(pages=(1 << 26) + 1) == -5 and _decode(pages=(1 << 31) - 1) == -5
    assert _evict(keep=0) == -1 and _evict(sink=-1) == -1 and _evict(recent=-1) == -1
    assert _evict(keep=8, sink=5, recent=4) == -1 and b"sink + recent" in text()
    assert _evict(sink=(1 << 31) - 1, recent=(1 << 31) - 1, keep=(1 << 31) - 1) == -1      # their sum passes 32 bits
    assert _evict(pos_out=ONE + 4) == -1 and b"positions" in text()
    assert _evict(pages=40000) == -5 and _evict(pages=40000, keep=40000 * 16 - 1) == -5
    bad = _lib.View(16, 0, 0, 0, 0)
    assert _decode(view=bad) == -1


def test_workspaces_are_sized_by_what_is_given():
    lib = _lib.load()
    shp = _shape()
    assert lib.ktk_decode_mass_workspace_bytes(shp, 100, -1) == 0                                  # short lists: a cluster each
    small = lib.ktk_decode_mass_workspace_bytes(shp, 4000, 50)
    assert lib.ktk_decode_mass_workspace_bytes(shp, 4000, -1) - small == 7950 * 16 * 4 * 4         # scores of 8000 pages instead of 50
    assert lib.ktk_decode_mass_workspace_bytes(shp, 4000, 10 ** 9) == lib.ktk_decode_mass_workspace_bytes(shp, 4000, -1)
    assert ops.decode_mass_workspace_bytes(2, 1, 4, 4000, torch.bfloat16, 50) == small
    assert lib.ktk_decode_mass_workspace_bytes(_shape(head_dim=64), 4000, -1) == 0
    assert lib.ktk_evict_workspace_bytes(shp, 4, 40) == 0                                         # 24 of 64 tokens can move: one launch
    assert lib.ktk_evict_workspace_bytes(shp, 40, 200) == 0                                       # 200, and few rows: the same
    assert lib.ktk_evict_workspace_bytes(_shape(batch=200), 40, 200) == 200 * 4 * (1 + 2 * 200)
    assert lib.ktk_evict_workspace_bytes(shp, 256, 2000) == 2 * 4 * (1 + 2 * 2000)
    assert lib.ktk_evict_workspace_bytes(shp, 256, 2500) == 2 * 4 * (1 + 2 * 1596)
    assert lib.ktk_evict_workspace_bytes(shp, 32769, 500) == 0                                    # refused
    # a share of scores in bytes passes 32 bits: no list of that length is kept in shared memory
    assert lib.ktk_decode_mass_workspace_bytes(_shape(group_size=8, batch=1), 1 << 26, 100) > 0
    # weights of few rows need their denominators only; of many, and few keys, sums over parts
    rows = lib.ktk_prefill_mass_workspace_bytes(shp, 10, 10, 4, -1, 0)
    assert rows == 768 and lib.ktk_prefill_mass_workspace_bytes(shp, 10, 10, 4, -1, 3) == rows     # 40 rows of 16 bytes
    assert lib.ktk_prefill_mass_workspace_bytes(shp, 8192, 8192, 4, -1, 0) > 8192 * 4 * 16
    assert lib.ktk_prefill_mass_workspace_bytes(shp, 8192, 8192, 4, -1, 64) == 8192 * 4 * 16


def _tensors(dtype=torch.bfloat16):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    return dict(q=torch.zeros(2, 4, 128, dtype=dtype), kv=torch.zeros(8, 2, 16, 1, 128, dtype=dtype), indices=i32(0, 1, 2),
                indptr=i32(0, 1, 3), last=i32(3, 4), mass=torch.zeros(2, 1, 64), positions=torch.zeros(2, 1, 64, dtype=torch.int32),
                counts=i32(0, 0), q_indptr=i32(0, 1, 2))


def test_no_cpu_fallback():
    t = _tensors()
    table = (t["kv"], t["indices"], t["indptr"], t["last"])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dense_decode_mass(t["q"], *table, 2, t["mass"])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.prefill_attention_mass(t["q"], t["q_indptr"], 1, *table, t["mass"])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.evict(*table, 2, t["mass"], t["positions"], t["counts"], t["counts"], 8)


def _plan(t, **kw):
    return ops._decode_mass_plan(t["q"].shape, t["q"].dtype, t["kv"].shape, t["kv"].dtype, t["mass"].shape, t["mass"].dtype, False, False,
                                 ops._tables(len(t["q"]), t["indices"], t["indptr"], t["last"], None), 2)


@pytest.mark.parametrize("name, value, error", [
    ("q", torch.zeros(2, 128, dtype=torch.bfloat16), ValueError),
    ("q", torch.zeros(2, 4, 64, dtype=torch.bfloat16), ValueError),
    ("q", torch.zeros(2, 4, 128), TypeError),
    ("q", torch.zeros(3, 4, 128, dtype=torch.bfloat16), ValueError),         # three queries, two sequences
    ("kv", torch.zeros(8, 16, 1, 128, dtype=torch.bfloat16), ValueError),
    ("kv", torch.zeros(8, 2, 16, 3, 128, dtype=torch.bfloat16), ValueError),  # four heads over three
    ("mass", torch.zeros(2, 1, 64, dtype=torch.float64), TypeError),
    ("mass", torch.zeros(2, 2, 64), ValueError),
    ("mass", torch.zeros(1, 1, 64), ValueError),                             # one row, two sequences
    ("mass", torch.zeros(2, 64), ValueError),
    ("indices", torch.zeros(3, dtype=torch.int64), TypeError),
    ("indptr", torch.zeros(3, dtype=torch.int64), TypeError),
    ("last", torch.zeros(1, dtype=torch.int32), ValueError),
])
def test_shapes_and_types(name, value, error):
    t = _tensors()
    _plan(t)
    t[name] = value
    with pytest.raises(error):
        _plan(t)


def test_half_precision_is_not_built():
    t = _tensors(torch.float16)
    with pytest.raises(TypeError, match="not supported"):
        _plan(t)


def test_manager_settings():
    from kinetics_b200 import EvictingKVManager, get_config
    for kw in (dict(keep=0), dict(keep=8, sink=5, recent=4), dict(keep=8, sink=-1), dict(keep=8, recent=-1), dict(keep=100, room=0),
               dict(keep=100, portion=0), dict(keep=100, window=-1)):
        with pytest.raises(ValueError):
            EvictingKVManager(get_config("cfg1"), 1, 64, "cuda", torch.bfloat16, **kw)
