"""Attention that accumulates weights and eviction, against plain fp64 forms."""
import math

import numpy as np
import pytest
import torch

from helpers import P, paged_state, to_dev
from mass_helpers import attend, evict_moves, evict_order, mass_after, place

pytestmark = pytest.mark.gpu
D = 128


def _case(seed, lens, new, kv_heads, group, dtype, sink=0, rows=None, fill=None):
    """Sequences of `lens` tokens whose last `new` have queries; masses of `rows` rows in a mixed order.  Stale places of the cache hold
    NaN, masses of the new and of the free places too."""
    g = torch.Generator().manual_seed(seed)
    batch, longest = len(lens), max(max(lens), 1)
    cast = lambda t: t.to(dtype).float()
    q = cast(1.3 * torch.randn(sum(new), kv_heads * group, D, generator=g))
    k, v = (cast(torch.randn(batch, kv_heads, longest, D, generator=g)) for _ in range(2))
    k[:, :, :3] += 0.5
    k = cast(k)
    st = paged_state(k, v, lens, dtype, seed=seed, sink=sink, fill=fill)
    rows = rows or batch
    slots = torch.randperm(rows, generator=g)[:batch].to(torch.int32)
    stride = longest + 1 + int(torch.randint(0, 9, (1,), generator=g))
    mass = torch.rand(rows, kv_heads, stride, generator=g)
    for b in range(batch):
        mass[slots[b], :, lens[b] - new[b]:] = float("nan")
    indptr = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
    return dict(q=q.to(dtype), k=k, v=v, st=st, mass=mass, slots=slots, q_indptr=indptr)


def _view(c, lens, sink, dev, padded):
    """A PageView with slots, and (padded) with page counts instead of packed lists."""
    from kinetics_b200 import ops
    count = None
    if padded:
        count = torch.tensor(c["st"]["npages"], dtype=torch.int32, device=dev)
    return ops.PageView(sink, 0, count, c["slots"].to(dev))


def _check(c, out, mass_out, lens, new, kv_heads, group, dtype, window, decay, scale):
    first = c["q_indptr"].tolist()
    before = c["mass"]
    others = [r for r in range(len(before)) if r not in c["slots"].tolist()]
    assert torch.equal(mass_out[others].cpu().nan_to_num(-1), before[others].nan_to_num(-1))
    for b, (n, w) in enumerate(zip(lens, new)):
        row = int(c["slots"][b])
        got = mass_out[row].cpu()
        if w == 0:
            assert torch.equal(got.nan_to_num(-1), before[row].nan_to_num(-1))
            continue
        for h in range(kv_heads):
            q = c["q"][first[b]:first[b + 1], h * group:(h + 1) * group]
            o, o_bound, paid, paid_bound = attend(q, c["k"][b, h, :n], c["v"][b, h, :n], w, window, scale, dtype)
            err = (out[first[b]:first[b + 1], h * group:(h + 1) * group].double().cpu() - o).abs()
            assert bool((err <= o_bound).all()), (b, h, float((err / o_bound).max()))
            want, more = mass_after(before, row, n, w, h, decay, paid)
            err = (got[h, :n].double() - want).abs()
            assert bool((err <= paid_bound + more).all()), (b, h, n, float((err / (paid_bound + more)).max()))
            assert torch.equal(got[h, n:].nan_to_num(-1), before[row, h, n:].nan_to_num(-1))


DECODE = [
    # lengths, kv heads, group, dtype, sink page, page counts
    ([1], 1, 1, torch.bfloat16, 0, False),
    ([1, 16, 17, 15], 2, 2, torch.bfloat16, 0, False),
    ([517], 8, 4, torch.bfloat16, 0, False),
    ([0, 33, 0, 700, 1, 1500, 64, 0], 2, 4, torch.bfloat16, 0, False),
    ([3000, 5, 2049], 2, 8, torch.bfloat16, 0, False),
    ([20000], 1, 1, torch.bfloat16, 0, False),
    ([300, 4, 21, 3, 1000, 20], 2, 4, torch.bfloat16, 4, True),
    ([300, 4, 0, 3, 1000], 3, 2, torch.bfloat16, 4, False),
    ([90 + 7 * i for i in range(70)], 4, 4, torch.bfloat16, 0, False),
    ([90 + 7 * i for i in range(70)], 4, 4, torch.bfloat16, 0, True),
    ([1], 1, 1, torch.float32, 0, False),
    ([0, 1, 17, 333, 0], 2, 4, torch.float32, 0, False),
    ([1300, 5], 4, 2, torch.float32, 0, True),
    ([260, 4, 2], 1, 8, torch.float32, 4, True),
]


@pytest.mark.parametrize("lens, kv_heads, group, dtype, sink, padded", DECODE)
def test_decode_accumulates(cuda_device, lens, kv_heads, group, dtype, sink, padded):
    from kinetics_b200 import ops
    dev, new = cuda_device, [1 if n else 0 for n in lens]
    c = _case(3, lens, new, kv_heads, group, dtype, sink, rows=len(lens) + 3)
    c["q_indptr"] = torch.arange(len(lens) + 1, dtype=torch.int32)
    q = torch.zeros(len(lens), kv_heads * group, D, dtype=dtype)
    q[[b for b, w in enumerate(new) if w]] = c["q"]
    c["q"] = q
    d, view, status = to_dev(c["st"], dev), _view(c, lens, sink, dev, padded), ops.new_status(dev)
    scale, decay = D ** -0.5, 0.75
    most = max(max(c["st"]["npages"]), 1)
    indptr = d["kv_indptr"][:-1].contiguous() if padded else d["kv_indptr"]
    mass = c["mass"].to(dev)
    kept = mass.clone()
    out, mass_out = ops.dense_decode_mass(q.to(dev), d["kv_cache"], d["kv_indices"], indptr, d["kv_last_page_len"], most, mass,
                                          decay, scale, mass_out=mass.clone(), status=status, view=view)
    ops.raise_on_status(status)
    assert torch.equal(mass.nan_to_num(-1), kept.nan_to_num(-1))
    _check(c, out, mass_out, lens, new, kv_heads, group, dtype, 0, decay, scale)
    empty = [b for b, n in enumerate(lens) if n == 0]
    assert not out[empty].any()
    # in place, and the attention alone, which it equals up to the normaliser's rounding
    again, inplace = ops.dense_decode_mass(q.to(dev), d["kv_cache"], d["kv_indices"], indptr, d["kv_last_page_len"], most, mass,
                                           decay, scale, status=status, view=view)
    assert inplace is mass and torch.equal(again, out) and torch.equal(mass.nan_to_num(-1), mass_out.nan_to_num(-1))


@pytest.mark.parametrize("lens, kv_heads, group, dtype, sink, padded", [case for case in DECODE if case[0] != [20000]])
def test_decode_with_a_bound_far_above_the_lists(cuda_device, lens, kv_heads, group, dtype, sink, padded):
    # the form whose scores go to memory, of the same lists
    from kinetics_b200 import ops
    dev, new = cuda_device, [1 if n else 0 for n in lens]
    c = _case(4, lens, new, kv_heads, group, dtype, sink, rows=len(lens) + 3)
    c["q_indptr"] = torch.arange(len(lens) + 1, dtype=torch.int32)
    q = torch.zeros(len(lens), kv_heads * group, D, dtype=dtype)
    q[[b for b, w in enumerate(new) if w]] = c["q"]
    c["q"] = q
    d, view, status = to_dev(c["st"], dev), _view(c, lens, sink, dev, padded), ops.new_status(dev)
    bound = 8000 if len(lens) < 10 else 1500
    if dtype == torch.float32:
        bound = 100000 // group
    assert ops.decode_mass_workspace_bytes(len(lens), kv_heads, group, bound, dtype) > 0
    indptr = d["kv_indptr"][:-1].contiguous() if padded else d["kv_indptr"]
    out, mass_out = ops.dense_decode_mass(q.to(dev), d["kv_cache"], d["kv_indices"], indptr, d["kv_last_page_len"], bound, c["mass"].to(dev),
                                          0.75, D ** -0.5, status=status, view=view)
    ops.raise_on_status(status)
    _check(c, out, mass_out, lens, new, kv_heads, group, dtype, 0, 0.75, D ** -0.5)
    assert not out[[b for b, n in enumerate(lens) if n == 0]].any()


PREFILL = [
    # tokens in all, new ones, kv heads, group, dtype, window, sink page, page counts
    ([1], [1], 1, 1, torch.bfloat16, 0, 0, False),
    ([17, 16, 5], [1, 16, 3], 2, 2, torch.bfloat16, 0, 0, False),
    ([700], [700], 2, 4, torch.bfloat16, 0, 0, False),
    ([700], [700], 1, 8, torch.bfloat16, 33, 0, False),
    ([2560], [512], 1, 4, torch.bfloat16, 64, 0, False),
    ([500, 40, 0, 333, 129], [100, 40, 0, 1, 128], 2, 4, torch.bfloat16, 0, 0, False),
    ([500, 40, 7, 333, 129], [100, 40, 0, 1, 128], 2, 4, torch.bfloat16, 20, 0, True),
    ([300, 4, 21, 3, 150], [130, 4, 1, 3, 150], 2, 2, torch.bfloat16, 0, 4, True),
    ([300, 4, 21], [130, 1, 20], 2, 1, torch.bfloat16, 7, 4, False),
    ([1500], [1100], 1, 1, torch.bfloat16, 0, 0, False),
    # few tokens behind many: blocks of keys are shared among CTAs
    ([6000], [3], 1, 4, torch.bfloat16, 0, 0, False),
    ([2049, 700, 64, 1, 130], [70, 1, 33, 1, 2], 1, 8, torch.bfloat16, 5, 0, False),
    ([4100, 3000, 260], [140, 64, 260], 2, 2, torch.bfloat16, 0, 12, True),
    ([1111], [300], 1, 1, torch.bfloat16, 0, 0, False),
    ([1], [1], 1, 1, torch.float32, 0, 0, False),
    ([140, 75, 9], [40, 75, 0], 2, 4, torch.float32, 0, 0, False),
    ([140, 75, 20], [40, 75, 1], 1, 2, torch.float32, 9, 4, True),
    ([900, 1, 33, 32, 0, 97], [5, 1, 2, 32, 0, 97], 2, 1, torch.float32, 0, 0, False),
    ([700, 64, 300], [9, 8, 130], 1, 8, torch.float32, 30, 12, True),
    ([300] * 40, [70] * 40, 3, 4, torch.float32, 0, 0, False),
]


@pytest.mark.parametrize("lens, new, kv_heads, group, dtype, window, sink, padded", PREFILL)
def test_prefill_accumulates(cuda_device, lens, new, kv_heads, group, dtype, window, sink, padded):
    from kinetics_b200 import ops
    dev = cuda_device
    c = _case(5, lens, new, kv_heads, group, dtype, sink, rows=len(lens) + 2)
    d, view, status = to_dev(c["st"], dev), _view(c, lens, sink, dev, padded), ops.new_status(dev)
    scale, decay = D ** -0.5, 0.75
    indptr = d["kv_indptr"][:-1].contiguous() if padded else d["kv_indptr"]
    mass = c["mass"].to(dev)
    table = (d["kv_cache"], d["kv_indices"], indptr, d["kv_last_page_len"])
    q, q_indptr = c["q"].to(dev), c["q_indptr"].to(dev)
    out, mass_out = ops.prefill_attention_mass(q, q_indptr, max(new), *table, mass, window, decay, scale, mass_out=mass.clone(),
                                               status=status, view=view)
    ops.raise_on_status(status)
    _check(c, out, mass_out, lens, new, kv_heads, group, dtype, window, decay, scale)
    _, inplace = ops.prefill_attention_mass(q, q_indptr, max(new), *table, mass, window, decay, scale, status=status, view=view)
    assert inplace is mass and torch.equal(mass.nan_to_num(-1), mass_out.nan_to_num(-1))


def _evict_case(seed, lens, kv_heads, dtype, sink_page, keep, stored, odd):
    """Caches of random contents, masses with ties (and, odd, what no sum of weights should be), positions of earlier evictions."""
    g = torch.Generator().manual_seed(seed)
    batch, longest = len(lens), max(max(lens), 1)
    k, v = (torch.randn(batch, kv_heads, longest, D, generator=g) for _ in range(2))
    st = paged_state(k, v, lens, dtype, seed=seed, sink=sink_page, fill=0.5)
    rows, stride = batch + 2, longest + 3
    slots = torch.randperm(rows, generator=g)[:batch].to(torch.int32)
    mass = torch.randint(0, 40, (rows, kv_heads, stride), generator=g).float() / 8
    mass = torch.where(torch.rand(mass.shape, generator=g) < 0.5, mass, torch.rand(mass.shape, generator=g))
    if odd:
        for value in (math.nan, math.inf, -math.inf, -0.0, 1e-42):
            mass[torch.rand(mass.shape, generator=g) < 0.06] = value
    positions = torch.zeros(rows, kv_heads, stride, dtype=torch.int32)
    known, seen = torch.zeros(rows, dtype=torch.int32), torch.zeros(rows, dtype=torch.int32)
    for b, n in enumerate(lens):
        r, s = int(slots[b]), min(stored, n)
        known[r] = s
        seen[r] = 3 * s + n - s
        for h in range(kv_heads):
            positions[r, h, :s] = torch.randperm(3 * s, generator=g)[:s].to(torch.int32)
    return dict(st=st, slots=slots, mass=mass, positions=positions, stored=known, seen=seen)


EVICT = [
    # lengths, kv heads, dtype, keep, sink, recent, stored, sink page, page counts, odd masses
    ([1], 1, torch.bfloat16, 1, 0, 0, 0, 0, False, False),
    ([2], 1, torch.bfloat16, 1, 0, 0, 0, 0, False, False),
    ([2, 1, 0, 5], 2, torch.bfloat16, 2, 1, 1, 1, 0, False, False),
    ([2049], 8, torch.bfloat16, 2048, 4, 256, 1800, 0, False, False),
    ([700, 333, 150, 334, 0, 701], 4, torch.float32, 333, 4, 40, 300, 0, False, True),
    ([700, 333, 150, 334, 0, 701], 4, torch.bfloat16, 333, 4, 40, 300, 0, True, True),
    ([500, 37, 70], 3, torch.bfloat16, 32, 0, 32, 0, 0, False, False),
    ([500, 37, 70], 3, torch.bfloat16, 33, 33, 0, 20, 4, True, True),
    ([5000, 3], 2, torch.bfloat16, 1000, 4, 100, 0, 0, False, True),
    ([9000], 1, torch.float32, 4500, 4, 1000, 4000, 0, False, False),
    ([70000], 1, torch.bfloat16, 4096, 4, 512, 0, 0, False, True),
    ([31, 32, 33, 64, 65], 1, torch.bfloat16, 31, 2, 3, 7, 0, False, True),
    ([40, 33, 31], 3, torch.float32, 32, 2, 3, 7, 0, False, True),
    ([5040] + [100] * 39, 2, torch.bfloat16, 5000, 4, 100, 0, 0, False, True),
    ([5040] + [100] * 39, 2, torch.float32, 4000, 4, 100, 2000, 0, False, True),
]


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("lens, kv_heads, dtype, keep, sink, recent, stored, sink_page, padded, odd", EVICT)
def test_evict(cuda_device, lens, kv_heads, dtype, keep, sink, recent, stored, sink_page, padded, odd, inplace):
    c = _evict_case(7, lens, kv_heads, dtype, sink_page, keep, stored, odd)
    _evict_equals(c, cuda_device, lens, kv_heads, keep, sink, recent, sink_page, padded, inplace)


MASSES = {
    "zeros": lambda u: torch.zeros_like(u),
    "equal": lambda u: torch.full_like(u, 0.37),
    "two": lambda u: torch.where(u < 0.4, 0.5, 0.25),
    "near": lambda u: 1.0 + torch.floor(u * 3000) * 2.0 ** -23,               # neighbours
    "octaves": lambda u: torch.exp2(250 * u - 126),
    "small": lambda u: u * 1e-39,                                             # below the normal numbers
    "negative": lambda u: -torch.exp2(40 * u - 20),
    "mixed": lambda u: torch.where(u < 0.5, -u, torch.where(u < 0.6, torch.zeros_like(u), torch.exp2(20 * u))),
    "infinite": lambda u: torch.where(u < 0.3, math.inf, torch.where(u < 0.6, -math.inf, u)),
    "none": lambda u: torch.full_like(u, math.nan),
}


@pytest.mark.parametrize("lens, keep", [([700, 300, 257], 256), ([5000, 1100], 1000), ([40000], 3000), ([66000], 700)])
@pytest.mark.parametrize("masses", sorted(MASSES))
def test_evict_by_masses_of_any_range(cuda_device, masses, lens, keep):
    c = _evict_case(8, lens, 1, torch.bfloat16, 0, keep, 0, False)
    c["mass"] = MASSES[masses](torch.rand(c["mass"].shape, generator=torch.Generator().manual_seed(9)))
    _evict_equals(c, cuda_device, lens, 1, keep, 2, 3, 0, False, True)


def _evict_equals(c, dev, lens, kv_heads, keep, sink, recent, sink_page, padded, inplace):
    from kinetics_b200 import ops
    st = c["st"]
    want_kv, want_mass, want_pos = st["kv_cache"].clone(), c["mass"].clone(), c["positions"].clone()
    moved = False
    for b, n in enumerate(lens):
        r, first = int(c["slots"][b]), int(st["kv_indptr"][b])
        s, seen = int(c["stored"][r]), int(c["seen"][r])
        page_of = lambda ts: (st["kv_indices"][[first + place(t, sink_page)[0] for t in ts]].long(), torch.tensor([place(t, sink_page)[1] for t in ts]))
        for h in range(kv_heads):
            position = np.concatenate([c["positions"][r, h, :s].numpy(), np.arange(seen - n + s, seen)])
            after = np.arange(min(n, keep))
            if n > keep:
                source, hole = evict_moves(evict_order(c["mass"][r, h, :n].numpy(), position, seen, keep, sink, recent), keep)
                after[hole] = source
                moved |= len(hole) > 0
                if len(hole):
                    (sp, ss), (dp, ds) = page_of(source.tolist()), page_of(hole.tolist())
                    want_kv[dp, :, ds, h] = st["kv_cache"][sp, :, ss, h]
            want_mass[r, h, :len(after)] = c["mass"][r, h, torch.from_numpy(after)]
            want_pos[r, h, :len(after)] = torch.from_numpy(position[after]).to(torch.int32)
    assert moved == any(n > keep for n in lens) or keep <= 2
    d, view, status = to_dev(st, dev), _view(c, lens, sink_page, dev, padded), ops.new_status(dev)
    indptr = d["kv_indptr"][:-1].contiguous() if padded else d["kv_indptr"]
    mass, positions = c["mass"].to(dev), c["positions"].to(dev)
    outs = {} if inplace else dict(mass_out=mass.clone(), positions_out=positions.clone())
    got_mass, got_pos = ops.evict(d["kv_cache"], d["kv_indices"], indptr, d["kv_last_page_len"], max(max(st["npages"]), 1), mass, positions,
                                  c["stored"].to(dev), c["seen"].to(dev), keep, sink, recent, status=status, view=view, **outs)
    ops.raise_on_status(status)
    assert (got_mass is mass) == inplace
    assert torch.equal(d["kv_cache"].cpu(), want_kv)
    assert torch.equal(got_pos.cpu(), want_pos)
    assert torch.equal(got_mass.cpu().view(torch.int32), want_mass.view(torch.int32))
    if not inplace:
        assert torch.equal(mass.cpu().view(torch.int32), c["mass"].view(torch.int32)) and torch.equal(positions.cpu(), c["positions"])
