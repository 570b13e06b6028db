"""The operators of a bounded cache at their limits: batches that shrink under a manager, sequences beyond a call's bounds, pages that are
none, host threads; against plain fp64 forms."""
import threading

import numpy as np
import pytest
import torch

from helpers import paged_state, to_dev
from mass_helpers import attend, mass_after

pytestmark = pytest.mark.gpu
D = 128


def _lists(seed, device, lens, kv_heads, group, dtype, padded, new=None):
    """Sequences of `lens` tokens whose last `new` (None: one each) have queries, in row b of the masses sequence b; the page table packed
    or with page counts."""
    from kinetics_b200 import ops
    g = torch.Generator().manual_seed(seed)
    new = new or [1] * len(lens)
    cast = lambda t: t.to(dtype).float()
    k, v = (cast(torch.randn(len(lens), kv_heads, max(lens), D, generator=g)) for _ in range(2))
    q = cast(1.3 * torch.randn(sum(new), kv_heads * group, D, generator=g))
    st = paged_state(k, v, lens, dtype, seed=seed, fill=0.5)
    d = to_dev(st, device)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    view = ops.PageView(0, 0, i32(st["npages"]) if padded else None, i32(range(len(lens))))
    starts = d["kv_indptr"][:-1].contiguous() if padded else d["kv_indptr"]
    mass = torch.rand(len(lens), kv_heads, max(lens) + 3, generator=g)
    return dict(k=k, v=v, q=q, mass=mass, lens=lens, new=new, group=group, dtype=dtype, view=view, pages=st["npages"], first=st["kv_indptr"].tolist(),
                table=[d["kv_cache"], d["kv_indices"], starts, d["kv_last_page_len"]], indptr=i32(np.concatenate([[0], np.cumsum(new)]).tolist()))


def _equals(c, b, out, mass, window, decay, without=None):
    """Outputs and masses of sequence b are those of the fp64 form, with the tokens `without` taking no part."""
    n, w, G = c["lens"][b], c["new"][b], c["group"]
    part = np.setdiff1d(np.arange(n), [] if without is None else without)
    first = sum(c["new"][:b])
    for h in range(c["k"].shape[1]):
        q = c["q"][first:first + w, h * G:(h + 1) * G]
        o, o_bound, some, some_bound = attend(q, c["k"][b, h, part], c["v"][b, h, part], w, window, D ** -0.5, c["dtype"])
        err = (out[first:first + w, h * G:(h + 1) * G].double().cpu() - o).abs()
        assert bool((err <= o_bound).all()), (b, h, float((err / o_bound).max()))
        paid, bound = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64)
        paid[part], bound[part] = some, some_bound
        want, more = mass_after(c["mass"], b, n, w, h, decay, paid)
        err = (mass[b, h, :n].double().cpu() - want).abs()
        assert bool((err <= bound + more).all()), (b, h, float((err - bound - more).max()))
        assert torch.equal(mass[b, h, n:].cpu(), c["mass"][b, h, n:])


# ---------------------------------------------------------------- a manager whose batch shrinks
class Cfg:
    hidden_size = 4096
    num_attention_heads = 32
    num_key_value_heads = 8
    head_dim = 128
    num_hidden_layers = 1


@pytest.mark.parametrize("dtype, active", [(torch.bfloat16, (16, 10, 16, 10, 3)), (torch.float32, (16, 4, 7, 1, 2))])
def test_a_manager_of_sixteen_slots_with_fewer_active(cuda_device, dtype, active):
    from kinetics_b200 import EvictingKVManager
    kv = EvictingKVManager(Cfg, 16, 4096, cuda_device, dtype, keep=2000)
    g = torch.Generator().manual_seed(31)
    keys, values = ([torch.zeros(0, 8, D) for _ in range(16)] for _ in range(2))
    for n in active:
        slots = torch.randperm(16, generator=g)[:n].tolist()
        q, k, v = (torch.randn(n, heads, 1, D, generator=g).to(dtype) for heads in (32, 8, 8))
        kv.begin_step(slots)
        out = kv.compute_attention(*(t.to(cuda_device) for t in (q, k, v)), 0, torch.tensor(slots, device=cuda_device)).view(n, 32, D)
        for i, s in enumerate(slots):
            keys[s], values[s] = torch.cat((keys[s], k[i].float().transpose(0, 1))), torch.cat((values[s], v[i].float().transpose(0, 1)))
            for h in range(8):
                o, bound, _, _ = attend(q[i, 4 * h:4 * h + 4].float().transpose(0, 1), keys[s][:, h], values[s][:, h], 1, 0, D ** -0.5, dtype)
                err = (out[i, 4 * h:4 * h + 4].double().cpu() - o[0]).abs()
                assert bool((err <= bound[0]).all()), (n, s, h)
    kv.check_status()


def test_an_engine_that_drains_its_slots(cuda_device):
    # requests of different lengths end one after the other: every number of active sequences from 16 down to 1
    from kinetics_b200 import DecoderStack, Engine, EvictingKVManager
    from kinetics_b200.config import LayerConfig
    cfg, dtype = LayerConfig(hidden_size=256, num_attention_heads=8, num_key_value_heads=4, intermediate_size=512, num_hidden_layers=2,
                             vocab_size=503), torch.float32
    g = torch.Generator().manual_seed(32)
    kv = EvictingKVManager(cfg, 16, 400, cuda_device, dtype, keep=2000)
    eng = Engine(DecoderStack(cfg, cuda_device, dtype, max_positions=400, seed=3), kv, 400, cuda_device, temperature=0.0, repeat_check=False)
    prompts = [torch.randint(0, 500, (1, 2 + i), generator=g) for i in range(16)]
    for slot, p in enumerate(prompts):
        eng.prefill(slot, p, 40)
    for n in range(16, 0, -1):
        eng.decode(list(range(n)))
        if n % 3 == 0:
            for _ in range(3):                                          # eager, captured, replayed
                eng.decode_graphed(list(range(n)))
    kv.check_status()
    assert kv.cached(0) == 2 + 16 + 15


# ---------------------------------------------------------------- beyond a call's bounds
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [(300, 340), (2500, 3000)])             # a CTA per tile, CTAs that share the keys
@pytest.mark.parametrize("indptr, good", [((0, 33, 133), 0), ((-7, 33, 73), 1), ((0, 33, 2 ** 31 - 1), 0)])
def test_new_tokens_outside_the_queries_are_not_touched(cuda_device, indptr, good, lens, dtype):
    from kinetics_b200 import _lib, ops
    c, status = _lists(47, cuda_device, list(lens), 2, 4, dtype, False, new=[33, 40]), ops.new_status(cuda_device)
    # outputs and workspace in the middle of more, which has to stay
    rows = torch.full((73 + 400, 8, D), 7.0, dtype=dtype, device=cuda_device)
    out = rows[200:273]
    pages = min(c["mass"].shape[2] // 16 + 2, sum(c["pages"]))
    shape = _lib.Shape(2, 2, 4, D, 16, 1 if dtype == torch.bfloat16 else 0, 0)
    need = _lib.load().ktk_prefill_mass_workspace_bytes(shape, 73, 40, pages, sum(c["pages"]), 0)
    space = torch.full((need + 2 ** 18,), 0x5a, dtype=torch.uint8, device=cuda_device)
    at = 2 ** 17
    _, mass = ops.prefill_attention_mass(c["q"].to(dtype).to(cuda_device), torch.tensor(indptr, dtype=torch.int32, device=cuda_device), 40,
                                         *c["table"], c["mass"].to(cuda_device), 0, 0.75, out=out, workspace=space[at:at + need], status=status,
                                         view=c["view"])
    assert int(status.item()) == 2 and torch.equal(mass[1 - good].cpu(), c["mass"][1 - good])
    assert bool((rows[:200] == 7).all()) and bool((rows[273:] == 7).all())
    assert bool((space[:at] == 0x5a).all()) and bool((space[at + need:] == 0x5a).all())
    _equals(c, good, out, mass, 0, 0.75)


BEYOND = [(700, 30, 2), (8100, 500, 1)]            # tokens of the long list, bound in pages, kv heads: by clusters, with scores in memory


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("long, most, kv_heads", BEYOND)
def test_a_list_beyond_the_bound_leaves_the_others_alone(cuda_device, long, most, kv_heads, padded, dtype):
    from kinetics_b200 import ops
    c, status = _lists(41, cuda_device, [300, long, 90, 5], kv_heads, 4, dtype, padded), ops.new_status(cuda_device)
    assert c["pages"][1] > most and (ops.decode_mass_workspace_bytes(4, kv_heads, 4, most, dtype) > 0) == (most > 30)
    for _ in range(4):
        out, mass = ops.dense_decode_mass(c["q"].to(dtype).to(cuda_device), *c["table"], most, c["mass"].to(cuda_device), 0.75, status=status,
                                          view=c["view"])
        assert int(status.item()) == 2
        for b in (0, 2, 3):
            _equals(c, b, out, mass, 0, 0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_new_tokens_than_the_bound_where_portions_go_by_length(cuda_device, dtype):
    # the portion of 600 has the most keys; the two within the bound of 40 are attended and counted as ever
    from kinetics_b200 import ops
    c, status = _lists(43, cuda_device, [660, 340, 140], 4, 8, dtype, False, new=[600, 40, 40]), ops.new_status(cuda_device)
    q = c["q"].to(dtype).to(cuda_device)
    out, mass = ops.prefill_attention_mass(q, c["indptr"], 40, *c["table"], c["mass"].to(cuda_device), 0, 0.75,
                                           out=torch.full_like(q, float("nan")), status=status, view=c["view"])
    assert int(status.item()) == 2 and torch.equal(mass[0].cpu(), c["mass"][0])
    for b in (1, 2):
        _equals(c, b, out, mass, 0, 0.75)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("long, most, kv_heads", BEYOND)
def test_a_list_beyond_the_bound_keeps_its_masses(cuda_device, long, most, kv_heads, padded, dtype):
    from kinetics_b200 import ops
    c, status = _lists(42, cuda_device, [300, long, 90], kv_heads, 4, dtype, padded), ops.new_status(cuda_device)
    _, mass = ops.dense_decode_mass(c["q"].to(dtype).to(cuda_device), *c["table"], most, c["mass"].to(cuda_device), 0.75, status=status,
                                    view=c["view"])
    assert int(status.item()) == 2 and torch.equal(mass[1].cpu(), c["mass"][1])


def test_starts_that_do_not_ascend_are_refused(cuda_device):
    # balanced partition: the list of sequence 0 passes the end that the table gives for all
    from kinetics_b200 import ops
    c, status = _lists(48, cuda_device, [16000, 640], 2, 4, torch.bfloat16, False), ops.new_status(cuda_device)
    assert c["first"] == [0, 1000, 1040] and ops.decode_mass_workspace_bytes(2, 2, 4, 8000, torch.bfloat16) > 0
    c["table"][2][2] = 40
    _, mass = ops.dense_decode_mass(c["q"].to(torch.bfloat16).to(cuda_device), *c["table"], 8000, c["mass"].to(cuda_device), 0.75, status=status,
                                    view=c["view"])
    assert int(status.item()) == 2 and torch.equal(mass.cpu(), c["mass"])

@pytest.mark.parametrize("window", [0, 20])                              # parts of the rows that are added, one part
def test_lists_beyond_the_bound_of_all_keep_their_masses(cuda_device, window):
    # eleven groups of sixteen pages where there are three, ten and ten: no sequence is counted in part
    from kinetics_b200 import _lib
    c, status = _lists(52, cuda_device, [700, 2400, 2400], 2, 8, torch.bfloat16, False, new=[5, 600, 40]), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    q, lib = c["q"].to(torch.bfloat16).to(cuda_device), _lib.load()
    shape, most, total = _lib.Shape(3, 2, 8, D, 16, 1, c["table"][0].shape[0]), 150, 130
    space = torch.empty(lib.ktk_prefill_mass_workspace_bytes(shape, 645, 600, most, total, window), dtype=torch.uint8, device=cuda_device)
    mass, out = c["mass"].to(cuda_device), torch.empty_like(q)
    view = c["view"].c()
    assert lib.ktk_prefill_attention_mass(
        q.data_ptr(), c["indptr"].data_ptr(), 645, 600, *(t.data_ptr() for t in c["table"]), view, most, total, window, D ** -0.5,
        _lib.Mass(mass.data_ptr(), mass.data_ptr(), mass.shape[2], 3, 0.75), out.data_ptr(), space.data_ptr(), space.nbytes, shape, status.data_ptr(),
        torch.cuda.current_stream().cuda_stream) == 0
    assert int(status.item()) == 2 and torch.equal(mass[1:].cpu(), c["mass"][1:])
    _equals(c, 0, out, mass, window, 0.75)


# ---------------------------------------------------------------- pages that are none
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("group", [1, 4, 8])
@pytest.mark.parametrize("most", [0, 8000])
def test_tokens_of_a_page_that_is_none_take_no_part(cuda_device, most, group, dtype):
    # pages 2 and 17 of sequence 1; in the masses their tokens' are decayed, as those that were paid nothing
    from kinetics_b200 import ops
    c = _lists(44, cuda_device, [300, 700, 90], 2, group, dtype, False)
    if most and dtype == torch.float32:
        most = 100000 // group
    assert (ops.decode_mass_workspace_bytes(3, 2, group, most or max(c["pages"]), dtype) > 0) == (most > 0)
    for page, none in ((2, -1), (17, c["table"][0].shape[0])):
        c["table"][1][c["first"][1] + page] = none
    without = np.concatenate([np.arange(32, 48), np.arange(17 * 16, 18 * 16)])
    status, q = ops.new_status(cuda_device), c["q"].to(dtype).to(cuda_device)
    # what a page's scores may find in their places: those of an earlier call, or NaN
    need = ops.decode_mass_workspace_bytes(3, 2, group, most or max(c["pages"]), dtype)
    workspace = torch.full((max(need, 16) // 4,), float("nan"), device=cuda_device)
    for _ in range(3):
        out, mass = ops.dense_decode_mass(q, *c["table"], most or max(c["pages"]), c["mass"].to(cuda_device), 0.75, workspace=workspace,
                                          status=status, view=c["view"])
        assert int(status.item()) == 1
        for b in range(3):
            _equals(c, b, out, mass, 0, 0.75, without if b == 1 else None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("most", [0, 8000])
def test_a_list_whose_pages_are_all_none(cuda_device, most, dtype):
    from kinetics_b200 import ops
    c, status = _lists(49, cuda_device, [300, 700, 90], 2, 4, dtype, False), ops.new_status(cuda_device)
    if most and dtype == torch.float32:
        most = 25000
    c["table"][1][c["first"][1]:c["first"][2]] = -1
    out, mass = ops.dense_decode_mass(c["q"].to(dtype).to(cuda_device), *c["table"], most or max(c["pages"]), c["mass"].to(cuda_device), 0.75,
                                      status=status, view=c["view"])
    assert int(status.item()) == 1 and not out[1].any()
    want = 0.75 * c["mass"][1]
    want[:, 699] = 0                                                     # the newest starts from its weights alone
    want[:, 700:] = c["mass"][1, :, 700:]
    assert torch.equal(mass[1].cpu(), want)
    for b in (0, 2):
        _equals(c, b, out, mass, 0, 0.75)


# ---------------------------------------------------------------- host threads
def _together(calls, rounds):
    """Each call(stream), which returns 0 or an error's code, `rounds` times in a thread and a stream of its own; the errors."""
    from kinetics_b200 import _lib
    errors, start = [], threading.Barrier(len(calls))

    def work(call):
        torch.cuda.set_device(0)
        stream = torch.cuda.Stream()
        start.wait()
        for i in range(rounds):
            if call(stream.cuda_stream) != 0:
                errors.append((i, _lib.load().ktk_last_error()))
                return
            if i % 500 == 499:
                stream.synchronize()
    workers = [threading.Thread(target=work, args=(call,)) for call in calls]
    torch.cuda.synchronize()
    for t in workers:
        t.start()
    for t in workers:
        t.join()
    torch.cuda.synchronize()
    return errors


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_threads_whose_lists_have_other_bounds(cuda_device, dtype):
    # the same kernels with other amounts of shared memory at once
    from kinetics_b200 import _lib, ops
    lens, heads, group = ([90, 33], 2, 4) if dtype == torch.bfloat16 else ([90, 33, 1, 2, 3, 4, 5, 6], 8, 8)
    c = _lists(45, cuda_device, lens, heads, group, dtype, False)
    cache, indices, starts, last = c["table"]
    q = c["q"].to(dtype).to(cuda_device)
    shape = _lib.Shape(len(lens), heads, group, D, 16, 1 if dtype == torch.bfloat16 else 0, cache.shape[0])
    bounds = (8, 400, 60, 300) if dtype == torch.bfloat16 else (200, 2500, 1200, 1900)
    call, kept = _lib.load().ktk_dense_decode_mass, []

    def of(most):
        mass, out = c["mass"].to(cuda_device), torch.empty_like(q)
        need = ops.decode_mass_workspace_bytes(len(lens), heads, group, most, dtype)
        assert need == 0
        m = _lib.Mass(mass.data_ptr(), mass.data_ptr(), mass.shape[2], len(lens), 1.0)
        kept.append((mass, out, m))
        args = (q.data_ptr(), cache.data_ptr(), indices.data_ptr(), starts.data_ptr(), last.data_ptr(), None, most, -1, 0.1, m, out.data_ptr(), 0, 0,
                shape, 0)
        return lambda stream: call(*args, stream)
    assert _together([of(most) for most in bounds], 10000) == []


def test_threads_that_evict_from_lists_of_other_bounds(cuda_device):
    from kinetics_b200 import _lib, ops
    c = _lists(46, cuda_device, [90, 33], 2, 4, torch.bfloat16, False)
    shape = _lib.Shape(2, 2, 1, D, 16, 1, c["table"][0].shape[0])
    seen, stored = torch.tensor([90, 33], dtype=torch.int32, device=cuda_device), torch.zeros(2, dtype=torch.int32, device=cuda_device)
    call, kept = _lib.load().ktk_evict, []

    def of(most):
        cache, mass = c["table"][0].clone(), c["mass"].to(cuda_device)
        positions = torch.zeros(mass.shape, dtype=torch.int32, device=cuda_device)
        space = torch.empty(_lib.load().ktk_evict_workspace_bytes(shape, most, 64), dtype=torch.uint8, device=cuda_device)
        m = _lib.Mass(mass.data_ptr(), mass.data_ptr(), mass.shape[2], 2, 1.0)
        kept.append((cache, mass, positions, space, m))
        args = (cache.data_ptr(), *(t.data_ptr() for t in c["table"][1:]), None, most, m, positions.data_ptr(), positions.data_ptr(), stored.data_ptr(),
                seen.data_ptr(), 64, 4, 0, space.data_ptr(), space.nbytes, shape, 0)
        return lambda stream: call(*args, stream)
    assert _together([of(most) for most in (4200, 32768, 9000)], 5000) == []


def test_calls_by_the_public_names_of_torch(cuda_device, monkeypatch):
    # what stands in for the private names where a torch lacks them: the same results, on a stream of their own and captured
    from kinetics_b200 import ops
    c, status = _lists(50, cuda_device, [300, 8100, 90], 1, 4, torch.bfloat16, False), ops.new_status(cuda_device)
    q, most = c["q"].to(torch.bfloat16).to(cuda_device), max(c["pages"])
    assert ops.decode_mass_workspace_bytes(3, 1, 4, most) > 0
    call = lambda: ops.dense_decode_mass(q, *c["table"], most, c["mass"].to(cuda_device), 0.75, status=status, view=c["view"])
    want = call()
    monkeypatch.setattr(ops, "_current_device", torch.cuda.current_device)
    monkeypatch.setattr(ops, "_current_stream", lambda dev: torch.cuda.current_stream(dev).cuda_stream)
    monkeypatch.setattr(ops, "_take", lambda size, stream: torch.cuda.caching_allocator_alloc(size, None, stream))
    monkeypatch.setattr(ops, "_give_back", torch.cuda.caching_allocator_delete)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    mass, graph = c["mass"].to(cuda_device), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.dense_decode_mass(q, *c["table"], most, mass, 0.75, mass_out=torch.empty_like(mass), status=status, view=c["view"])
    got[1].copy_(mass)
    graph.replay()
    ops.raise_on_status(status)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_prompt_behind_more_than_2_28_tokens(cuda_device):
    """Rows are counted in (token, head) pairs: eight heads behind 2^28 tokens pass 31 bits.  The cache is five pages, listed over and over.
    A weight's error: the denominators add 2^18 blocks of keys a CTA, half a step of 2^-23 of their sum each (2^-6); the rest is below 2^-10."""
    from kinetics_b200 import ops
    g = torch.Generator().manual_seed(51)
    n, G = 2 ** 28 + 40, 8
    kv = (0.3 * torch.randn(5, 2, 16, 1, D, generator=g)).to(torch.bfloat16)
    q = torch.randn(1, G, D, generator=g).to(torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    pages, status = (n + 15) // 16, ops.new_status(cuda_device)
    indices = torch.arange(pages, device=cuda_device, dtype=torch.int32) % 5
    mass = torch.zeros(1, 1, n + 8, device=cuda_device)
    ops.prefill_attention_mass(q.to(cuda_device), i32(0, 1), 1, kv.to(cuda_device), indices, i32(0, pages), i32(n - 16 * (pages - 1)), mass, status=status)
    ops.raise_on_status(status)
    # the 80 tokens of the five pages, each listed `often` times
    score = torch.einsum("gd,td->gt", q[0].double(), kv[:, 0, :, 0].reshape(80, D).double()) * D ** -0.5
    often = torch.full((80,), n // 80, dtype=torch.float64)
    often[:n % 80] += 1
    weight = score.exp()
    want = (weight / (weight * often).sum(1, keepdim=True)).sum(0).to(cuda_device)
    for first in range(0, n - 80, 80 * 2 ** 20):                         # piece by piece
        got = mass[0, 0, first:min(first + 80 * 2 ** 20, n // 80 * 80)].view(-1, 80).double()
        assert bool(((got - want).abs() <= 2.0 ** -5 * want).all()), (first, float(((got - want) / want).abs().max()))
    assert not mass[0, 0, n:].any()
