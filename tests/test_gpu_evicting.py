"""The operators of a bounded cache together, as they are used: EvictingKVManager against a plain fp64 cache of lists, the engine on
it, captured steps, other streams, bad tables."""
import numpy as np
import pytest
import torch

from helpers import paged_state, to_dev
from mass_helpers import attend, evict_moves, evict_order

pytestmark = pytest.mark.gpu
D = 128


class Cfg:
    hidden_size = 1024
    num_attention_heads = 8
    num_key_value_heads = 2
    head_dim = 128
    num_hidden_layers = 2


SET = dict(keep=40, sink=4, recent=8, window=6, room=8, portion=24, decay=0.9)


class PlainCache:
    """One (layer, slot): per kv head keys, values, positions and masses in fp64, in the places that they have in the cache."""

    def __init__(self, heads, s):
        self.s = s
        self.k, self.v = (torch.zeros(heads, 0, D, dtype=torch.float64) for _ in range(2))
        self.pos, self.mass = np.zeros((heads, 0), dtype=np.int64), np.zeros((heads, 0))
        self.seen, self.margin = 0, np.inf

    def evict(self):
        n, keep = self.pos.shape[1], self.s["keep"]
        if n <= keep:
            return
        for h in range(len(self.pos)):
            stays = evict_order(self.mass[h], self.pos[h], self.seen, keep, self.s["sink"], self.s["recent"])
            free = (self.pos[h] >= self.s["sink"]) & (self.pos[h] < self.seen - self.s["recent"])
            low, high = self.mass[h][stays & free], self.mass[h][~stays]
            if len(low) and len(high):
                self.margin = min(self.margin, (low.min() - high.max()) / low.min())
            at = np.arange(n)
            source, hole = evict_moves(stays, keep)
            at[hole] = source
            self.k[h, :keep], self.v[h, :keep] = self.k[h, at[:keep]], self.v[h, at[:keep]]
            self.pos[h, :keep], self.mass[h, :keep] = self.pos[h, at[:keep]], self.mass[h, at[:keep]]
        self.k, self.v, self.pos, self.mass = self.k[:, :keep], self.v[:, :keep], self.pos[:, :keep], self.mass[:, :keep]

    def attend(self, q, k, v, window, dtype):
        """q [w, Hq, D], k, v [w, Hkv, D] -> output and its bound."""
        w, heads = k.shape[0], len(self.pos)
        group = q.shape[1] // heads
        self.k, self.v = (torch.cat((old, new.double().transpose(0, 1)), 1) for old, new in ((self.k, k), (self.v, v)))
        self.pos = np.concatenate((self.pos, np.tile(np.arange(self.seen, self.seen + w), (heads, 1))), 1)
        self.seen += w
        out, bound = torch.empty(q.shape, dtype=torch.float64), torch.empty(q.shape, dtype=torch.float64)
        self.mass = np.concatenate((self.s["decay"] * self.mass, np.zeros((heads, w))), 1)
        for h in range(heads):
            at = slice(h * group, (h + 1) * group)
            out[:, at], bound[:, at], paid, _ = attend(q[:, at], self.k[h], self.v[h], w, window, D ** -0.5, dtype)
            self.mass[h] += paid.numpy()
        return out, bound


def _drive(dtype, seed, step):
    """Prompts of 150, 30 and 1 tokens in slots 1, 0 and 3, then 45 decode steps of all; step(plain, slot, layer, q, k, v) compares.
    Returns the caches and the smallest margin of any eviction."""
    g = torch.Generator().manual_seed(seed)
    rnd = lambda heads, n: (torch.randn(n, heads, D, generator=g)).to(dtype)
    caches = {(layer, slot): PlainCache(2, SET) for layer in range(2) for slot in (0, 1, 3)}
    for slot, n in ((1, 150), (0, 30), (3, 1)):
        for layer in range(2):
            c, q, k, v = caches[layer, slot], 1.5 * rnd(8, n), rnd(2, n), rnd(2, n)
            outs, at, capacity = [], 0, SET["keep"] + max(SET["room"], SET["portion"])
            while at < n:
                m = min(n - at, SET["portion"])
                if n == 1:
                    pass
                elif c.pos.shape[1] + m > capacity:
                    c.evict()
                m = min(m, capacity - c.pos.shape[1])
                outs.append(c.attend(q[at:at + m].float(), k[at:at + m].float(), v[at:at + m].float(), SET["window"] if n > 1 else 0, dtype))
                at += m
            step([slot], layer, q[None], k[None], v[None], [tuple(torch.cat(x) for x in zip(*outs))])
    for _ in range(45):
        slots = [3, 0, 1]
        for layer in range(2):
            q, k, v = 1.5 * rnd(8, 3), rnd(2, 3), rnd(2, 3)
            want = []
            for i, slot in enumerate(slots):
                c = caches[layer, slot]
                if c.pos.shape[1] + 1 > SET["keep"] + SET["room"]:
                    c.evict()
                want.append(c.attend(q[i:i + 1].float(), k[i:i + 1].float(), v[i:i + 1].float(), 0, dtype))
            step(slots, layer, q[:, None], k[:, None], v[:, None], want)
    return caches, min(c.margin for c in caches.values())


@pytest.mark.parametrize("dtype, seed", [(torch.float32, 1), (torch.float32, 10), (torch.bfloat16, 1)])
def test_manager_equals_a_plain_cache(cuda_device, dtype, seed):
    from kinetics_b200 import EvictingKVManager
    kv = EvictingKVManager(Cfg, 5, 512, cuda_device, dtype, **SET)

    def step(slots, layer, q, k, v, want):
        to = lambda t: t.transpose(1, 2).to(cuda_device)                # [B, heads, tokens, D]
        kv.begin_step(slots)
        out = kv.compute_attention(to(q), to(k), to(v), layer, torch.tensor(slots, device=cuda_device))
        for i, (o, bound) in enumerate(want):
            err = (out[i].view(o.shape).double().cpu() - o).abs()
            assert bool((err <= bound).all()), float((err / bound).max())

    caches, margin = _drive(dtype, seed, step)
    # the eviction's order is that of the fp64 masses: no two are nearer than a thousand roundings of fp32 (the bounds of the weights
    # themselves are near 2e-4 of them)
    assert margin > 1e-3, margin
    for (layer, slot), c in caches.items():
        n = c.pos.shape[1]
        assert kv.cached(slot, layer) == n <= SET["keep"] + SET["room"]
        stored = int(kv._stored[layer, slot])
        assert np.array_equal(kv.positions[layer][slot, :, :stored].cpu().numpy(), c.pos[:, :stored])
        np.testing.assert_allclose(kv.mass[layer][slot, :, :n].cpu().numpy(), c.mass, rtol=1e-3, atol=1e-6)
    assert kv.evictions > 12
    kv.check_status()


def _engine(kv, cfg, device, dtype, prompts, **kw):
    from kinetics_b200 import DecoderStack, Engine
    model = DecoderStack(cfg, device, dtype, max_positions=400, seed=3)
    eng = Engine(model, kv, 400, device, temperature=0.0, repeat_check=False, **kw)
    for slot, p in enumerate(prompts):
        eng.prefill(slot, p, 100)
    return eng


def _small():
    from kinetics_b200.config import LayerConfig
    return LayerConfig(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512, num_hidden_layers=3,
                       vocab_size=503)


def test_engine_on_a_cache_that_holds_everything(cuda_device):
    # nothing is evicted: the tokens are those of the dense manager
    from kinetics_b200 import BatchKVManager, EvictingKVManager
    cfg, dtype = _small(), torch.float32
    g = torch.Generator().manual_seed(21)
    prompts = [torch.randint(0, 500, (1, n), generator=g) for n in (150, 37, 3)]
    kv = EvictingKVManager(cfg, 3, 256, cuda_device, dtype, keep=256, portion=64)
    runs = [_engine(m, cfg, cuda_device, dtype, prompts) for m in (BatchKVManager(cfg, 3, 256, cuda_device, dtype), kv)]
    for _ in range(30):
        for eng in runs:
            eng.decode([0, 1, 2])
    assert torch.equal(runs[0].slots_tokens, runs[1].slots_tokens) and kv.evictions == 0


def test_engine_generates_far_beyond_its_cache(cuda_device):
    from kinetics_b200 import EvictingKVManager
    cfg, dtype = _small(), torch.bfloat16
    g = torch.Generator().manual_seed(22)
    kv = EvictingKVManager(cfg, 2, 400, cuda_device, dtype, keep=48, recent=16, window=8, room=16, portion=32)
    from kinetics_b200 import DecoderStack, Engine
    eng = Engine(DecoderStack(cfg, cuda_device, dtype, max_positions=400, seed=3), kv, 400, cuda_device, temperature=0.0, eos=[502],
                 repeat_check=False, prefill_chunk=100)
    requests = [{"id": i, "input_ids": torch.randint(0, 500, (n,), generator=g).tolist()} for i, n in enumerate((250, 9, 120))]
    done = eng.offline_exec(requests, max_new_tokens=120)
    assert sorted(r["id"] for r in done) == [0, 1, 2] and all(1 <= len(r["output_tokens"]) <= 120 for r in done)
    kv.check_status()
    assert kv.evictions > 0 and not kv._held.any()                       # retired slots are free


def test_captured_steps_equal_eager_ones(cuda_device):
    from kinetics_b200 import EvictingKVManager
    cfg, dtype = _small(), torch.bfloat16
    g = torch.Generator().manual_seed(23)
    prompts = [torch.randint(0, 500, (1, n), generator=g) for n in (150, 37, 3)]
    # a page table of padded lists either way: the same launches, the same bits
    kvs = [EvictingKVManager(cfg, 3, 400, cuda_device, dtype, keep=48, recent=16, window=8, room=8, portion=32) for _ in range(2)]
    eager, captured = (_engine(kv, cfg, cuda_device, dtype, prompts) for kv in kvs)
    slots = [0, 1, 2]
    for step in range(40):
        eager.decode(slots)
        captured.decode_graphed(slots)
        assert torch.equal(eager.slots_tokens, captured.slots_tokens), step
    for kv in kvs:
        kv.check_status()
    assert kvs[0].evictions == kvs[1].evictions > 20
    assert np.array_equal(kvs[0]._held, kvs[1]._held)
    for layer in range(3):
        for slot in slots:
            n = kvs[0].cached(slot)
            assert torch.equal(kvs[0].mass[layer][slot, :, :n], kvs[1].mass[layer][slot, :, :n])


# ---------------------------------------------------------------- calls that overlap, captured ones, bad tables
def _state(seed, device, lens=(700, 40, 1300), kv_heads=2, group=4, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(len(lens), kv_heads, max(lens), D, generator=g) for _ in range(2))
    st = to_dev(paged_state(k, v, lens, dtype, seed=seed, fill=0.0), device)
    put = lambda *s: torch.randn(*s, generator=g).to(dtype).to(device)
    new = [33, 40, 200]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    return dict(table=(st["kv_cache"], st["kv_indices"], st["kv_indptr"], st["kv_last_page_len"]), most=max(st["npages"]),
                q=put(len(lens), kv_heads * group, D), qs=put(sum(new), kv_heads * group, D), indptr=i32(np.concatenate([[0], np.cumsum(new)]).tolist()),
                new=max(new), mass=torch.rand(len(lens), kv_heads, max(lens) + 5, generator=g).to(device),
                positions=torch.zeros(len(lens), kv_heads, max(lens) + 5, dtype=torch.int32, device=device), stored=i32([0] * len(lens)),
                seen=i32(list(lens)))


def _chain(s, status=None):
    """All three on clones of the state's cache and masses: everything that they write."""
    from kinetics_b200 import ops
    cache, mass, positions = s["table"][0].clone(), s["mass"].clone(), s["positions"].clone()
    table = (cache, *s["table"][1:])
    a, _ = ops.prefill_attention_mass(s["qs"], s["indptr"], s["new"], *table, mass, window=20, status=status)
    b, _ = ops.dense_decode_mass(s["q"], *table, s["most"], mass, decay=0.9, status=status)
    ops.evict(*table, s["most"], mass, positions, s["stored"], s["seen"], 500, 4, 64, status=status)
    return a, b, cache, mass, positions


def test_a_call_on_another_stream_and_two_at_once(cuda_device):
    from kinetics_b200 import ops
    status = ops.new_status(cuda_device)
    states = [_state(s, cuda_device) for s in (1, 2)]
    want = [_chain(s, status) for s in states]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in states]
    for _ in range(4):
        got = []
        for side, s in zip(sides, states):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append(_chain(s, status))
        torch.cuda.synchronize()
        for w, r in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(w, r))
    ops.raise_on_status(status)


def test_two_captured_chains_replayed_at_once(cuda_device):
    from kinetics_b200 import ops
    status = ops.new_status(cuda_device)
    states = [_state(s, cuda_device) for s in (3, 4)]
    want = [_chain(s, status) for s in states]
    graphs, outs = [], []
    for s in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_chain(s, status))
        graphs.append(graph)
    sides = [torch.cuda.Stream() for _ in states]
    for _ in range(4):
        for side, graph in zip(sides, graphs):
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for w, r in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(w, r))
    ops.raise_on_status(status)


def test_runs_give_the_same_bits(cuda_device):
    s = _state(5, cuda_device)
    first = _chain(s)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, _chain(s)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fault", ["page", "slot", "places", "last", "most"])
def test_bad_tables_are_reported_and_touch_nothing_else(cuda_device, dtype, fault):
    # sequence 1 of three is bad: the others' results are those of a good call, and the status word says so
    from kinetics_b200 import ops
    good, bad = (_state(6, cuda_device, lens=(300, 700, 90), dtype=dtype) for _ in range(2))
    for s in (good, bad):
        s["view"] = ops.PageView(0, 0, None, torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda_device))
    new = [33, 40, 20]
    for s in (good, bad):
        s["indptr"] = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=cuda_device)
        s["qs"], s["new"] = s["qs"][:sum(new)].contiguous(), max(new)
    want_codes = {2}
    if fault == "page":
        bad["table"][1][19 + 43] = bad["table"][0].shape[0] + 3          # behind sequence 0's 19 pages; the newest tokens, which stay
        want_codes = {1}
    elif fault == "slot":
        bad["view"] = ops.PageView(0, 0, None, torch.tensor([0, 9, 2], dtype=torch.int32, device=cuda_device))
    elif fault == "places":
        for s in (good, bad):
            s["mass"], s["positions"] = s["mass"][:, :, :600].contiguous(), s["positions"][:, :, :600].contiguous()
    elif fault == "last":
        bad["table"][3][1] = 17
    elif fault == "most":
        bad["most"] = 30                                                 # 44 pages
    if fault == "places":                                                # a good call has no long sequence
        good = _state(6, cuda_device, lens=(300, 700, 90), dtype=dtype)
        good["view"], good["indptr"], good["qs"], good["new"] = bad["view"], bad["indptr"], bad["qs"], bad["new"]

    def run(s, which):
        status, cache, mass, positions = ops.new_status(cuda_device), s["table"][0].clone(), s["mass"].clone(), s["positions"].clone()
        table = (cache, *s["table"][1:])
        if which == "decode":
            out, _ = ops.dense_decode_mass(s["q"], *table, s["most"], mass, status=status, view=s["view"])
        elif which == "prefill":
            out, _ = ops.prefill_attention_mass(s["qs"], s["indptr"], s["new"], *table, mass, window=20, status=status, view=s["view"])
        else:
            out = cache
            ops.evict(*table, s["most"], mass, positions, s["stored"], s["seen"], 64, 4, 16, status=status, view=s["view"])
        return int(status.item()), out, mass, positions
    for which in ("decode", "prefill", "evict"):
        if fault == "most" and which == "prefill":
            continue                                                     # the bound there is the list's own
        (fine, out, mass, positions), (code, out2, mass2, positions2) = run(good, which), run(bad, which)
        assert fine == 0 and code in want_codes, (which, code)
        others = [0, 2]
        width = min(mass.shape[2], mass2.shape[2])
        lens = {0: 300, 2: 90}
        for b in others:
            n = min(lens[b], 64) if which == "evict" else lens[b]
            torch.testing.assert_close(mass2[b, :, :n], mass[b, :, :n], rtol=1e-5, atol=1e-6)
            assert torch.equal(positions2[b, :, :n], positions[b, :, :n])
        if which == "decode":
            torch.testing.assert_close(out2[others], out[others], rtol=2 ** -7, atol=1e-3)
        if which == "prefill":
            rows = [i for i in range(sum(new)) if not new[0] <= i < new[0] + new[1]]
            assert torch.equal(out2[rows], out[rows])
        assert torch.equal(mass2[:, :, 700:width], bad["mass"][:, :, 700:width])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_new_tokens_than_the_bound(cuda_device, dtype):
    # sequences of 33 and 40 new tokens are within it; the masses of the one of 200 stay as they are
    from kinetics_b200 import ops
    s, status = _state(8, cuda_device, dtype=dtype), ops.new_status(cuda_device)
    _, mass = ops.prefill_attention_mass(s["qs"], s["indptr"], 40, *s["table"], s["mass"], mass_out=s["mass"].clone(), status=status)
    assert int(status.item()) == 2
    status.zero_()
    _, want = ops.prefill_attention_mass(s["qs"], s["indptr"], 200, *s["table"], s["mass"], mass_out=s["mass"].clone(), status=status)
    ops.raise_on_status(status)
    assert torch.equal(mass[2], s["mass"][2])
    torch.testing.assert_close(mass[:2], want[:2], rtol=1e-5, atol=1e-6)      # other parts, other orders of fp32 sums


def test_nothing_to_do(cuda_device):
    from kinetics_b200 import ops
    s = _state(9, cuda_device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    before, status = s["mass"].clone(), ops.new_status(cuda_device)
    out, _ = ops.prefill_attention_mass(s["qs"][:0], i32(0, 0, 0, 0), 1, *s["table"], s["mass"], status=status)
    assert out.shape == (0, 8, D)
    none = (s["table"][0], i32(), i32(0), i32())
    out, _ = ops.dense_decode_mass(s["q"][:0], *none, 1, s["mass"], status=status)
    assert out.shape == (0, 8, D)
    out, _ = ops.prefill_attention_mass(s["qs"][:0], i32(0), 1, *none, s["mass"], status=status)
    ops.evict(*none, 1, s["mass"], s["positions"], s["stored"], s["seen"], 500, status=status)
    ops.raise_on_status(status)
    assert torch.equal(s["mass"], before)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_idle_rows_of_a_padded_batch(cuda_device, dtype):
    # a batch of five places, three of them idle: no pages, no new tokens, slots that are none
    from kinetics_b200 import ops
    s, status = _state(11, cuda_device, dtype=dtype), ops.new_status(cuda_device)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda_device)
    cache, indices, indptr, last = s["table"]
    view = ops.PageView(0, 0, i32(0, 44, 0, 82, 0), i32(-1, 2, 7, 0, -5))
    padded = (i32(0, 0, 99, 47, 3), i32(99, 12, 0, 4, -1))               # starts; 700 and 1300 tokens
    q = s["q"].new_zeros(5, 8, D)
    q[1], q[3] = s["q"][0], s["q"][2]
    rows = [0, 2]
    mass = s["mass"].clone()
    out, got = ops.dense_decode_mass(q, cache, indices, *padded, 82, mass, mass_out=mass.clone(), status=status, view=view)
    plain = ops.PageView(0, 0, i32(44, 82), i32(2, 0))
    two = (i32(0, 47), i32(12, 4))
    want_out, want = ops.dense_decode_mass(s["q"][rows], cache, indices, *two, 82, mass, mass_out=mass.clone(), status=status, view=plain)
    ops.raise_on_status(status)
    assert not out[[0, 2, 4]].any()
    torch.testing.assert_close(out[[1, 3]], want_out, rtol=2 ** -7, atol=1e-3)        # forms differ by the number of lists
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    new = torch.cat([s["qs"][:33], s["qs"][73:273]])
    _, got = ops.prefill_attention_mass(new, i32(0, 0, 33, 33, 233, 233), 200, cache, indices, *padded, mass, mass_out=mass.clone(),
                                        status=status, view=view)
    _, want = ops.prefill_attention_mass(new, i32(0, 33, 233), 200, cache, indices, *two, mass, mass_out=mass.clone(), status=status, view=plain)
    ops.raise_on_status(status)
    torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-6)
    runs = []
    for table, v in ((padded, view), (two, plain)):
        c, positions = cache.clone(), s["positions"].clone()
        got, _ = ops.evict(c, indices, *table, 82, mass, positions, s["stored"], i32(1300, 40, 700), 500, 4, 64, mass_out=mass.clone(),
                           status=status, view=v)
        runs.append((c, positions, got))
    ops.raise_on_status(status)
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_behind_2_31_elements(cuda_device, dtype):
    # the same sequences in the last pages of a cache whose elements pass 31 bits (and bytes 32)
    from kinetics_b200 import ops
    small = _state(12, cuda_device, dtype=dtype)
    cache, indices, indptr, last = small["table"]
    shift = 2 ** 31 // cache[0].numel() + 64
    big = torch.empty(shift + cache.shape[0], *cache.shape[1:], dtype=dtype, device=cuda_device)
    big[shift:] = cache
    status = ops.new_status(cuda_device)

    def chain(kv, indices):
        mass, positions = small["mass"].clone(), small["positions"].clone()
        table = (kv, indices, indptr, last)
        a, _ = ops.prefill_attention_mass(small["qs"], small["indptr"], small["new"], *table, mass, window=20, status=status)
        b, _ = ops.dense_decode_mass(small["q"], *table, small["most"], mass, decay=0.9, status=status)
        c, _ = ops.dense_decode_mass(small["q"], *table, 30000, mass, decay=0.9, status=status)
        ops.evict(*table, small["most"], mass, positions, small["stored"], small["seen"], 500, 4, 64, status=status)
        return a, b, c, mass, positions
    want, got = chain(cache, indices), chain(big, indices + shift)
    ops.raise_on_status(status)
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and torch.equal(big[shift:], cache)


def test_launches_are_counted(cuda_device):
    from kinetics_b200 import ops
    s = _state(10, cuda_device)

    def count(call):
        before = ops.launch_count()
        call()
        return ops.launch_count() - before
    decode = lambda most: ops.dense_decode_mass(s["q"], *s["table"], most, s["mass"])
    prefill = lambda window: ops.prefill_attention_mass(s["qs"], s["indptr"], s["new"], *s["table"], s["mass"], window=window)
    evict = lambda keep, most: ops.evict(*s["table"], most, s["mass"], s["positions"], s["stored"], s["seen"], keep)
    assert [count(lambda: decode(most)) for most in (s["most"], 30000)] == [1, 2]
    assert [count(lambda: prefill(window)) for window in (20, 0)] == [2, 3]           # 800 rows in parts of 512
    assert [count(lambda: evict(keep, most)) for keep, most in ((1300, s["most"]), (500, s["most"]), (500, 4000))] == [1, 1, 2]


def test_refusals_on_the_device(cuda_device):
    from kinetics_b200 import _lib, ops
    s = _state(7, cuda_device)
    call = lambda **kw: ops.dense_decode_mass(kw.pop("q", s["q"]), *s["table"], s["most"], kw.pop("mass", s["mass"]), **kw)
    with pytest.raises(RuntimeError, match="contiguous"):
        call(mass=s["mass"].transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        call(mass_out=s["mass"].cpu())
    with pytest.raises(TypeError):
        call(out=torch.empty_like(s["q"], dtype=torch.float32))
    with pytest.raises(TypeError):
        call(mass_out=s["mass"][:, :, :100].contiguous())
    with pytest.raises(_lib.KtkError, match="workspace"):                # lists of a bound that needs one
        ops.dense_decode_mass(s["q"], *s["table"], 30000, s["mass"], workspace=torch.empty(64, dtype=torch.uint8, device=cuda_device))
    odd = torch.empty(s["q"].numel() + 1, dtype=torch.bfloat16, device=cuda_device)[1:].view(s["q"].shape)
    with pytest.raises(_lib.KtkError, match="aligned"):
        call(q=odd)
    with pytest.raises(ValueError):
        ops.evict(*s["table"], s["most"], s["mass"], s["positions"], s["stored"][:1], s["seen"], 500)
    with pytest.raises(_lib.KtkError, match="sink"):
        ops.evict(*s["table"], s["most"], s["mass"], s["positions"], s["stored"], s["seen"], 10, sink=4, recent=7)
