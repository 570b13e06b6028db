"""Operators of a cache of bounded size, measured: attention that also accumulates what every cached token was paid, and the
eviction that goes by it.

* ``decode``: one token of every sequence over its paged cache, ``ops.dense_decode_mass``.
* ``prefill``: new tokens of every sequence over the paged cache, ``ops.prefill_attention_mass``.
* ``evict``: the tokens beyond a budget leave the cache, ``ops.evict``.

``run`` computes either the plain form (elementary torch operations in 32 bits over padded tensors) or, where ``own`` is
true, the framework's kernels.  Inputs come from a seed: N(0, 1) keys and values, queries whose logits have a spread of 1.3 and
a common part that favours the first tokens, as trained models do; pages lie in the cache in random order.
"""
import math

import numpy as np
import torch

own = False

PAGE, DIM = 16, 128
FIRST = 4                        # first tokens, which draw attention and are never evicted


def listed():
    decode = lambda name, **kw: dict(dict(name=name, op="decode", dtype="bfloat16", heads=32, kv_heads=8, decay=1.0), **kw)
    prefill = lambda name, **kw: dict(dict(name=name, op="prefill", dtype="bfloat16", heads=32, kv_heads=8, decay=1.0), **kw)
    evict = lambda name, **kw: dict(dict(name=name, op="evict", dtype="bfloat16", kv_heads=8, first=False), **kw)
    return [
        # one short sequence: launches and latency
        decode("decode b1 517", sequences=1, shortest=517, longest=517),
        # a served batch whose caches are near a budget of 2048 tokens, all lengths different
        decode("decode b48 2k", sequences=48, shortest=1790, longest=2303, decay=0.97),
        # long contexts before their first eviction
        decode("decode b32 16k", sequences=32, shortest=15000, longest=16384),
        # the fp32 form, at odd lengths
        decode("decode fp32 b5", sequences=5, shortest=301, longest=1333, heads=8, kv_heads=4, dtype="float32"),
        # a portion of a prompt on top of a cache at its budget, judged by its last 64 tokens
        prefill("portion 512+2k", sequences=1, new=512, history=2048, window=64),
        # a long prompt at once, every token's attention counted
        prefill("prompt 8k", sequences=1, new=8192, history=0, window=0),
        # ragged portions of several prompts, eight query heads per kv head, a short window
        prefill("portions 6x700", sequences=6, new=700, history=1800, window=33, heads=64, decay=0.9),
        # the fp32 form: a few dozen tokens of two sequences
        prefill("prefill fp32", sequences=2, new=75, history=333, window=0, heads=8, kv_heads=4, dtype="float32"),
        # a step that evicts one token of one sequence
        evict("evict 1 of 2049", sequences=1, shortest=2049, longest=2049, keep=2048, recent=256),
        # a served batch that ran over its budget by a quarter of a thousand tokens
        evict("evict b48 2304", sequences=48, shortest=2304, longest=2304, keep=2048, recent=256),
        # two long prompts cut to an eighth
        evict("evict b2 32k", sequences=2, shortest=32768, longest=32768, keep=4096, recent=512, first=True),
        # the fp32 cache, odd lengths, some of them within the budget
        evict("evict fp32 b7", sequences=7, shortest=150, longest=701, keep=333, recent=40, kv_heads=4, dtype="float32"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(("decode", "decode", "prefill", "prefill", "evict", "evict"))
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 8))
    size = 4 if dtype == "float32" else 2
    if op == "prefill":
        sequences = _spread(rng, 1, 8)
        history = rng.choice((0, _spread(rng, 5, 8192)))
        most = 256 if dtype == "float32" else 8192
        room = 8192 * 8192 * 16 // (sequences * heads)           # new tokens times keys, per sequence and head
        new = _spread(rng, 2, max(2, min(most // sequences, room // (history + most))))
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, sequences=sequences, new=new, history=history,
                    window=rng.choice((0, 0, _spread(rng, 1, 128))), decay=rng.choice((1.0, 0.95)))
    sequences = _spread(rng, 1, 128)
    most = min(32768, 32 * 16384 * 8 // (sequences * kv_heads * size // 2))
    longest = _spread(rng, 3, max(3, most))
    shortest = longest if rng.random() < 0.3 else rng.randint(1, longest)
    if op == "decode":
        return dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, sequences=sequences, shortest=shortest, longest=longest,
                    decay=rng.choice((1.0, 0.95)))
    keep = _spread(rng, 1 + longest // 10, longest)
    return dict(op=op, dtype=dtype, kv_heads=kv_heads, sequences=sequences, shortest=shortest, longest=longest, keep=keep,
                recent=rng.randint(0, max(0, keep - FIRST)), first=rng.random() < 0.5)


def _lengths(case):
    """Cached tokens of every sequence: evenly spread, in a mixed order."""
    n = case["sequences"]
    if case["op"] == "prefill":
        return [h + w for h, w in zip(_portions(case)[1], _portions(case)[0])]
    lo, hi = case["shortest"], case["longest"]
    return [hi - (hi - lo) * ((i * 37 + 11) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _portions(case):
    """New tokens and tokens before them, of every sequence."""
    n, new, history = case["sequences"], case["new"], case["history"]
    part = [1.0 - 0.6 * ((i * 5) % n) / n for i in range(n)]
    return [max(1, int(new * f)) for f in part], [int(history * part[-1 - i]) for i in range(n)]


def _evicted(case):
    """Places whose positions are known, and tokens seen, of every sequence."""
    known = [0 if case["first"] else min(case["keep"], n * 8 // 9) for n in _lengths(case)]
    known = [k if k >= FIRST else 0 for k in known]
    return known, [(2 * k + 5 if k else 0) + n - k for k, n in zip(known, _lengths(case))]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _random(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + part) % (1 << 62))


def prepare(case, seed):
    dtype, lengths = getattr(torch, case["dtype"]), _lengths(case)
    batch, kv_heads = len(lengths), case["kv_heads"]
    g = _random(seed, 1)
    pages = [(n + PAGE - 1) // PAGE for n in lengths]
    total = sum(pages) + 3
    kv = torch.randn(total, 2, PAGE, kv_heads, DIM, dtype=dtype, device="cuda", generator=g)
    indices = torch.randperm(total, device="cuda", generator=g)[:sum(pages)].to(torch.int32)
    indptr = np.concatenate([[0], np.cumsum(pages)])
    common = torch.randn(kv_heads, DIM, device="cuda", generator=g)
    starts = indices[torch.tensor(indptr[:-1], device="cuda")].long()
    kv[starts, 0, :FIRST] += common.to(dtype)
    s = dict(op=case["op"], kv=kv, indices=indices, indptr=_ints(indptr.tolist()),
             last=_ints([n - (p - 1) * PAGE for n, p in zip(lengths, pages)]), most_pages=max(pages), scale=DIM ** -0.5,
             lengths=_ints(lengths), status=torch.zeros(1, dtype=torch.int32, device="cuda"))
    width = max(pages) * PAGE
    if case["op"] == "evict":
        known, seen = _evicted(case)
        mass = (2 * torch.randn(batch, kv_heads, width, device="cuda", generator=g)).exp()
        # one in ten was never paid anything: ties
        s["mass"] = mass * (torch.rand(mass.shape, device="cuda", generator=g) > 0.1)
        positions = torch.zeros(batch, kv_heads, width, dtype=torch.int32, device="cuda")
        for b, k in enumerate(known):                            # the first tokens and others, in any order
            if k:
                any_order = torch.rand(kv_heads, 2 * k + 5 - FIRST, device="cuda", generator=g).argsort(dim=-1)
                positions[b, :, :FIRST] = torch.arange(FIRST, device="cuda", dtype=torch.int32)
                positions[b, :, FIRST:k] = any_order[:, :k - FIRST].to(torch.int32) + FIRST
        s.update(positions=positions, stored=_ints(known), seen=_ints(seen), keep=case["keep"], sink=min(FIRST, case["keep"] - case["recent"]),
                 recent=case["recent"], positions_out=torch.zeros_like(positions))
    else:
        if case["op"] == "prefill":
            new = _portions(case)[0]
            s.update(q_indptr=_ints(np.concatenate([[0], np.cumsum(new)]).tolist()), most_new=max(new), window=case["window"],
                     new=_ints(new))
            rows = sum(new)
        else:
            rows = batch
        q = 1.3 * torch.randn(rows, kv_heads, case["heads"] // kv_heads, DIM, device="cuda", generator=g)
        s["q"] = (q + 0.4 * common[:, None]).to(dtype).view(rows, case["heads"], DIM)
        # what some steps have paid: as large as what this call adds
        s["mass"] = torch.randn(batch, kv_heads, width, device="cuda", generator=g).exp() * (8 / width)
        s["decay"] = case["decay"]
    s["mass_out"] = torch.zeros_like(s["mass"])
    return s


def run(s):
    return {"decode": _decode, "prefill": _prefill, "evict": _evict}[s["op"]](s)


# ---------------------------------------------------------------- the operators
def _rows(s):
    """The place of every token of padded sequences: rows [batch, width] of the cache seen as [pages, 2, page, ...], and whether
    there is a token."""
    width = s["most_pages"] * PAGE
    at = torch.arange(width, device="cuda")
    held = at < s["lengths"][:, None]
    entry = (s["indptr"][:-1, None] + at // PAGE).clamp(max=s["indices"].numel() - 1)
    return s["indices"].long()[entry], (at % PAGE).expand(held.shape), held


def _cached(s):
    """Keys and values of padded sequences, fp32 [batch, kv heads, width, 128]."""
    page, slot, held = _rows(s)
    k, v = (s["kv"][page, which, slot].transpose(1, 2).float() for which in (0, 1))
    return k, v, held


def _decode(s):
    if own:
        from kinetics_b200 import ops
        return ops.dense_decode_mass(s["q"], s["kv"], s["indices"], s["indptr"], s["last"], s["most_pages"], s["mass"], s["decay"],
                                     s["scale"], mass_out=s["mass_out"], status=s["status"])
    k, v, held = _cached(s)
    batch, kv_heads, width, _ = k.shape
    q = s["q"].float().view(batch, kv_heads, -1, DIM)
    z = (q @ k.transpose(2, 3)) * s["scale"]
    z = z.masked_fill(~held[:, None, None], -math.inf)
    p = (z - z.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = (p @ v).to(s["q"].dtype).view(s["q"].shape)
    newest = torch.arange(width, device="cuda") == s["lengths"][:, None] - 1
    before = s["decay"] * s["mass"].masked_fill(newest[:, None], 0.0)
    return out, torch.where(held[:, None], before + p.sum(2), s["mass_out"])


def _prefill(s):
    if own:
        from kinetics_b200 import ops
        return ops.prefill_attention_mass(s["q"], s["q_indptr"], s["most_new"], s["kv"], s["indices"], s["indptr"], s["last"],
                                          s["mass"], s["window"], s["decay"], s["scale"], mass_out=s["mass_out"], status=s["status"])
    k, v, held = _cached(s)
    batch, kv_heads, width, _ = k.shape
    row = torch.arange(s["most_new"], device="cuda")
    new = row < s["new"][:, None]                                                       # [batch, rows]
    at = (s["q_indptr"][:-1, None] + row).clamp(max=s["q"].shape[0] - 1).long()
    q = s["q"][at].float().view(batch, s["most_new"], kv_heads, -1, DIM).permute(0, 2, 3, 1, 4)
    z = q @ k[:, :, None].transpose(3, 4)                                                # [batch, kv heads, group, rows, width]
    z.mul_(s["scale"])
    behind = torch.arange(width, device="cuda") > (s["lengths"] - s["new"])[:, None, None] + row[:, None]
    z.masked_fill_(behind[:, None, None], -math.inf)
    z.sub_(z.amax(-1, keepdim=True)).exp_()
    z.div_(z.sum(-1, keepdim=True))
    o = (z @ v[:, :, None]).permute(0, 3, 1, 2, 4).reshape(batch, s["most_new"], -1, DIM).to(s["q"].dtype)
    seq = torch.searchsorted(s["q_indptr"][1:].long(), torch.arange(s["q"].shape[0], device="cuda"), right=True)
    out = o[seq, torch.arange(s["q"].shape[0], device="cuda") - s["q_indptr"].long()[seq]]
    counted = new & (row >= s["new"][:, None] - (s["window"] or s["most_new"]))
    paid = (z * counted[:, None, None, :, None]).sum((2, 3))
    fresh = torch.arange(width, device="cuda") >= (s["lengths"] - s["new"])[:, None]
    before = s["decay"] * s["mass"].masked_fill(fresh[:, None], 0.0)
    return out, torch.where(held[:, None], before + paid, s["mass_out"])


def _evict(s):
    if own:
        from kinetics_b200 import ops
        mass, positions = ops.evict(s["kv"], s["indices"], s["indptr"], s["last"], s["most_pages"], s["mass"], s["positions"],
                                    s["stored"], s["seen"], s["keep"], s["sink"], s["recent"], mass_out=s["mass_out"],
                                    positions_out=s["positions_out"], status=s["status"])
        return s["kv"], mass, positions
    page, slot, held = _rows(s)
    batch, kv_heads, width = s["mass"].shape
    at = torch.arange(width, device="cuda").expand(batch, kv_heads, width)
    appended = (s["seen"] - s["lengths"])[:, None, None] + at
    position = torch.where(at < s["stored"][:, None, None], s["positions"].long(), appended)
    safe = (position < s["sink"]) | (position >= s["seen"][:, None, None] - s["recent"])
    rank_by = s["mass"].masked_fill(safe, math.inf).masked_fill(~held[:, None], -1.0)
    order = rank_by.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(held[:, None].expand(rank_by.shape)).scatter(-1, order, at < s["keep"]) & held[:, None]
    # the i-th hole in front of place `keep` takes the i-th kept token behind it
    front = at < s["keep"]
    hole = front & ~kept & held[:, None]
    movers = torch.where(~front & kept, at, width - 1).sort(dim=-1).values
    source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), at)
    stays = front & held[:, None]
    head = torch.arange(kv_heads, device="cuda")[:, None]
    most = min(s["keep"], width)
    b = torch.arange(batch, device="cuda")[:, None, None]
    src = torch.where(stays, source, 0)[..., :most]
    rows = s["kv"][page[b, src], :, slot[b, src], head]                                  # [batch, kv heads, kept, 2, 128]
    dst = torch.where(stays, at, 0)[..., :most]                                          # padding writes place 0 onto itself
    rows = torch.where(stays[..., :most, None, None], rows, rows[:, :, :1])
    s["kv"][page[b, dst], :, slot[b, dst], head] = rows
    mass = torch.where(stays, s["mass"].gather(-1, source), s["mass_out"])
    return s["kv"], mass, torch.where(stays, position.gather(-1, source).to(torch.int32), s["positions_out"])


# ---------------------------------------------------------------- what a pass cannot do without
def _kept(case):
    """Tokens of all sequences that stay in front of place `keep`, and an estimate of those that move there: the safe newest ones
    all lie behind it after a first pass, the others are kept in proportion."""
    stay = moved = 0
    for n in _lengths(case):
        stay += min(n, case["keep"])
        if n > case["keep"]:
            moved += max(1, (n - case["keep"]) * case["keep"] // n)
    return stay, moved


def work(case):
    size, kv_heads, tokens = (4 if case["dtype"] == "float32" else 2), case["kv_heads"], sum(_lengths(case))
    if case["op"] == "evict":
        stay, moved = _kept(case)
        read = sum(_evicted(case)[0])
        return {"bytes": kv_heads * (4 * tokens + 4 * read + 8 * stay + moved * 2 * 2 * DIM * size), "flops": 0}
    pairs, rows = tokens, case["sequences"]
    if case["op"] == "prefill":
        new, history = _portions(case)
        pairs, rows = sum(h * w + w * (w + 1) // 2 for h, w in zip(history, new)), sum(new)
    return {"bytes": kv_heads * tokens * (2 * DIM * size + 8) + 2 * rows * case["heads"] * DIM * size,
            "flops": 4 * DIM * case["heads"] * pairs}


# ---------------------------------------------------------------- in 64 bits, sequence by sequence
def _tokens(s, b):
    """Keys and values of sequence b, [kv heads, tokens, 128]."""
    lo, hi = int(s["indptr"][b]), int(s["indptr"][b + 1])
    flat = s["kv"][s["indices"][lo:hi].long()].transpose(0, 1).reshape(2, -1, *s["kv"].shape[3:])
    return flat[:, :int(s["lengths"][b])].transpose(1, 2).double()


def exact(case, seed):
    s = prepare(case, seed)
    batch, kv_heads = case["sequences"], case["kv_heads"]
    mass = s["mass_out"].double()
    if case["op"] == "evict":
        return _exact_evict(case, s, mass)
    group = case["heads"] // kv_heads
    if case["op"] == "decode":
        new, window, first = [1] * batch, 0, list(range(batch + 1))
    else:
        new, window, first = _portions(case)[0], case["window"], s["q_indptr"].tolist()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(batch):
        k, v = _tokens(s, b)
        n, w = k.shape[1], new[b]
        horizon = torch.arange(n - w, n, device="cuda")
        mass[b, :, :n] = s["decay"] * s["mass"][b, :, :n].double() * (torch.arange(n, device="cuda") < n - w)
        counted = horizon >= n - (window or w)
        for h in range(kv_heads):
            q = s["q"][first[b]:first[b + 1], h * group:(h + 1) * group].double()
            p = torch.einsum("wgd,td->gwt", q, k[h]) / math.sqrt(DIM)
            p.masked_fill_(torch.arange(n, device="cuda") > horizon[:, None], -math.inf)
            p = torch.softmax(p, -1)
            out[first[b]:first[b + 1], h * group:(h + 1) * group] = torch.einsum("gwt,td->wgd", p, v[h])
            mass[b, h, :n] += p[:, counted].sum((0, 1))
    return out, mass


def _exact_evict(case, s, mass):
    positions, kv, keep = s["positions_out"].cpu().numpy(), s["kv"].clone(), s["keep"]
    for b, n in enumerate(_lengths(case)):
        pages = s["indices"][int(s["indptr"][b]):int(s["indptr"][b + 1])].cpu().numpy()
        stored, seen = int(s["stored"][b]), int(s["seen"][b])
        for h in range(case["kv_heads"]):
            paid = s["mass"][b, h, :n].double().cpu().numpy()
            where = np.concatenate([s["positions"][b, h, :stored].cpu().numpy(), np.arange(seen - n + stored, seen)]).astype(np.int64)
            safe = (where < s["sink"]) | (where >= seen - s["recent"])
            chosen = np.lexsort((np.arange(n), -paid, ~safe))[:keep]
            places = np.arange(min(n, keep))
            holes = np.setdiff1d(places, chosen)
            movers = np.sort(chosen[chosen >= keep])
            at = lambda t: (torch.from_numpy(pages[t // PAGE].astype(np.int64)).cuda(), torch.from_numpy(t % PAGE).cuda())
            (sp, ss), (dp, ds) = at(movers), at(holes)
            kv[dp, :, ds, h] = s["kv"][sp, :, ss, h]
            places[holes] = movers
            mass[b, h, :len(places)] = torch.from_numpy(paid[places]).cuda()
            positions[b, h, :len(places)] = where[places]
    return kv, mass, torch.from_numpy(positions).cuda()
