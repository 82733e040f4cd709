"""Workloads of the 4-bit KV cache: append (with read-back), attention over the pages, eviction.

Sizes are those of the shapes in provekv_b200/pool.py (24 layers x 32 heads x 64, 2 kv heads x 64 with 14 query heads,
8 kv heads x 128 with 32 query heads) at serving lengths, one layer at a time.

The cache format, restated here for the plain forms: channels come in blocks of 16 with one scale; a value is
(n - 8) * s with a 4-bit n and an 8-bit s (bits 14..7 of a binary16: 5 exponent and 3 fraction bits).  Sixteen
tokens of one kv head form an atom: K codes, V codes (low nibble = even channel), K scales, V scales, token after
token; for 128 channels the two halves of a V code row are swapped where the token's number has bit 1 set.  A page holds
page_tokens / 16 atoms of each kv head.
"""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
INF = float("inf")


def listed():
    return [
        # one decode step of a busy server: a token for each of 32 sequences
        dict(name="append-step", op="append", seqs=32, max_len=4096, new=1, ragged=True, heads=8, dim=128, dtype="bf16", page=64),
        # four prompts of different lengths become resident
        dict(name="append-prompts", op="append", seqs=4, max_len=8192, new=8192, ragged=True, heads=8, dim=128, dtype="bf16", page=64),
        # f32 vectors as the codecs decode them, 32 narrow heads
        dict(name="append-decoded-f32", op="append", seqs=2, max_len=4099, new=4099, ragged=False, heads=32, dim=64, dtype="f32", page=16),
        # the smallest decode: one sequence, 2 kv heads with 7 query heads each
        dict(name="decode-one", op="attend", seqs=1, max_len=517, q_len=1, ragged=False, heads=2, group=7, dim=64, dtype="bf16", page=16,
             window=0, sinks=0, mass=False, moved=False),
        # a batch of sequences of many lengths
        dict(name="decode-batch", op="attend", seqs=32, max_len=8192, q_len=1, ragged=True, heads=8, group=4, dim=128, dtype="bf16", page=64,
             window=0, sinks=0, mass=False, moved=False),
        # one very long context: the work of a row has to be split
        dict(name="decode-long", op="attend", seqs=1, max_len=131071, q_len=1, ragged=False, heads=8, group=4, dim=128, dtype="bf16", page=64,
             window=0, sinks=0, mass=False, moved=False),
        # no shared heads, f32 queries and outputs
        dict(name="decode-wide-f32", op="attend", seqs=8, max_len=4099, q_len=1, ragged=False, heads=32, group=1, dim=64, dtype="f32", page=32,
             window=0, sinks=0, mass=False, moved=False),
        # a sliding window with sinks over long sequences
        dict(name="decode-window", op="attend", seqs=32, max_len=16384, q_len=1, ragged=True, heads=8, group=4, dim=128, dtype="f16", page=64,
             window=1024, sinks=4, mass=False, moved=False),
        # decode over an evicted cache, accumulating what eviction will go by
        dict(name="decode-mass", op="attend", seqs=16, max_len=4096, q_len=1, ragged=True, heads=8, group=4, dim=128, dtype="bf16", page=64,
             window=0, sinks=0, mass=True, moved=True),
        # a prompt's chunk of 1024 tokens against what is cached before it and itself
        dict(name="chunk", op="attend", seqs=1, max_len=8192, q_len=1024, ragged=False, heads=8, group=4, dim=128, dtype="bf16", page=64,
             window=0, sinks=0, mass=False, moved=False),
        # prompts cut down to a budget
        dict(name="evict-prompts", op="evict", seqs=4, max_len=16384, budget=4096, sinks=4, recent=512, heads=8, dim=128, page=64),
        # the usual small eviction, a page's worth of tokens beyond the budget
        dict(name="evict-step", op="evict", seqs=16, max_len=2112, budget=2048, sinks=4, recent=128, heads=32, dim=64, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "evict"])
    dim = rng.choice([64, 128])
    heads = rng.choice([1, 2, 4, 8] if dim == 128 else [2, 3, 8, 32])
    page = rng.choice([16, 32, 48, 64, 128])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "append":
        new = _log(rng, 1, 8192)
        seqs = max(1, min(_log(rng, 1, 64), (1 << 20) // (new * heads * (dim // 64) * SIZE[dtype])))
        return dict(op=op, seqs=seqs, max_len=new + rng.randrange(0, 2000), new=new, ragged=rng.random() < 0.6, heads=heads, dim=dim,
                    dtype=dtype, page=page)
    if op == "evict":
        n = _log(rng, 100, 30000)
        seqs = max(1, min(_log(rng, 1, 32), (1 << 20) // (n * heads)))
        budget = max(40, int(n * rng.uniform(0.1, 0.98)))
        return dict(op=op, seqs=seqs, max_len=n, budget=budget, sinks=rng.choice([0, 1, 4, 16]), recent=rng.randrange(0, budget - 20),
                    heads=heads, dim=dim, page=page)
    q_len = rng.choice([1, 1, 1, 2, 5, _log(rng, 8, 1024)])
    group = rng.choice([1, 2, 4, 7, 8, 12])
    n = max(q_len, _log(rng, 30, 100000))
    if q_len > 8:
        n = max(q_len, min(n, 8192))
    # at most the tokens of the long case, and scores that the plain form can hold
    seqs = max(1, min(_log(rng, 1, 48), (1 << 20) // (n * heads), (1 << 28) // (n * heads * group * q_len)))
    return dict(op=op, seqs=seqs, max_len=n, q_len=q_len, ragged=rng.random() < 0.6, heads=heads, group=group, dim=dim, dtype=dtype, page=page,
                window=rng.choice([0, 0, _log(rng, 16, 4096)]), sinks=rng.choice([0, 4, 20]), mass=rng.random() < 0.4, moved=rng.random() < 0.4)


# -- the format, in elementary operations ---------------------------------------------------------------------------
def _round_scale(amax):
    """amax / 7 to a scale (3 fraction bits, round to nearest even, exponent from -14), in 64 bits."""
    s = amax.double() / 7
    e = torch.frexp(s)[1] - 1
    step = torch.ldexp(torch.ones_like(s), e.clamp(min=-14) - 3)
    return torch.round(s / step) * step


def _quantise(x):
    """[..., d] -> codes [..., d/2] and scales [..., d/16] (uint8).  In 64 bits: quotients lie next to a border."""
    b = x.double().unflatten(-1, (-1, 16))
    s = _round_scale(b.abs().amax(-1, keepdim=True))
    n = torch.where(s > 0, torch.round(b / torch.where(s > 0, s, 1.0)), 0.0).clamp(-8, 7).to(torch.int16) + 8
    n = n.flatten(-2).unflatten(-1, (-1, 2))
    return (n[..., 0] | (n[..., 1] << 4)).to(torch.uint8), (s[..., 0].half().view(torch.int16) >> 7).to(torch.uint8)


def _values(codes, scales):
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float() - 8
    s = (scales.to(torch.int16) << 7).view(torch.float16).float()
    return (n.unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)


def _swap(v):
    """The order of a V code row's halves: [..., 16, d/2] -> the same, its own inverse."""
    if v.shape[-1] != 64:
        return v
    odd = ((torch.arange(16, device=v.device) & 2) != 0)[:, None]
    return torch.where(odd, v.roll(32, -1), v)


def _split(pages, dim):
    """pages [n, heads, page/16, 18 dim] -> K codes, V codes, K scales, V scales, each [n, heads, page, ..]."""
    a, d = pages, dim
    kc = a[..., :8 * d].unflatten(-1, (16, d // 2))
    vc = _swap(a[..., 8 * d:16 * d].unflatten(-1, (16, d // 2)))
    ks = a[..., 16 * d:17 * d].unflatten(-1, (16, d // 16))
    vs = a[..., 17 * d:].unflatten(-1, (16, d // 16))
    return [t.flatten(2, 3) for t in (kc, vc, ks, vs)]


def _join(kc, vc, ks, vs):
    kc, vc, ks, vs = (t.unflatten(2, (-1, 16)) for t in (kc, vc, ks, vs))
    return torch.cat([t.flatten(-2) for t in (kc, _swap(vc), ks, vs)], -1)


def _of_sequences(planes, table):
    """[n, heads, page, w] -> [seqs, heads, max_pages * page, w]"""
    return [p[table.clamp(min=0).long()].transpose(1, 2).flatten(2, 3) for p in planes]


def _back_to_pages(rows, table, planes, page):
    """Writes [seqs, heads, capacity, w] rows to their pages (each page belongs to one sequence)."""
    used = table >= 0
    for r, p in zip(rows, planes):
        p[table[used].long()] = r.unflatten(2, (-1, page)).transpose(1, 2)[used]


# -- inputs -----------------------------------------------------------------------------------------------------------
def _vectors(gen, shape, spread):
    """Keys or values as models have them: channels of different size, a few tokens larger than the rest."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(spread * torch.randn((shape[1], 1, shape[-1]), generator=gen, device="cuda"))
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    S, H, d, page, top = case["seqs"], case["heads"], case["dim"], case["page"], case["max_len"]
    max_pages = -(-top // page)
    cap = max_pages * page
    ints = lambda lo, hi, n: torch.randint(lo, hi, n, generator=gen, device="cuda", dtype=torch.int32)  # noqa: E731
    floor = case.get("q_len", 1) if case["op"] == "attend" else 1
    lens = torch.full((S,), top, dtype=torch.int32, device="cuda")
    if case.get("ragged"):
        lens[1:] = ints(max(floor, top // 8), top + 1, (S,))[1:]
    if case["op"] == "evict":
        lens[1::2] -= (top - case["budget"]) // 3
        lens[2:3] = case["budget"] - 1  # one that has nothing to give up
    # pages of a sequence are spread over the pool; entries behind its last page are not used
    n_pages = S * max_pages + 3
    table = torch.randperm(n_pages, generator=gen, device="cuda")[:S * max_pages].view(S, max_pages).int()
    table = torch.where(torch.arange(max_pages, device="cuda") * page < lens[:, None], table, -1)
    pages = ints(0, 256, (n_pages, H, page // 16, 18 * d)).to(torch.uint8)  # recycled pages: any bytes
    st = dict(case=case, lens=lens, table=table, pages=pages, ends=None, positions=None, mass=None)
    if case["op"] == "append":
        dt = DT[case["dtype"]]
        st["new"] = torch.minimum(lens, ints(1, case["new"] + 1, (S,))) if case["ragged"] else None
        if case["ragged"]:
            st["new"][0] = min(top, case["new"])
        st["k"], st["v"] = (_vectors(gen, (S, H, case["new"], d), 0.5).to(dt).transpose(1, 2).contiguous() for _ in range(2))
        return st
    if case["op"] == "attend":
        k, v = (_vectors(gen, (S, H, cap, d), 0.5) for _ in range(2))
        rows = [t for x in (k, v) for t in _quantise_in_parts(x)]
        rows = [rows[0], rows[2], rows[1], rows[3]]
        planes = _split(pages, d)
        live = (torch.arange(cap, device="cuda") < lens[:, None])[:, None, :, None]
        rows = [torch.where(live, r, o) for r, o in zip(rows, _of_sequences(planes, table))]
        _back_to_pages(rows, table, planes, page)
        st["pages"] = _join(*planes)
        q = torch.randn((S, case["q_len"], H * case["group"], d), generator=gen, device="cuda") * 1.5
        st["q"] = q.to(DT[case["dtype"]])
        st["scale"] = d ** -0.5
    if case["op"] == "evict" or case.get("moved"):
        # a cache that was evicted from before: tokens of any position, in any order of slots; the last ones are new
        st["ends"] = lens + ints(0, 3000, (S,))
        fresh = case.get("q_len", 64)
        slot = torch.arange(cap, device="cuda", dtype=torch.int32)
        shuffled = torch.where(slot < lens[:, None, None], torch.rand((S, H, cap), generator=gen, device="cuda"), 2.0)
        pos = torch.argsort(torch.argsort(shuffled, -1), -1).int()
        old = slot < (lens - fresh)[:, None, None]
        pos = torch.where(old, (pos.double() * ((st["ends"] - fresh).double() / lens.double())[:, None, None]).int(),
                          (st["ends"] - lens)[:, None, None] + slot)
        st["positions"] = pos.int().contiguous()
    if case["op"] == "evict" or case.get("mass"):
        # most tokens have hardly any weight, some equal amounts, a few a lot
        m = torch.exp(3 * torch.randn((S, H, cap), generator=gen, device="cuda") - 4)
        st["mass"] = torch.where(torch.rand((S, H, cap), generator=gen, device="cuda") < 0.2, torch.round(m * 8) / 8, m)
        if st["positions"] is None:
            st["positions"] = torch.arange(cap, device="cuda", dtype=torch.int32).expand(S, H, cap).contiguous()
    if st["mass"] is not None:
        # one buffer, so that a pass can put back with one copy what the pass before it changed
        st["stats"] = torch.stack([st["positions"], st["mass"].view(torch.int32)])
        st["stats_before"] = st["stats"].clone()
        st["positions"], st["mass"] = st["stats"][0], st["stats"][1].view(torch.float32)
    return st


def _quantise_in_parts(x):
    """_quantise of a large tensor, a few sequences' heads at a time (its 64-bit intermediates are large)."""
    flat = x.flatten(0, 1)
    parts = [_quantise(p) for p in flat.split(max(1, (1 << 26) // flat[0].numel()))]
    return [torch.cat(t).unflatten(0, x.shape[:2]) for t in zip(*parts)]


# -- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "append":
        return _append(state)
    if state["mass"] is not None:
        state["stats"].copy_(state["stats_before"])
    return _attend(state) if op == "attend" else _evict(state)


def _run_own(st):
    c = st["case"]
    cache = st.get("cache")
    if cache is None:  # a program makes this once for its tensors
        from provekv_b200 import kv4
        cache = st["cache"] = kv4.Kv4Cache(st["pages"], st["table"], st["lens"], ends=st["ends"], positions=st["positions"], mass=st["mass"])
    if c["op"] == "append":
        cache.append(st["k"], st["v"], st["new"])
        k, v = cache.read(c["new"], DT[c["dtype"]], st["new"])
        return {"k": k, "v": v}
    if st["mass"] is not None:
        st["stats"].copy_(st["stats_before"])
    if c["op"] == "attend":
        out, lse = cache.attend(st["q"], scale=st["scale"], window=c["window"], sinks=c["sinks"], accumulate=c["mass"])
        return {"out": out, "lse": lse, "mass": st["mass"]} if c["mass"] else {"out": out, "lse": lse}
    cache.evict(c["budget"], sinks=c["sinks"], recent=c["recent"])
    return {"pages": st["pages"], "positions": st["positions"], "mass": st["mass"]}


def _slots_of_new(st):
    """For each row of an append its slot, and whether it is one of the sequence's."""
    n = st["case"]["new"]
    new = st["new"] if st["new"] is not None else torch.full_like(st["lens"], n)
    i = torch.arange(n, device="cuda")
    return (st["lens"] - new)[:, None] + i, i < new[:, None]


def _bytes_of_rows(dim, t):
    """Where a token's K codes, V codes, K scales and V scales lie in its atom: t [n] -> four [n, w]."""
    byte, group = torch.arange(dim // 2, device="cuda"), torch.arange(dim // 16, device="cuda")
    t = t[:, None]
    flip = (t & 2) << 4 if dim == 128 else 0
    return [t * (dim // 2) + byte, 8 * dim + t * (dim // 2) + (byte ^ flip), 16 * dim + t * (dim // 16) + group, 17 * dim + t * (dim // 16) + group]


def _append(st):
    c = st["case"]
    slot, live = _slots_of_new(st)
    seq = torch.arange(c["seqs"], device="cuda")[:, None].expand_as(slot)[live]
    slot = slot[live]
    page = st["table"][seq, slot // c["page"]].long()[:, None, None]
    atom = (slot % c["page"] // 16)[:, None, None]
    head = torch.arange(c["heads"], device="cuda")[None, :, None]
    places = [(page, head, atom, w[:, None]) for w in _bytes_of_rows(c["dim"], slot % 16)]
    kc, ks = _quantise(st["k"][live])
    vc, vs = _quantise(st["v"][live])
    for where, rows in zip(places, (kc, vc, ks, vs)):
        st["pages"][where] = rows
    kc, vc, ks, vs = (st["pages"][where] for where in places)
    out = []
    for codes, scales in ((kc, ks), (vc, vs)):
        o = torch.zeros(st["k"].shape, dtype=torch.float32, device="cuda")
        o[live] = _values(codes, scales)
        out.append(o.to(DT[c["dtype"]]))
    return {"k": out[0], "v": out[1]}


def _mask(st):
    """[seqs, heads or 1, q_len, capacity]: which cached token a query token sees."""
    c = st["case"]
    cap = st["table"].shape[1] * c["page"]
    slot = torch.arange(cap, device="cuda")
    kpos = st["positions"][:, :, None] if c["moved"] else slot[None, None, None]
    ends = st["ends"] if c["moved"] else st["lens"]
    qpos = (ends[:, None] - c["q_len"] + torch.arange(c["q_len"], device="cuda"))[:, None, :, None]
    see = (kpos <= qpos) & (slot < st["lens"][:, None])[:, None, None]
    if c["window"]:
        see = see & ((qpos - kpos < c["window"]) | (kpos < c["sinks"]))
    return see


def _attend(st):
    c = st["case"]
    S, H, G, d, n = c["seqs"], c["heads"], c["group"], c["dim"], c["q_len"]
    kc, vc, ks, vs = _of_sequences(_split(st["pages"], d), st["table"])
    live = (torch.arange(kc.shape[2], device="cuda") < st["lens"][:, None])[:, None, :, None]
    k = torch.where(live, _values(kc, ks), 0.0)
    v = torch.where(live, _values(vc, vs), 0.0)
    q = st["q"].float().view(S, n, H, G, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = (q @ k.transpose(-1, -2) * st["scale"]).unflatten(2, (G, n))
    s = s.masked_fill(~_mask(st)[:, :, None], -INF)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -INF, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total > 0, total, 1.0)
    out = (p.flatten(2, 3) @ v).unflatten(2, (G, n)).permute(0, 3, 1, 2, 4).flatten(2, 3).to(DT[c["dtype"]])
    lse = (top + torch.log(total))[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
    if not c["mass"]:
        return {"out": out, "lse": lse}
    st["mass"] += p.sum((2, 3))
    return {"out": out, "lse": lse, "mass": st["mass"]}


def _evict(st):
    c = st["case"]
    B, page = c["budget"], c["page"]
    pos, mass, lens, ends = st["positions"], st["mass"], st["lens"][:, None, None], st["ends"][:, None, None]
    cap = pos.shape[-1]
    slot = torch.arange(cap, device="cuda")
    held = slot < lens
    # weights are not negative: their bits order like they do
    key = mass.view(torch.int32).long()
    key = torch.where((pos < c["sinks"]) | (pos >= ends - c["recent"]), 1 << 31, key)
    key = torch.where(held, key, -1)
    order = torch.argsort(key, dim=-1, descending=True, stable=True)
    kept = torch.zeros_like(held.expand_as(key)).scatter_(-1, order[..., :B], True) & held
    kept = torch.where(lens > B, kept, held)
    # the j-th survivor behind the budget goes to the j-th hole before it
    hole = ~kept & (slot < B) & (lens > B)
    source = torch.argsort((kept & (slot >= B)).int(), dim=-1, descending=True, stable=True)
    rank = (hole.cumsum(-1) - 1).clamp(min=0)
    src = torch.where(hole, source.gather(-1, rank), slot)
    planes = _split(st["pages"], c["dim"])
    rows = _of_sequences(planes, st["table"])
    rows = [r.gather(2, src[..., None].expand_as(r)) for r in rows]
    _back_to_pages(rows, st["table"], planes, page)
    st["pages"].copy_(_join(*planes))
    pos.copy_(pos.gather(-1, src))
    mass.copy_(mass.gather(-1, src))
    return {"pages": st["pages"], "positions": pos, "mass": mass}


# -- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    c = case
    H, d, S = c["heads"], c["dim"], c["seqs"]
    mean = (0.5625 if c.get("ragged") else 1.0) * c["max_len"]
    if c["op"] == "append":
        n = S * c["new"] * (0.5 if c["ragged"] and c["new"] > 1 else 1.0) * H * 2
        # in, coded, read again, out
        return {"bytes": n * (2 * d * SIZE[c["dtype"]] + 2 * 9 * d / 16), "flops": 4 * n * d}
    if c["op"] == "attend":
        seen = min(mean, c["window"] + c["sinks"]) if c["window"] else mean - (c["q_len"] - 1) / 2
        read = min(mean, seen + c["q_len"]) if c["window"] else mean
        rows = S * c["q_len"] * H * c["group"]
        b = S * H * read * (d + d / 8 + (8 if c["mass"] else 0) + (4 if c["moved"] else 0)) + rows * (2 * d * SIZE[c["dtype"]] + 4)
        return {"bytes": b, "flops": 4 * rows * seen * d}
    n, B = c["max_len"], c["budget"]
    held = n - (n - B) / 6
    moved = max(0.0, B * (1 - B / held))
    return {"bytes": S * H * (8 * held + 2 * moved * (9 * d / 8 + 8)), "flops": S * H * held}


# -- the definition in 64 bits --------------------------------------------------------------------------------------------
def _decoded64(pages, dim, table, page, lens):
    """K and V of every sequence from the bytes, numpy-style indexing token by token of the atoms; f64."""
    cap = table.shape[1] * page
    slot = torch.arange(cap, device="cuda")
    at = table.clamp(min=0).long()[:, slot // page]                         # [S, cap]
    atom = pages[at, :, ((slot % page) // 16).expand_as(at)]                # [S, cap, H, 18 d]
    t = slot % 16
    byte = torch.arange(dim // 2, device="cuda")
    group = torch.arange(dim // 16, device="cuda")
    flip = ((t & 2) << 4)[:, None] if dim == 128 else torch.zeros_like(t)[:, None]
    out = []
    for first, swap, scale_at in ((0, 0, 16 * dim), (8 * dim, 1, 17 * dim)):
        where = first + t[:, None] * (dim // 2) + (byte ^ flip if swap else byte)
        b = atom.gather(-1, where[None, :, None, :].expand(*atom.shape[:3], -1)).long()
        n = torch.stack([b % 16, b // 16], -1).flatten(-2).double() - 8
        g = scale_at + t[:, None] * (dim // 16) + group
        e = atom.gather(-1, g[None, :, None, :].expand(*atom.shape[:3], -1)).long()
        s = torch.where(e < 8, (e % 8).double() / 8 * 2.0 ** -14, (1 + (e % 8).double() / 8) * torch.exp2((e // 8).double() - 15))
        x = n * s.repeat_interleave(16, -1)
        out.append(torch.where((slot < lens[:, None])[:, :, None, None], x, 0.0).transpose(1, 2))
    return out


def exact(case, seed):
    c = case
    if c["op"] == "evict":
        st = prepare(case, seed)
        r = _evicted_lists(st)
        return {"pages": None, "positions": None, "mass": r}
    st = prepare(case, seed)
    if c["op"] == "append":
        out = {}
        live = _slots_of_new(st)[1][:, :, None, None]
        for name in ("k", "v"):
            x = st[name].double()
            groups = x.view(*x.shape[:-1], -1, 16)
            ideal = groups.abs().max(-1).values / 7
            # the nearest of the 224 scales; between two, the one with an even last bit
            code = torch.arange(224, device="cuda")
            scales = torch.where(code < 8, code / 8 * 2.0 ** -14, (1 + (code % 8) / 8) * torch.exp2((code // 8).double() - 15)).double()
            hi = torch.searchsorted(scales, ideal).clamp(1, 223)
            lo = hi - 1
            up, down = scales[hi] - ideal, ideal - scales[lo]
            pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
            s = scales[pick][..., None]
            r = groups / torch.where(s > 0, s, 1.0)
            whole = torch.floor(r)
            rest = r - whole
            whole = whole + ((rest > 0.5) | ((rest == 0.5) & (whole % 2 != 0)))
            y = whole.clamp(-8, 7) * s
            out[name] = torch.where(live, y.view(x.shape), 0.0)
        return out
    S, H, G, n, d = c["seqs"], c["heads"], c["group"], c["q_len"], c["dim"]
    if S * H * G * n * c["max_len"] > 1 << 29:
        return None
    k, v = _decoded64(st["pages"], d, st["table"], c["page"], st["lens"])
    see = _mask(st)
    q = st["q"].double().view(S, n, H, G, d)
    out = torch.zeros((S, n, H, G, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((S, n, H, G), dtype=torch.float64, device="cuda")
    mass = st["mass"].double() if c["mass"] else None
    for g in range(G):
        s = torch.einsum("snhd,shkd->shnk", q[:, :, :, g], k) * st["scale"]
        s = torch.where(see, s, -INF)
        z = torch.logsumexp(s, -1)
        p = torch.where(see, torch.exp(s - torch.where(z == -INF, 0.0, z)[..., None]), 0.0)
        out[:, :, :, g] = torch.einsum("shnk,shkd->snhd", p, v)
        lse[:, :, :, g] = z.transpose(1, 2)
        if mass is not None:
            mass += p.sum(2)
    r = {"out": out.flatten(2, 3), "lse": lse.flatten(2, 3)}
    if mass is not None:
        r["mass"] = mass
    return r


def _evicted_lists(st):
    """The weights after an eviction, list by list as the definition reads."""
    c = st["case"]
    B = c["budget"]
    pos, mass = st["positions"].cpu().numpy(), st["mass"].double().cpu().numpy().copy()
    lens, ends = st["lens"].tolist(), st["ends"].tolist()
    for s in range(c["seqs"]):
        n = lens[s]
        if n <= B:
            continue
        for h in range(c["heads"]):
            m = mass[s, h]
            forced = (pos[s, h, :n] < c["sinks"]) | (pos[s, h, :n] >= ends[s] - c["recent"])
            order = np.lexsort((np.arange(n), -m[:n], ~forced))
            kept = np.zeros(n, bool)
            kept[order[:B]] = True
            m[np.flatnonzero(~kept[:B])] = m[B + np.flatnonzero(kept[B:])]
    return torch.from_numpy(mass)
