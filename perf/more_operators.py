"""Timed cases of the operators for ragged batches and beam search: what a program that
serves chunks and single tokens of many sequences over the paged K/V cache, with models
that cap or bias their attention scores and norm their blocks on both sides, and that
searches with beams, asks of the framework.

  chunk   attention of every sequence's newest tokens (one of them, or a part of its
          prompt) over the paged cache: scores capped by a tanh, or lowered with the
          distance, a sliding window, a prefix that all tokens see
  beam    the best continuations over beams and vocabulary, and which beam each goes on from
  fork    the cached K and V of beams that go on from another one, copied in all layers
  post    the norm behind a block, the residual add and the norm before the next block

``run`` computes them in their plain form (elementary torch operations in 32 bits, in 64
where values meet at a border) where ``own`` is false, and through ``voom_amd.ops`` where
it is true.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
EPS = 1e-6
END = 2  # the token that ends a beam
# (q heads, kv heads, head dim): SmolLM2-135M, Llama-3-8B, Qwen2.5-7B, and the 64-head
# shape of the long-context workload
HEADS = [(9, 3, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128)]
# a chunk pass costs at most this many (query head, key) pairs: chunk_prompt's
PAIRS = 2011 * 6007 * 32


def _chunk(**kw) -> dict:
    return {"kind": "chunk", "cap": 0.0, "bias": False, "window": 0, "prefix": 0, "packed": True,
            "page": 64} | kw


def listed() -> list[dict]:
    return [
        # one decode token of one small model's request: a latency-bound call
        _chunk(name="chunk_token", batch=1, new=1, nq=9, nkv=3, d=64, ctx_max=640, cap=30.0,
               packed=False),
        # the decode step of a serving batch in a layer that sees everything
        _chunk(name="chunk_tokens", batch=16, new=1, nq=32, nkv=8, d=128, ctx_max=32768,
               cap=50.0),
        # the same step in a layer with a sliding window, the first tokens always seen
        _chunk(name="chunk_window", batch=32, new=1, nq=28, nkv=4, d=128, ctx_max=32768,
               window=4096, prefix=4),
        # a step that takes in parts of new prompts beside the running requests' tokens
        _chunk(name="chunk_mixed", batch=16, new=509, nq=32, nkv=8, d=128, ctx_max=8192,
               cap=50.0),
        # the last part of a long prompt (ragged sizes)
        _chunk(name="chunk_prompt", batch=1, new=2011, nq=32, nkv=8, d=128, ctx_max=6007,
               cap=50.0),
        # prompts with a part that is seen in both directions, scores lowered with the distance
        _chunk(name="chunk_bias", batch=2, new=1021, nq=64, nkv=8, d=128, ctx_max=1999,
               bias=True, prefix=300, packed=False, page=256),
        # a request that searches with a few beams
        {"name": "beam_one", "kind": "beam", "batch": 1, "beams": 4, "vocab": 49152,
         "fp32": False, "ended": False},
        # a batch of them, some beams at their end, a large vocabulary
        {"name": "beam_batch", "kind": "beam", "batch": 16, "beams": 8, "vocab": 128256,
         "fp32": True, "ended": True},
        # a small model's beams, apart for a few tokens
        {"name": "fork_one", "kind": "fork", "batch": 1, "beams": 4, "layers": 30, "nkv": 3,
         "d": 64, "page": 64, "ctx_max": 640, "apart": 24},
        # a batch of requests, some of whose beams went apart long ago
        {"name": "fork_batch", "kind": "fork", "batch": 8, "beams": 5, "layers": 8, "nkv": 8,
         "d": 128, "page": 64, "ctx_max": 1531, "apart": 700},
        # one decode token of a small model
        {"name": "post_token", "kind": "post", "rows": 1, "hidden": 576, "gates": 0,
         "scale": 1.0},
        # a long prompt, each of its sequences with a gate of its own
        {"name": "post_prompt", "kind": "post", "rows": 6006, "hidden": 4096, "gates": 3,
         "scale": 0.22},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(["chunk", "chunk", "chunk", "chunk", "beam", "beam", "fork", "post"])
    nq, nkv, d = rng.choice(HEADS)
    page = rng.choice([32, 64, 256])
    if kind == "chunk":
        batch = _log(rng, 1, 48)
        new = 1 if rng.random() < 0.4 else _log(rng, 2, 2011)
        case = _chunk(batch=batch, new=new, nq=nq, nkv=nkv, d=d, page=page,
                      cap=rng.choice([0.0, 30.0, 50.0]), bias=rng.random() < 0.3,
                      window=_log(rng, 64, 4096) if rng.random() < 0.4 else 0,
                      prefix=_log(rng, 1, 300) if rng.random() < 0.3 else 0,
                      packed=rng.random() < 0.7)
        rows = sum(_chunks(case)) if case["packed"] else batch * new
        hi = min(131072, 266000 * 64 // (batch * nkv * d // 16), PAIRS // (rows * nq))
        case["ctx_max"] = new + _log(rng, 1, max(hi - new, 1))
        return case
    if kind == "beam":
        batch, beams = _log(rng, 1, 32), rng.randint(1, 16)
        return {"kind": kind, "batch": batch, "beams": beams,
                "vocab": _log(rng, 1000, min(152064, 16 * 8 * 128256 // (batch * beams))),
                "fp32": rng.random() < 0.5, "ended": rng.random() < 0.5}
    if kind == "fork":
        batch, beams, layers = _log(rng, 1, 8), rng.randint(2, 8), rng.choice([4, 8, 30])
        ctx = _log(rng, 20, 8 * 8 * 5 * 8 * 1531 * 128 // (batch * beams * layers * nkv * d))
        return {"kind": kind, "batch": batch, "beams": beams, "layers": layers, "nkv": nkv,
                "d": d, "page": page, "ctx_max": ctx, "apart": _log(rng, 1, ctx)}
    hidden = rng.choice([576, 2048, 4096, 8192, 8 * rng.randint(1, 1024)])
    rows = _log(rng, 1, 6006 * 4096 // hidden)
    return {"kind": kind, "rows": rows, "hidden": hidden, "gates": rng.choice([0, 1, rows]),
            "scale": rng.choice([1.0, 0.22])}


# ---- inputs -------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(1000003 + seed)


def _randn(g: torch.Generator, *shape, std: float = 1.0, dtype=BF16) -> torch.Tensor:
    return torch.randn(shape, generator=g, dtype=dtype, device=DEV).mul_(std)


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# Sizes (lengths, parents, tokens apart) belong to the case and not to the seed.


def _chunks(case: dict) -> list[int]:
    """New tokens of each sequence: one chunk as long as ``new``, of the others three in
    four a single token and the rest of any length."""
    r = random.Random(case["batch"] * 1000003 + case["new"])
    lens = [1 if r.random() < 0.75 else _log(r, 1, case["new"]) for _ in range(case["batch"])]
    lens[r.randrange(len(lens))] = case["new"]
    return lens


def _lengths(case: dict) -> list[int]:
    """Cached tokens of each sequence, the new ones included: the longest as long as
    ``ctx_max``, the rest uniform down to a thirty-second of it."""
    r = random.Random(case["batch"] * 1000003 + case["ctx_max"] * 31)
    hi, chunks = case["ctx_max"], _chunks(case)
    lens = [max(n, r.randint(max(1, hi // 32), hi)) for n in chunks]
    lens[r.randrange(len(lens))] = hi
    return lens


def _family(case: dict):
    """Of each request's beams the one that each goes on from, and how many of its newest
    tokens differ from that one's.  A beam that others go on from stays."""
    r = random.Random(case["batch"] * 1000003 + case["beams"] * 8191 + case["ctx_max"])
    parents, apart = [], []
    for _ in range(case["batch"]):
        stay = sorted(r.sample(range(case["beams"]), r.randint(1, max(1, case["beams"] - 1))))
        parents.append([j if j in stay else r.choice(stay) for j in range(case["beams"])])
        apart.append([0 if p == j else _log(r, 1, min(case["apart"], case["ctx_max"]))
                      for j, p in enumerate(parents[-1])])
    return parents, apart


def _paged(lengths: list[int], page: int, seed: int):
    """Slots of the pool and a block table of pages in random order."""
    pages = [-(-n // page) for n in lengths]
    order = list(range(sum(pages)))
    random.Random(seed * 7919 + 13).shuffle(order)
    width, at, rows = max(pages), 0, []
    for n in pages:
        rows.append(order[at:at + n] + [0] * (width - n))
        at += n
    return sum(pages), _i32(rows)


def _pools(g: torch.Generator, slots: int, nkv: int, page: int, d: int):
    vb = min(page, 32)
    return _randn(g, slots, nkv, page, d), _randn(g, slots, nkv, page // vb, d, vb)


def prepare(case: dict, seed: int) -> dict:
    kind, g = case["kind"], _gen(seed)
    st = {"case": case}
    if kind == "chunk":
        nq, nkv, d, page, b = (case[k] for k in ("nq", "nkv", "d", "page", "batch"))
        lengths, chunks = _lengths(case), _chunks(case)
        slots, st["table"] = _paged(lengths, page, seed)
        st["k"], st["v"] = _pools(g, slots, nkv, page, d)
        st["ctx"] = _i32(lengths)
        st["starts"] = st["new_lens"] = st["slopes"] = st["prefix"] = None
        if case["packed"]:
            st["q"] = _randn(g, sum(chunks), nq, d, std=2.0)
            st["starts"] = _i32([sum(chunks[:i]) for i in range(b + 1)])
        else:
            st["q"] = _randn(g, b, nq, case["new"], d, std=2.0)
            st["new_lens"] = _i32(chunks)
        if case["bias"]:  # a geometric row of slopes, one a head
            st["slopes"] = torch.exp2(-8.0 * torch.arange(1, nq + 1, device=DEV) / nq)
        if case["prefix"]:
            st["prefix"] = _i32([min(case["prefix"], n) for n in lengths])
        return st
    if kind == "beam":
        b, k, vocab = case["batch"], case["beams"], case["vocab"]
        st["logits"] = _randn(g, b, k, vocab, std=2.5,
                              dtype=torch.float32 if case["fp32"] else BF16)
        st["scores"] = -torch.rand((b, k), generator=g, device=DEV).mul_(4).cumsum(1) - 5.0
        st["last"] = torch.randint(3, vocab, (b, k), generator=g, device=DEV)
        if case["ended"]:
            over = torch.rand((b, k), generator=g, device=DEV) < 0.25
            st["last"] = torch.where(over, END, st["last"])
        # how many leading tokens each two beams have in common
        ctx = torch.randint(60, 2000, (b,), generator=g, device=DEV)
        common = (torch.rand((b, k, k), generator=g, device=DEV) * ctx[:, None, None]).int()
        common = torch.minimum(common, common.transpose(1, 2))
        eye = torch.eye(k, dtype=torch.bool, device=DEV)
        st["ctx"] = ctx.int()
        st["shared"] = torch.where(eye, ctx[:, None, None].int(), common).contiguous()
        return st
    if kind == "fork":
        rows, n = case["batch"] * case["beams"], case["ctx_max"]
        parents, apart = _family(case)
        st["k"], st["v"], st["tables"] = [], [], []
        for layer in range(case["layers"]):
            slots, table = _paged([n] * rows, case["page"], seed * 64 + layer)
            k, v = _pools(g, slots, case["nkv"], case["page"], case["d"])
            st["k"].append(k)
            st["v"].append(v)
            st["tables"].append(table)
        st["ctx"] = _i32([n] * case["batch"])
        st["parents"] = _i32(parents)
        st["first"] = _i32([[n - a for a in row] for row in apart])
        return st
    rows, hidden = case["rows"], case["hidden"]
    st["x"], st["delta"] = _randn(g, rows, hidden, std=3.0), _randn(g, rows, hidden)
    st["post_weight"] = 1.0 + _randn(g, hidden, std=0.2)
    st["weight"] = 1.0 + _randn(g, hidden, std=0.2)
    st["gate"] = _randn(g, case["gates"], hidden, std=0.5) if case["gates"] else None
    st["x_out"] = torch.empty_like(st["x"])
    return st


# ---- the plain forms ----------------------------------------------------------


def _cached(st: dict, i: int, n: int):
    """K and V of sequence i's first n tokens, fp32 [NKV, n, D]."""
    page = st["case"]["page"]
    slots = st["table"][i, :-(-n // page)].long()
    k = st["k"][slots].transpose(0, 1).flatten(1, 2)[:, :n].float()
    v = st["v"][slots].permute(1, 0, 2, 4, 3).flatten(1, 3)[:, :n].float()
    return k, v


def _sees(case: dict, n: int, m: int, prefix: int) -> torch.Tensor:
    """bool [m, n]: which cached tokens the newest m see."""
    at = torch.arange(n - m, n, device=DEV)[:, None]
    key = torch.arange(n, device=DEV)
    seen = key <= at
    if case["window"]:
        seen = seen & (at - key < case["window"])
    return seen | (key < prefix)


def _plain_chunk(st: dict, case: dict):
    nq, nkv, d = case["nq"], case["nkv"], case["d"]
    q = st["q"] if case["packed"] else st["q"].transpose(1, 2)
    out = torch.zeros(q.shape, dtype=BF16, device=DEV)
    lse = torch.full(q.shape[:-1], -math.inf, device=DEV)
    at = 0
    for i, (n, m) in enumerate(zip(_lengths(case), _chunks(case))):
        rows = (slice(at, at + m),) if case["packed"] else (i, slice(0, m))
        at += m
        k, v = _cached(st, i, n)
        s = q[rows].float().transpose(0, 1).reshape(nkv, -1, d) @ k.transpose(1, 2)
        s = s.view(nq, m, n).mul_(d ** -0.5)
        if case["cap"]:
            s = case["cap"] * torch.tanh(s / case["cap"])
        if case["bias"]:
            token = torch.arange(n, device=DEV)
            s -= st["slopes"][:, None, None] * (token[n - m:, None] - token).abs()
        s.masked_fill_(~_sees(case, n, m, min(case["prefix"], n)), -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        total = p.sum(-1, keepdim=True)
        o = (p.view(nkv, -1, n) @ v).view(nq, m, d) / total
        out[rows] = o.transpose(0, 1).to(BF16)
        lse[rows] = (top + total.log())[..., 0].t()
    return {"out": out, "lse": lse}


def _plain_beam(st: dict, case: dict):
    b, k, vocab = st["logits"].shape
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - top - torch.exp(x - top).sum(-1, keepdim=True).log()
    over = st["last"] == END
    x = x.masked_fill(over[..., None], -math.inf) + st["scores"].double()[..., None]
    x[..., END] = torch.where(over, st["scores"].double(), x[..., END])
    x = x.flatten(1)
    cell = torch.arange(x.shape[1], device=DEV)
    best, at = [], []
    for _ in range(k):  # the largest, the first of equal ones
        v = x.amax(1)
        i = torch.where(x == v[:, None], cell, x.shape[1]).amin(1)
        x.scatter_(1, i[:, None], -math.inf)
        best.append(v)
        at.append(i)
    best, at = torch.stack(best, 1), torch.stack(at, 1)
    parent = at // vocab
    # a beam's best continuation keeps its row, the others take the rows left free
    rank = torch.arange(k, device=DEV)
    stays = ~((parent[:, :, None] == parent[:, None]) & (rank < rank[:, None])).any(-1)
    taken = torch.zeros((b, k + 1), dtype=torch.bool, device=DEV)
    taken.scatter_(1, torch.where(stays, parent, k), True)
    free = torch.sort(taken[:, :k].int(), dim=1, stable=True).indices
    row = torch.where(stays, parent, free.gather(1, ((~stays).cumsum(1) - 1).clamp(min=0)))
    order = torch.sort(row, dim=1).indices
    parent = parent.gather(1, order)
    pick = st["shared"].gather(1, parent[..., None].expand(-1, -1, k))  # [row's parent, beam]
    first = torch.where(parent == rank, st["ctx"][:, None], pick.gather(2, rank.expand(b, k)[
        ..., None])[..., 0])
    both = pick.gather(2, parent[:, None].expand(-1, k, -1))
    both = torch.where(parent[:, :, None] == parent[:, None], st["ctx"][:, None, None], both)
    return {"scores": best.gather(1, order).float(), "tokens": (at % vocab).gather(1, order),
            "parents": parent.int(), "first": first.int(), "shared": both.int()}


def _plain_fork(st: dict, case: dict):
    n, page, beams = case["ctx_max"], case["page"], case["beams"]
    token = torch.arange(n, device=DEV)
    row, at = (token >= st["first"].view(-1, 1)).nonzero(as_tuple=True)
    from_row = row // beams * beams + st["parents"].view(-1).long()[row]
    vb = min(page, 32)
    off = at % page
    for k, v, table in zip(st["k"], st["v"], st["tables"]):
        src, dst = table[from_row, at // page].long(), table[row, at // page].long()
        k[dst, :, off] = k[src, :, off]
        v[dst, :, off // vb, :, off % vb] = v[src, :, off // vb, :, off % vb]
    return {"k": st["k"], "v": st["v"]}


def _normed(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_post(st: dict, case: dict):
    y = _normed(st["delta"].float(), st["post_weight"]) * case["scale"]
    if st["gate"] is not None:
        y = y * st["gate"].float().repeat_interleave(case["rows"] // case["gates"], 0)
    y = st["x"].float() + y
    return {"x": y.to(BF16), "out": _normed(y, st["weight"]).to(BF16)}


# ---- the framework's calls ----------------------------------------------------


def _framework(st: dict, case: dict):
    from voom_amd import ops

    kind = case["kind"]
    if kind == "chunk":
        out, lse = ops.paged_gqa_chunk(
            st["q"], st["k"], st["v"], st["table"], st["ctx"], starts=st["starts"],
            new_lens=st["new_lens"], softcap=case["cap"], slopes=st["slopes"],
            window=case["window"], prefix_lens=st["prefix"], return_lse=True)
        return {"out": out, "lse": lse}
    if kind == "beam":
        scores, tokens, parents, first, shared = ops.beam_select(
            st["logits"], st["scores"], last=st["last"], end_token=END, shared=st["shared"],
            ctx_lens=st["ctx"])
        return {"scores": scores, "tokens": tokens, "parents": parents, "first": first,
                "shared": shared}
    if kind == "fork":
        ops.fork_kv(st["k"], st["v"], st["tables"], st["ctx"], st["parents"], st["first"])
        return {"k": st["k"], "v": st["v"]}
    out = ops.add_post_norm(st["x"], st["delta"], st["post_weight"], st["weight"], EPS,
                            gate=st["gate"], scale=case["scale"], x_out=st["x_out"])
    return {"x": st["x_out"], "out": out}


def run(st: dict):
    kind = st["case"]["kind"]
    if own:
        return _framework(st, st["case"])
    return {"chunk": _plain_chunk, "beam": _plain_beam, "fork": _plain_fork,
            "post": _plain_post}[kind](st, st["case"])


# ---- what a pass cannot do without ---------------------------------------------


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "chunk":
        nq, nkv, d = case["nq"], case["nkv"], case["d"]
        pairs = tokens = 0
        for n, m in zip(_lengths(case), _chunks(case)):
            prefix, window = min(case["prefix"], n), case["window"] or n
            low = max(0, n - m + 1 - window)  # the first key of the first new token
            tokens += n - max(0, low - prefix)
            for at in range(n - m, n):
                lo = max(0, at + 1 - window)
                pairs += at + 1 - max(0, lo - prefix) + max(0, prefix - at - 1)
        rows = sum(_chunks(case)) * nq
        return {"bytes": 4 * d * nkv * tokens + rows * (4 * d + 4), "flops": 4 * d * nq * pairs}
    if kind == "beam":
        cells = case["batch"] * case["beams"] * case["vocab"]
        # (beams at their end need none of their logits; about a quarter of them)
        cells = cells * 3 // 4 if case["ended"] else cells
        return {"bytes": cells * (4 if case["fp32"] else 2), "flops": 3 * cells}
    if kind == "fork":
        moved = sum(a for row in _family(case)[1] for a in row)
        return {"bytes": moved * case["layers"] * case["nkv"] * case["d"] * 8, "flops": 0}
    cells = case["rows"] * case["hidden"]
    return {"bytes": 8 * cells + 2 * case["hidden"] * (2 + case["gates"]), "flops": 10 * cells}


# ---- the definitions in 64 bits -------------------------------------------------


def _exact_chunk(st: dict, case: dict):
    """Row by row of the definition, a sequence and a kv head at a time."""
    nq, nkv, d, page = case["nq"], case["nkv"], case["d"], case["page"]
    group, vb = nq // nkv, min(page, 32)
    shape = (*st["q"].shape,) if case["packed"] else (case["batch"], case["new"], nq, d)
    out = torch.zeros(shape, dtype=torch.float64, device=DEV)
    lse = torch.full(shape[:-1], -math.inf, dtype=torch.float64, device=DEV)
    begin = 0
    for i in range(case["batch"]):
        n, m = _lengths(case)[i], _chunks(case)[i]
        token = torch.arange(n, device=DEV)
        slot, off = st["table"][i].long()[token // page], token % page
        distance = (token[n - m:, None] - token).double()
        hidden = distance < 0
        if case["window"]:
            hidden |= distance >= case["window"]
        hidden &= token >= case["prefix"]
        for h in range(nkv):
            heads = slice(h * group, (h + 1) * group)
            if case["packed"]:
                q = st["q"][begin:begin + m, heads].double().transpose(0, 1)
            else:
                q = st["q"][i, heads, :m].double()
            k = st["k"][slot, h, off].double()
            v = st["v"][slot, h, off // vb, :, off % vb].double()
            s = torch.matmul(q, k.t()).div_(math.sqrt(d))
            if case["cap"]:
                s.div_(case["cap"]).tanh_().mul_(case["cap"])
            if case["bias"]:
                s -= st["slopes"].double()[heads, None, None] * distance.abs()
            s.masked_fill_(hidden, -math.inf)
            total = torch.logsumexp(s, -1)
            o = torch.matmul(s.sub_(total[..., None]).exp_(), v).transpose(0, 1)
            if case["packed"]:
                out[begin:begin + m, heads], lse[begin:begin + m, heads] = o, total.t()
            else:
                out[i, :m, heads], lse[i, :m, heads] = o, total.t()
        begin += m
    return {"out": out, "lse": lse}


def _exact_beam(st: dict, case: dict):
    """The search on the host, request by request, over the beams' best few tokens."""
    k, vocab, ctx = case["beams"], case["vocab"], st["ctx"].tolist()
    x = st["logits"].double()
    norm = torch.logsumexp(x, -1).cpu().tolist()
    # (more tokens than a beam can place, so that ties at the last place are all there)
    few = x.topk(min(vocab, 4 * k + 32), dim=-1)
    values, index = few.values.cpu().tolist(), few.indices.cpu().tolist()
    scores, last = st["scores"].double().tolist(), st["last"].tolist()
    shared = st["shared"].tolist()
    got = {"scores": [], "tokens": [], "parents": [], "first": [], "shared": []}
    for b in range(case["batch"]):
        found = []
        for j in range(k):
            if last[b][j] == END:
                found.append((-scores[b][j], j, END))
                continue
            found += [(-(scores[b][j] + (v - norm[b][j])), j, t)
                      for v, t in zip(values[b][j], index[b][j])]
        rows, rest = {}, []
        for c in sorted(found)[:k]:
            if c[1] in rows:
                rest.append(c)
            else:
                rows[c[1]] = c
        for j in range(k):
            if j not in rows:
                rows[j] = rest.pop(0)
        order = [rows[j] for j in range(k)]
        parents = [c[1] for c in order]
        got["scores"].append([-c[0] for c in order])
        got["tokens"].append([c[2] for c in order])
        got["parents"].append(parents)
        got["first"].append([ctx[b] if p == j else shared[b][p][j]
                             for j, p in enumerate(parents)])
        got["shared"].append([[ctx[b] if p == r else shared[b][p][r] for r in parents]
                              for p in parents])
    kinds = {"scores": torch.float64, "tokens": torch.int64}
    return {name: torch.tensor(v, dtype=kinds.get(name, torch.int32), device=DEV)
            for name, v in got.items()}


def _exact_fork(st: dict, case: dict):
    """Sequence by sequence in logical order."""
    parents, apart = _family(case)
    n, page, vb = case["ctx_max"], case["page"], min(case["page"], 32)
    for k, v, table in zip(st["k"], st["v"], st["tables"]):
        for b, (family, tails) in enumerate(zip(parents, apart)):
            for j, (p, tail) in enumerate(zip(family, tails)):
                token = torch.arange(n - tail, n, device=DEV)
                src, dst = (table[b * case["beams"] + r].long()[token // page] for r in (p, j))
                off = token % page
                k[dst, :, off] = k[src, :, off]
                v[dst, :, off // vb, :, off % vb] = v[src, :, off // vb, :, off % vb]
    return {"k": st["k"], "v": st["v"]}


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "chunk":
        return _exact_chunk(st, case)
    if case["kind"] == "beam":
        return _exact_beam(st, case)
    if case["kind"] == "fork":
        return _exact_fork(st, case)
    x, delta = st["x"].double(), st["delta"].double()
    n = case["hidden"]
    y = delta / ((delta * delta).sum(-1, keepdim=True) / n + EPS).sqrt()
    y *= st["post_weight"].double() * case["scale"]
    if case["gates"]:
        y = (y.view(case["gates"], -1, n) * st["gate"].double()[:, None]).view(-1, n)
    y += x
    out = y / ((y * y).sum(-1, keepdim=True) / n + EPS).sqrt() * st["weight"].double()
    return {"x": y, "out": out}
