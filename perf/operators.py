"""Timed cases of the operators for drafted tokens and bounded caches: what a program
that verifies drafts over the paged K/V cache, and keeps that cache within a budget, asks
of the framework.

  qk_write   the projected q, k, v of new tokens: RMS norm of every query and key head,
             rotary positions, K and V written into their pages
  tree       attention of a tree of drafted tokens over the paged cache
  observe    the attention weight that each cached token received from the newest tokens,
             added to the sums that the cache keeps
  select     which tokens of each head stay within a budget: the first ones, the newest
             ones, and of the others those of largest weight
  keep       the K and V rows that stay moved to the front: an accepted branch of drafts in
             place, the tokens of a selection into pages of their own

``run`` computes them in their plain form (elementary torch operations in 32 bits) where
``own`` is false, and through ``voom_amd.ops`` where it is true.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
BF16 = torch.bfloat16
EPS = 1e-6
THETA = 5e5
# (q heads, kv heads, head dim): SmolLM2-135M, Llama-3-8B, Qwen2.5-7B, and the 64-head
# shape of the long-context workload
HEADS = [(9, 3, 64), (32, 8, 128), (28, 4, 128), (64, 8, 128)]


def listed() -> list[dict]:
    return [
        # one decode token of one small model's request: a latency-bound call
        {"name": "qk_write_token", "kind": "qk_write", "batch": 1, "new": 1, "nq": 9, "nkv": 3,
         "d": 64, "rot": 64, "pairs": False, "norm": True, "page": 64, "ctx_max": 640},
        # the drafts of a serving batch, adjacent pairs rotated in a part of the head, ragged
        {"name": "qk_write_drafts", "kind": "qk_write", "batch": 16, "new": 13, "nq": 28,
         "nkv": 4, "d": 128, "rot": 64, "pairs": True, "norm": True, "page": 64,
         "ctx_max": 1531},
        # a chunk of a long prompt (ragged sizes)
        {"name": "qk_write_prompt", "kind": "qk_write", "batch": 1, "new": 2011, "nq": 32,
         "nkv": 8, "d": 128, "rot": 128, "pairs": False, "norm": True, "page": 64,
         "ctx_max": 6007},
        # a few drafts of one small model's request
        {"name": "tree_one", "kind": "tree", "batch": 1, "drafts": 7, "nq": 9, "nkv": 3,
         "d": 64, "page": 64, "ctx_max": 640},
        # the verify step of a serving batch with contexts and trees of all sizes
        {"name": "tree_batch", "kind": "tree", "batch": 16, "drafts": 16, "nq": 32, "nkv": 8,
         "d": 128, "page": 64, "ctx_max": 32768},
        # a wide tree over one long context
        {"name": "tree_long", "kind": "tree", "batch": 1, "drafts": 61, "nq": 64, "nkv": 8,
         "d": 128, "page": 256, "ctx_max": 131072},
        # the decode step of a serving batch whose caches are bounded
        {"name": "observe_token", "kind": "observe", "batch": 16, "window": 1, "nq": 32,
         "nkv": 8, "d": 128, "page": 64, "ctx_max": 32768},
        # the last tokens of a prompt, by which its cache is cut down
        {"name": "observe_window", "kind": "observe", "batch": 1, "window": 33, "nq": 28,
         "nkv": 4, "d": 128, "page": 64, "ctx_max": 6007},
        # a small model's request over its budget by a page
        {"name": "select_one", "kind": "select", "batch": 1, "nkv": 3, "ctx_max": 640,
         "budget": 576, "sink": 4, "recent": 64},
        # a serving batch cut down, some of its contexts still within the budget
        {"name": "select_batch", "kind": "select", "batch": 16, "nkv": 8, "ctx_max": 32768,
         "budget": 4096, "sink": 4, "recent": 256},
        # one of five drafted continuations accepted, in a serving batch
        {"name": "keep_accepted", "kind": "keep", "batch": 32, "chains": 5, "depth": 5,
         "nkv": 8, "d": 128, "page": 64, "ctx_max": 1531, "budget": 0},
        # the caches of four requests cut down to a quarter
        {"name": "keep_selected", "kind": "keep", "batch": 4, "chains": 0, "depth": 0,
         "nkv": 8, "d": 128, "page": 64, "ctx_max": 16384, "budget": 4096},
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng: random.Random) -> dict:
    """One more case of the ranges that the listed ones stand for."""
    kind = rng.choice(["qk_write", "tree", "tree", "observe", "observe", "select", "keep"])
    nq, nkv, d = rng.choice(HEADS)
    page = rng.choice([32, 64, 256])
    if kind == "qk_write":
        batch = _log(rng, 1, 48)
        new = _log(rng, 1, max(1, 2011 * 48 // (batch * (nq + 2 * nkv))))
        return {"kind": kind, "batch": batch, "new": new, "nq": nq, "nkv": nkv, "d": d,
                "rot": rng.choice([d, d, d // 2]), "pairs": rng.random() < 0.5,
                "norm": rng.random() < 0.75, "page": page,
                "ctx_max": new + _log(rng, 1, 4000)}
    if kind == "tree":
        batch = _log(rng, 1, 32)
        drafts = _log(rng, 1, 64)
        hi = min(131072, 266000 // batch, 131072 * 61 * 16 // (drafts * nq * batch))
        return {"kind": kind, "batch": batch, "drafts": drafts, "nq": nq, "nkv": nkv, "d": d,
                "page": page, "ctx_max": _log(rng, drafts + 1, max(hi, 2 * drafts))}
    if kind == "observe":
        batch = _log(rng, 1, 32)
        window = _log(rng, 1, 64)
        hi = min(131072, 266000 // batch, 131072 * 61 * 16 // (window * nq * batch))
        return {"kind": kind, "batch": batch, "window": window, "nq": nq, "nkv": nkv, "d": d,
                "page": page, "ctx_max": _log(rng, window + 1, max(hi, 2 * window))}
    if kind == "select":
        batch = _log(rng, 1, 16)
        ctx = _log(rng, 100, min(131072, 524288 // batch))
        budget = _log(rng, 32, ctx)
        recent = rng.randint(0, budget // 4)
        return {"kind": kind, "batch": batch, "nkv": nkv, "ctx_max": ctx, "budget": budget,
                "sink": rng.randint(0, min(8, budget // 4)), "recent": recent}
    batch = _log(rng, 1, 32)
    if rng.random() < 0.5:
        chains, depth = rng.randint(2, 8), rng.randint(1, 8)
        return {"kind": kind, "batch": batch, "chains": chains, "depth": depth, "nkv": nkv,
                "d": d, "page": page, "ctx_max": chains * depth + _log(rng, 1, 3000), "budget": 0}
    ctx = _log(rng, 100, min(32768, 65536 // batch))
    return {"kind": kind, "batch": batch, "chains": 0, "depth": 0, "nkv": nkv, "d": d,
            "page": page, "ctx_max": ctx, "budget": _log(rng, 32, ctx)}


# ---- inputs -------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(1000003 + seed)


def _randn(g: torch.Generator, *shape, std: float = 1.0) -> torch.Tensor:
    return torch.randn(shape, generator=g, dtype=BF16, device=DEV).mul_(std)


def _least(case: dict) -> int:
    """The shortest context of a case: its newest tokens and one before them."""
    new = (case.get("new") or case.get("drafts") or case.get("window")
           or case.get("chains", 0) * case.get("depth", 0))
    return max(new + 1, case["ctx_max"] // 32)


def _lengths(case: dict) -> list[int]:
    """Context lengths of a batch, newest tokens included: the longest, the shortest, and
    the rest uniform between them.  Sizes belong to the case, so they do not depend on
    the seed."""
    lo, hi, n = _least(case), case["ctx_max"], case["batch"]
    lo = min(lo, hi)
    r = random.Random(n * 1000003 + hi * 31 + lo)
    return [hi] + [r.randint(lo, hi) for _ in range(n - 2)] + ([lo] if n > 1 else [])


def _ragged(case: dict, most: int, salt: int) -> list[int]:
    """How many of at most ``most`` new tokens each sequence has: all, one, and between."""
    n = case["batch"]
    r = random.Random(n * 1009 + most * 17 + salt)
    return [most] + [r.randint(1, most) for _ in range(n - 1)]


def _i32(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _paged(lengths: list[int], page: int, seed: int, spare: int = 0):
    """(slots, block table [B, max_pages] int32, spare table or None): pages at shuffled
    pool slots, as requests that come and go leave them; ``spare`` pages of every sequence
    in a table of their own."""
    per = np.array([-(-n // page) for n in lengths])
    rng = np.random.RandomState(seed % (1 << 31))
    slots = int(per.sum()) + spare * len(lengths)
    perm = rng.permutation(slots).astype(np.int32)
    table = np.zeros((len(lengths), int(per.max())), np.int32)
    inside = np.arange(table.shape[1])[None, :] < per[:, None]
    table[inside] = perm[:int(per.sum())]
    rest = perm[int(per.sum()):].reshape(len(lengths), spare)
    return (slots, torch.from_numpy(table).to(DEV),
            torch.from_numpy(rest.copy()).to(DEV) if spare else None)


def _pools(g: torch.Generator, slots: int, nkv: int, page: int, d: int):
    vb = min(page, 32)
    return _randn(g, slots, nkv, page, d), _randn(g, slots, nkv, page // vb, d, vb)


def prepare(case: dict, seed: int) -> dict:
    def trees(batch: int, drafts: int) -> torch.Tensor:
        """bool [B, T, T]: draft i sees itself and its ancestors.  Parents are random
        earlier drafts or the last accepted token."""
        rng = np.random.RandomState((seed * 7 + 11) % (1 << 31))
        sees = np.zeros((batch, drafts, drafts), bool)
        rows = np.arange(batch)
        for i in range(drafts):
            parent = rng.randint(-1, i, batch) if i else np.full(batch, -1)
            sees[:, i] = np.where((parent >= 0)[:, None], sees[rows, np.maximum(parent, 0)],
                                  False)
            sees[:, i, i] = True
        return torch.from_numpy(sees).to(DEV)

    kind, g = case["kind"], _gen(seed)
    lengths = _lengths(case)
    st = {"kind": kind, "case": case, "ctx": _i32(lengths)}
    if kind == "select":
        # sums of attention weights: heavy tails, many tokens that nothing attends to
        cap = case["ctx_max"]
        u = torch.rand((case["batch"], case["nkv"], cap), generator=g, device=DEV)
        st["scores"] = torch.where(u < 0.25, 0.0, (0.05 / (u + 1e-3)).square())
        return st
    nkv, d, page = case["nkv"], case["d"], case["page"]
    if kind == "keep":
        spare = -(-case["budget"] // page)
        slots, st["table"], st["dst_table"] = _paged(lengths, page, seed, spare)
        st["k"], st["v"] = _pools(g, slots, nkv, page, d)
        if not case["budget"]:
            # the accepted part of one continuation, which stands behind the others
            b = torch.arange(case["batch"], device=DEV)
            chain = torch.randint(1, case["chains"], (case["batch"],), generator=g, device=DEV)
            count = torch.randint(case["depth"], (case["batch"],), generator=g, device=DEV) + 1
            start = st["ctx"].long() - case["chains"] * case["depth"]
            at = start[b, None] + chain[:, None] * case["depth"] \
                + torch.arange(case["depth"], device=DEV)
            st["start"], st["keep_lens"] = start.int(), count.int()
            st["keep"] = at[:, None].int().contiguous()
            return st
        cap, n = case["ctx_max"], case["budget"]
        u = torch.rand((case["batch"], nkv, cap), generator=g, device=DEV)
        inside = torch.arange(cap, device=DEV) < st["ctx"][:, None, None]
        best = u.masked_fill(~inside, -1.0).topk(min(n, cap), dim=-1).indices
        kept = torch.minimum(st["ctx"], torch.tensor(n, device=DEV, dtype=torch.int32))
        slot = torch.arange(best.shape[-1], device=DEV)
        best = torch.where(slot < kept[:, None, None], best, cap).sort(-1).values
        st["keep"] = torch.where(slot < kept[:, None, None], best, -1).int().contiguous()
        st["keep_lens"] = kept
        st["scores"], st["scores_out"] = u * 40.0, torch.empty_like(u)
        return st
    slots, st["table"], _ = _paged(lengths, page, seed)
    st["k"], st["v"] = _pools(g, slots, nkv, page, d)
    if kind == "qk_write":
        nq, new, rot = case["nq"], case["new"], case["rot"]
        st["qkv"] = _randn(g, case["batch"], new, (nq + 2 * nkv) * d)
        inv = THETA ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) / (rot // 2))
        angles = torch.arange(max(lengths), dtype=torch.float64, device=DEV)[:, None] * inv
        st["cos"], st["sin"] = angles.cos().float(), angles.sin().float()
        st["q_weight"] = st["k_weight"] = None
        if case["norm"]:
            st["q_weight"] = 1.0 + _randn(g, d, std=0.2)
            st["k_weight"] = 1.0 + _randn(g, d, std=0.2)
        st["start"] = st["ctx"] - new
        st["lens"] = _i32(_ragged(case, new, 3))
        # a draft's position is its depth in the tree, not its place in the cache
        depth = torch.arange(new, device=DEV)
        if 1 < new <= 64:
            depth = trees(1, new)[0].sum(-1) - 1
        st["positions"] = (st["start"][:, None] + depth).int().contiguous()
        return st
    new = case["drafts"] if kind == "tree" else case["window"]
    st["q"] = _randn(g, case["batch"], case["nq"], new, d, std=2.0)
    if kind == "tree":
        st["lens"] = _i32(_ragged(case, new, 5))
        st["sees"] = trees(case["batch"], new)
        return st
    # what a serving step has in hand: the log-sum-exp of its queries, and the sums so far
    st["lens"] = _i32(_ragged(case, new, 9))
    cap = st["table"].shape[1] * page
    st["lse"] = torch.empty((case["batch"], new, case["nq"]), device=DEV)
    st["lse"].copy_(torch.logsumexp(_window_scores(st, case), -1).transpose(1, 2))
    st["scores"] = torch.rand((case["batch"], nkv, cap), generator=g, device=DEV)
    st["out"] = torch.zeros_like(st["scores"])
    return st


# ---- the plain forms ----------------------------------------------------------


def _tokens_k(pool: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """The cached keys in logical order, fp32 [B, NKV, S, D]."""
    x = pool[table.long()].transpose(1, 2)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).float()


def _tokens_v(pool: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """The cached values in logical order, fp32 [B, NKV, S, D] (blocks hold V transposed)."""
    x = pool[table.long()].permute(0, 2, 1, 3, 5, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).float()


def _grouped(q: torch.Tensor, nkv: int) -> torch.Tensor:
    """q [B, NQ, T, D] -> fp32 [B, NKV, G * T, D]."""
    b, nq, t, d = q.shape
    return q.float().reshape(b, nkv, (nq // nkv) * t, d)


def _window_scores(st: dict, case: dict) -> torch.Tensor:
    """Scaled scores [B, NQ, L, S] of the newest tokens' queries, -inf where a key is not
    yet visible; queries past a sequence's own window see nothing."""
    b, nq, new, d = st["q"].shape
    s = _grouped(st["q"], case["nkv"]) @ _tokens_k(st["k"], st["table"]).transpose(2, 3)
    s = s.view(b, nq, new, -1) * d ** -0.5
    row = torch.arange(new, device=DEV)
    last = (st["ctx"] - st["lens"])[:, None] + row
    last = torch.where(row < st["lens"][:, None], last, -1)
    key = torch.arange(s.shape[-1], device=DEV)
    return s.masked_fill(key > last[:, None, :, None], -math.inf)


def _plain_tree(st: dict, case: dict):
    b, nq, t, d = st["q"].shape
    nkv = case["nkv"]
    s = _grouped(st["q"], nkv) @ _tokens_k(st["k"], st["table"]).transpose(2, 3)
    s = s.view(b, nq, t, -1) * d ** -0.5
    key = torch.arange(s.shape[-1], device=DEV)
    prefix = (st["ctx"] - st["lens"]).long()
    draft = (key - prefix[:, None])[:, None, :].expand(b, t, -1)  # the draft at each key
    seen = st["sees"].gather(2, draft.clamp(0, t - 1)) & (draft < st["lens"][:, None, None])
    seen = (draft < 0) | seen
    seen = seen & (torch.arange(t, device=DEV)[:, None] < st["lens"][:, None, None])
    s = s.masked_fill(~seen[:, None], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.clamp(min=-3e38)[..., None])
    out = p.view(b, nkv, -1, p.shape[-1]) @ _tokens_v(st["v"], st["table"])
    return {"out": out.view(b, nq, t, d).transpose(1, 2).to(BF16).contiguous(),
            "lse": lse.transpose(1, 2).contiguous()}


def _plain_observe(st: dict, case: dict):
    b, nq, new, d = st["q"].shape
    s = _window_scores(st, case)
    lse = st["lse"].transpose(1, 2)
    live = torch.isfinite(lse)
    w = torch.exp(s - lse.masked_fill(~live, 0.0)[..., None]) * live[..., None]
    w = w.view(b, case["nkv"], -1, w.shape[-1]).sum(2)
    inside = torch.arange(w.shape[-1], device=DEV) < st["ctx"][:, None, None]
    st["out"].copy_(torch.where(inside, st["scores"] + w, st["out"]))
    return st["out"]


def _plain_select(st: dict, case: dict):
    ctx, n = st["ctx"][:, None, None], case["budget"]
    pos = torch.arange(st["scores"].shape[-1], device=DEV)
    rank = st["scores"].masked_fill((pos < case["sink"]) | (pos >= ctx - case["recent"]), math.inf)
    rank = rank.masked_fill(pos >= ctx, -math.inf)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :n]
    kept = torch.minimum(st["ctx"], torch.tensor(n, dtype=torch.int32, device=DEV))
    real = torch.arange(best.shape[-1], device=DEV) < kept[:, None, None]
    best = torch.where(real, best, pos.numel()).sort(-1).values
    best = torch.where(real, best, -1).int()
    keep = torch.nn.functional.pad(best, (0, n - best.shape[-1]), value=-1)
    return {"keep": keep, "keep_lens": kept}


def _plain_keep(st: dict, case: dict):
    page, keep, nkv = case["page"], st["keep"].long().expand(-1, case["nkv"], -1), case["nkv"]
    n = keep.shape[-1]
    table = st["table"].long()
    to = table if st["dst_table"] is None else st["dst_table"].long()
    real = (torch.arange(n, device=DEV) < st["keep_lens"][:, None]).unsqueeze(1)
    real = real.expand(-1, nkv, -1)
    bi, hi, ii = real.nonzero(as_tuple=True)
    src = keep[bi, hi, ii]
    dst = ii if "start" not in st else ii + st["start"].long()[bi]
    a, b = table[bi, src // page], to[bi, dst // page]
    vb = min(page, 32)
    so, do = src % page, dst % page
    rows, cols = st["k"][a, hi, so], st["v"][a, hi, so // vb, :, so % vb]
    st["k"][b, hi, do] = rows
    st["v"][b, hi, do // vb, :, do % vb] = cols
    out = {"k": st["k"], "v": st["v"]}
    if "scores" in st:
        moved = torch.zeros_like(st["scores"])
        moved[bi, hi, dst] = st["scores"][bi, hi, src]
        out["scores"] = st["scores_out"].copy_(moved)
    return out


def _turned(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, pairs: bool) -> torch.Tensor:
    """fp32 heads [B, L, H, D] with their first 2 * cos.shape[-1] dims rotated."""
    half = cos.shape[-1]
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if pairs else (turn[..., :half], turn[..., half:])
    c, s = cos[:, :, None], sin[:, :, None]
    a, b = a * c - b * s, b * c + a * s
    turn = torch.stack((a, b), -1).flatten(-2) if pairs else torch.cat((a, b), -1)
    return torch.cat((turn, rest), -1)


def _normed(x: torch.Tensor, weight) -> torch.Tensor:
    if weight is None:
        return x
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()


def _plain_write(st: dict, case: dict):
    nq, nkv, d, page = case["nq"], case["nkv"], case["d"], case["page"]
    b, new = st["qkv"].shape[:2]
    x = st["qkv"].float().view(b, new, nq + 2 * nkv, d)
    at = st["positions"].long()
    cos, sin = st["cos"][at], st["sin"][at]
    q = _turned(_normed(x[:, :, :nq], st["q_weight"]), cos, sin, case["pairs"])
    k = _turned(_normed(x[:, :, nq:nq + nkv], st["k_weight"]), cos, sin, case["pairs"])
    bi, ti = (torch.arange(new, device=DEV) < st["lens"][:, None]).nonzero(as_tuple=True)
    dst = st["start"].long()[bi] + ti
    slot, off, vb = st["table"].long()[bi, dst // page], dst % page, min(page, 32)
    st["k"][slot, :, off] = k.to(BF16)[bi, ti]
    st["v"][slot, :, off // vb, :, off % vb] = x[:, :, nq + nkv:].to(BF16)[bi, ti]
    return {"q": q.transpose(1, 2).to(BF16).contiguous(), "k": st["k"], "v": st["v"]}


def _plain(st: dict, case: dict):
    return {"qk_write": _plain_write, "tree": _plain_tree, "observe": _plain_observe,
            "select": _plain_select, "keep": _plain_keep}[case["kind"]](st, case)


# ---- the framework's calls ----------------------------------------------------


def _framework(st: dict, case: dict):
    from voom_amd import ops

    kind = case["kind"]
    if kind == "qk_write":
        q = ops.qk_norm_rope_append(
            st["qkv"], st["cos"], st["sin"], st["positions"], st["k"], st["v"], st["table"],
            st["start"], case["nq"], case["nkv"], q_weight=st["q_weight"],
            k_weight=st["k_weight"], eps=EPS, interleaved=case["pairs"], new_lens=st["lens"])
        return {"q": q, "k": st["k"], "v": st["v"]}
    if kind == "tree":
        out, lse = ops.paged_gqa_tree(st["q"], st["k"], st["v"], st["table"], st["ctx"],
                                      mask=st["sees"], draft_lens=st["lens"], return_lse=True)
        return {"out": out, "lse": lse}
    if kind == "observe":
        return ops.paged_gqa_observe(st["q"], st["lse"], st["k"], st["table"], st["ctx"],
                                     st["scores"], window_lens=st["lens"], out=st["out"])
    if kind == "select":
        keep, keep_lens = ops.evict_select(st["scores"], st["ctx"], case["budget"],
                                           sink=case["sink"], recent=case["recent"])
        return {"keep": keep, "keep_lens": keep_lens}
    if "scores" not in st:
        ops.compact_kv(st["k"], st["v"], st["table"], st["keep"], st["keep_lens"],
                       start=st["start"])
        return {"k": st["k"], "v": st["v"]}
    ops.compact_kv(st["k"], st["v"], st["table"], st["keep"], st["keep_lens"],
                   dst_table=st["dst_table"], scores=st["scores"], scores_out=st["scores_out"])
    return {"k": st["k"], "v": st["v"], "scores": st["scores_out"]}


def run(st: dict):
    return _framework(st, st["case"]) if own else _plain(st, st["case"])


# ---- what a pass cannot do without ---------------------------------------------


def work(case: dict) -> dict:
    kind, lengths, nkv, b = case["kind"], _lengths(case), case["nkv"], case["batch"]
    total = sum(lengths)
    if kind == "qk_write":
        tokens, kept = b * case["new"], sum(_ragged(case, case["new"], 3))
        nq, d = case["nq"], case["d"]
        return {"bytes": 2 * d * (tokens * (nq + nkv) + kept * nkv) + 2 * d * tokens * nq
                + 4 * d * kept * nkv + 4 * case["rot"] * tokens,
                "flops": tokens * (nq + nkv) * (4 * d + 3 * case["rot"])}
    if kind == "tree":
        lens = _ragged(case, case["drafts"], 5)
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(lens, lengths))
        rows = b * case["drafts"] * case["nq"]
        return {"bytes": 4 * total * nkv * case["d"] + rows * (4 * case["d"] + 4)
                + b * case["drafts"] ** 2,
                "flops": 4 * pairs * case["nq"] * case["d"]}
    if kind == "observe":
        lens = _ragged(case, case["window"], 9)
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(lens, lengths))
        return {"bytes": total * nkv * (2 * case["d"] + 8)
                + sum(lens) * case["nq"] * (2 * case["d"] + 4),
                "flops": 2 * pairs * case["nq"] * case["d"]}
    if kind == "select":
        kept = sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": 4 * nkv * (total + kept), "flops": nkv * total}
    if not case["budget"]:
        kept = b * (case["depth"] + 1) // 2
        return {"bytes": nkv * kept * 8 * case["d"] + 4 * kept, "flops": 0}
    kept = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": nkv * (kept * (8 * case["d"] + 8) + 4 * b * case["ctx_max"]), "flops": 0}


# ---- the definitions in 64 bits -------------------------------------------------


def _pages64(st: dict, which: str, i: int, n: int, page: int) -> torch.Tensor:
    """K or V [NKV, n, D] of sequence i's first n tokens, in fp64."""
    at = torch.arange(n, device=DEV)
    slot, off = st["table"][i].long()[at // page], at % page
    if which == "k":
        return st["k"].permute(0, 2, 1, 3)[slot, off].double().transpose(0, 1)
    vb = min(page, 32)
    return st["v"].permute(0, 2, 4, 1, 3)[slot, off // vb, off % vb].double().transpose(0, 1)


def exact(case: dict, seed: int):
    kind = case["kind"]
    st = prepare(case, seed)

    def rows(visible):
        """(sequence, its keys, its new tokens m, scores [NKV, G, m, keys] of those).
        ``visible(i, n, m)`` gives bool [m, n]: which of n keys each of the m rows sees."""
        for i, n in enumerate(_lengths(case)):
            m = int(st["lens"][i])
            q = st["q"][i, :, :m].double().reshape(case["nkv"], -1, m, case["d"])
            k = _pages64(st, "k", i, n, case["page"])
            s = torch.matmul(q, k[:, None].transpose(2, 3)) / math.sqrt(case["d"])
            yield i, n, m, s.masked_fill_(~visible(i, n, m), -math.inf)

    if kind == "tree":
        b, nq, t, d = st["q"].shape
        out = torch.zeros((b, t, nq, d), dtype=torch.float64, device=DEV)
        lse = torch.full((b, t, nq), -math.inf, dtype=torch.float64, device=DEV)

        def visible(i, n, m):
            v = torch.ones((m, n), dtype=torch.bool, device=DEV)
            v[:, n - m:] = st["sees"][i, :m, :m]
            return v

        for i, n, m, s in rows(visible):
            top = s.amax(-1, keepdim=True)
            w = s.sub_(top).exp_()
            total = w.sum(-1, keepdim=True)
            o = torch.matmul(w, _pages64(st, "v", i, n, case["page"])[:, None]) / total
            out[i, :m] = o.reshape(nq, m, d).transpose(0, 1)
            lse[i, :m] = (top + total.log()).reshape(nq, m).t()
        return {"out": out, "lse": lse}
    if kind == "observe":
        got = st["out"].double()

        def visible(i, n, m):
            return torch.arange(n, device=DEV) <= torch.arange(n - m, n, device=DEV)[:, None]

        for i, n, m, s in rows(visible):
            lse = st["lse"][i, :m].double().t().reshape(s.shape[:3])
            weight = (s - lse[..., None]).exp().sum((1, 2))
            got[i, :, :n] = st["scores"][i, :, :n].double() + weight
        return got
    if kind == "select":
        scores, n = st["scores"].cpu().numpy(), case["budget"]
        keep = np.full((case["batch"], case["nkv"], n), -1, np.int32)
        lens = [min(c, n) for c in _lengths(case)]
        for i, c in enumerate(_lengths(case)):
            if c <= n:
                keep[i, :, :c] = np.arange(c)
                continue
            first, last = case["sink"], c - case["recent"]
            for h in range(case["nkv"]):
                order = np.argsort(-scores[i, h, first:last], kind="stable")
                chosen = order[:n - case["sink"] - case["recent"]] + first
                keep[i, h] = np.sort(np.concatenate([np.arange(first), chosen,
                                                     np.arange(last, c)]))
        return {"keep": keep, "keep_lens": np.array(lens, np.int32)}
    page, vb = case["page"], min(case["page"], 32)
    k, v = st["k"].double(), st["v"].double()
    table = st["table"].cpu().numpy()
    if kind == "keep":
        keep, lens = st["keep"].cpu().numpy(), st["keep_lens"].cpu().numpy()
        to = table if st["dst_table"] is None else st["dst_table"].cpu().numpy()
        moved = torch.zeros(st["scores"].shape, dtype=torch.float64, device=DEV) \
            if "scores" in st else None
        for i in range(case["batch"]):
            first = int(st["start"][i]) if "start" in st else 0
            for h in range(case["nkv"]):
                src = keep[i, h if keep.shape[1] > 1 else 0, :lens[i]].astype(np.int64)
                dst = first + np.arange(len(src))
                a, b = (torch.from_numpy(x.astype(np.int64)).to(DEV)
                        for x in (table[i][src // page], to[i][dst // page]))
                so, do = (torch.from_numpy(x % page).to(DEV) for x in (src, dst))
                k[b, h, do] = st["k"][a, h, so].double()
                v[b, h, do // vb, :, do % vb] = st["v"][a, h, so // vb, :, so % vb].double()
                if moved is not None:
                    moved[i, h, :len(src)] = st["scores"][i, h][torch.from_numpy(src).to(DEV)]
        return {"k": k, "v": v} if moved is None else {"k": k, "v": v, "scores": moved}
    nq, nkv, d, half = case["nq"], case["nkv"], case["d"], case["rot"] // 2
    x = st["qkv"].double().reshape(case["batch"], case["new"], nq + 2 * nkv, d)
    heads = x[:, :, :nq + nkv].clone()
    if case["norm"]:
        weight = torch.cat((st["q_weight"].double().expand(nq, d),
                            st["k_weight"].double().expand(nkv, d)))
        heads = heads / torch.sqrt((heads ** 2).mean(-1, keepdim=True) + EPS) * weight
    at = st["positions"].long()
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, :, None]
    i = torch.arange(half, device=DEV)
    one, two = (2 * i, 2 * i + 1) if case["pairs"] else (i, i + half)
    z = torch.complex(heads[..., one], heads[..., two]) * turn
    heads[..., one], heads[..., two] = z.real, z.imag
    for b in range(case["batch"]):
        n = int(st["lens"][b])
        dst = int(st["start"][b]) + torch.arange(n, device=DEV)
        slot, off = st["table"][b].long()[dst // page], dst % page
        k[slot, :, off] = heads[b, :n, nq:]
        v[slot, :, off // vb, :, off % vb] = x[b, :n, nq + nkv:]
    return {"q": heads[:, :, :nq].transpose(1, 2), "k": k, "v": v}
