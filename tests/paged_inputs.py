"""Inputs of the tests of paged attention operators: pools with shuffled slots, random
trees of drafts."""
import torch

from voom_amd.page_pool import v_tokens_to_pages


def cache(k, v, page, spare=0, seed=0):
    """Pools and table that hold k, v [B, NKV, S, D] at shuffled slots; what no token
    fills, ``spare`` pages per sequence included, holds NaN."""
    B, NKV, S, D = k.shape
    pages = -(-S // page)
    n = B * (pages + spare)
    fill = torch.full((B, NKV, pages * page, D), float("nan"), dtype=k.dtype, device=k.device)
    kp, vp = fill.clone(), fill
    kp[:, :, :S], vp[:, :, :S] = k, v
    g = torch.Generator().manual_seed(seed)
    perm = torch.randperm(n, generator=g).view(B, pages + spare)
    k_pool = torch.full((n, NKV, page, D), float("nan"), dtype=k.dtype, device=k.device)
    v_pool = v_tokens_to_pages(k_pool)
    at = perm[:, :pages].reshape(-1).to(k.device)
    k_pool[at] = kp.view(B, NKV, pages, page, D).transpose(1, 2).reshape(-1, NKV, page, D)
    v_pool[at] = v_tokens_to_pages(
        vp.view(B, NKV, pages, page, D).transpose(1, 2).reshape(-1, NKV, page, D))
    return k_pool, v_pool, perm.to(torch.int32).to(k.device).contiguous()


def trees(B, T, seed):
    """bool [B, T, T]: ancestors and self of random trees."""
    g = torch.Generator().manual_seed(seed)
    sees = torch.zeros((B, T, T), dtype=torch.bool)
    for b in range(B):
        for i in range(T):
            parent = int(torch.randint(-1, i, (1,), generator=g)) if i else -1
            if parent >= 0:
                sees[b, i] = sees[b, parent]
            sees[b, i, i] = True
    return sees


def inputs(B, NQ, NKV, D, S, T, seed=1, qstd=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    return rnd(B, NQ, T, D, std=qstd), rnd(B, NKV, S, D), rnd(B, NKV, S, D)


def lens_tensor(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")
