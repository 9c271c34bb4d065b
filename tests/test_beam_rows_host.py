"""Rows that beams go on from, on the host: parents that are none of a request's never
become an index (no GPU needed)."""
import torch

from voom_amd.kv_paged import PagedKVCache


def test_rows_of_wild_parents_are_their_own():
    parents = torch.tensor([[0, -1, 3], [2, 2 ** 31 - 1, 2], [1, 1, -2 ** 31]], dtype=torch.int32)
    assert PagedKVCache._rows_of(parents).tolist() == [0, 1, 2, 5, 4, 5, 7, 7, 8]
    g = torch.Generator().manual_seed(1)
    inside = torch.randint(0, 5, (7, 5), generator=g).int()
    want = [b * 5 + p for b, row in enumerate(inside.tolist()) for p in row]
    assert PagedKVCache._rows_of(inside).tolist() == want
