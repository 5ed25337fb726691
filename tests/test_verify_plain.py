"""The host's form of verify_drafts: it refuses what the kernel's form refuses, and walks 64-bit and odd rows alike."""
from __future__ import annotations

import pytest
import torch

from model.speculative import plain_verify


def args(**kw):
    p = torch.rand(5, 9)
    return {**dict(probs=p, tokens=torch.zeros(5, dtype=torch.int64), cu_seqlens=torch.tensor([0, 3, 5], dtype=torch.int32)), **kw}


BAD = {
    "probs of one row": lambda: args(probs=torch.rand(9)), "no vocabulary": lambda: args(probs=torch.rand(5, 0)),
    "whole numbers": lambda: args(probs=torch.ones(5, 9, dtype=torch.int64)),
    "tokens int32": lambda: args(tokens=torch.zeros(5, dtype=torch.int32)), "tokens of 4": lambda: args(tokens=torch.zeros(4, dtype=torch.int64)),
    "parents int64": lambda: args(parents=torch.zeros(5, dtype=torch.int64)), "parents of 4": lambda: args(parents=torch.zeros(4, dtype=torch.int32)),
    "draft without uniforms": lambda: args(draft_probs=torch.rand(5, 9)),
    "draft of another shape": lambda: args(draft_probs=torch.rand(5, 8), uniforms=torch.rand(5)),
    "draft of whole numbers": lambda: args(draft_probs=torch.ones(5, 9, dtype=torch.int32), uniforms=torch.rand(5)),
    "uniforms of whole numbers": lambda: args(uniforms=torch.zeros(5, dtype=torch.int64)), "uniforms of 4": lambda: args(uniforms=torch.rand(4)),
    "bounds int64": lambda: args(cu_seqlens=torch.tensor([0, 3, 5])), "bounds of two dimensions": lambda: args(cu_seqlens=torch.zeros(1, 2, dtype=torch.int32)),
}


@pytest.mark.parametrize("what", BAD)
def test_refused(what):
    with pytest.raises((TypeError, ValueError), match="mhc_amd"):
        plain_verify(**BAD[what]())


def test_verify_step_refuses_drafts_without_numbers():
    from test_paged import batch, pages, tiny
    model = tiny()
    cache = pages(model, 1)
    with pytest.raises(ValueError, match="uniforms"):
        model.verify_step(torch.zeros(1, 3, dtype=torch.int64), batch([3]), cache, draft_probs=torch.rand(3, 50))
    assert cache.lengths.tolist() == [0]


def test_greedy_rows_of_64_bits_and_without_finite_numbers():
    """The first of the largest numbers: not of their fp32 roundings, and never a NaN."""
    nan, inf = float("nan"), float("inf")
    rows = torch.tensor([[1.0, 1.0 + 2.0 ** -40, 0.5], [nan, -inf, -inf], [nan, nan, nan], [-inf, -inf, nan],
                         [-3.0, nan, -2.0]], dtype=torch.float64)
    cu = torch.arange(6, dtype=torch.int32)
    kept, path, following = plain_verify(rows, torch.zeros(5, dtype=torch.int64), cu)
    assert following.tolist() == [1, 1, -1, 0, 2] and kept.tolist() == [1] * 5
    # drafts after each: accepted where they are that token
    both = rows.repeat_interleave(2, 0)
    tokens = torch.tensor([0, 1, 0, 1, 0, 0, 0, 0, 0, 2])
    kept, _, _ = plain_verify(both, tokens, torch.arange(0, 11, 2, dtype=torch.int32))
    assert kept.tolist() == [2, 2, 1, 2, 2]
