"""Verification of drafted tokens at the ends of its arguments' ranges."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error(cuda_device):
    from robustgemq_b200 import _lib

    _lib.device_error()
    yield
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("temperature", [1e-30, 1e-38, 3e-39, 1e-41, 1.4e-45])
def test_the_smallest_temperatures_are_greedy(dtype, probs, temperature):
    """All of the probability on a maximum that stands apart, as T goes to 0, down to the
    smallest subnormal: the greedy form's tokens, and log probabilities of 0."""
    from robustgemq_b200.serving import verify_draft

    g = torch.Generator(device="cuda").manual_seed(3)
    B, n, V = 6, 3, 2003
    logits = torch.randn((B, n + 1, V), generator=g, device="cuda")
    top = torch.randint(0, V, (B, n + 1), generator=g, device="cuda")
    logits.scatter_(-1, top[..., None], 9.0)
    drafts = top[:, :n].clone()
    drafts[1::2, 1] = (drafts[1::2, 1] + 1) % V
    q = torch.softmax(torch.randn((B, n, V), generator=g, device="cuda"), -1) if probs else None
    u = torch.rand((B, n), generator=g, device="cuda")
    e = torch.empty((B, V), device="cuda").exponential_(generator=g)
    args = (logits.to(dtype), drafts, u, e)
    want = verify_draft(*args, draft_probs=q, temperature=torch.zeros(B, device="cuda"))
    got = verify_draft(*args, draft_probs=q, temperature=torch.full((B,), temperature, device="cuda"))
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.num_accepted, want.num_accepted)
    assert want.num_accepted.tolist() == [n, 1] * 3 and (got.logprobs == 0).all()
