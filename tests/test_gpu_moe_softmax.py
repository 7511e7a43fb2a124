"""GPU tests of the routing's softmax and of its 16-bit selection (keys that carry their expert, a sort per lane), against the plain
loops of oracle/w4_oracle.py."""
import math

import pytest
import torch

import w4_oracle as W

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def L():
    import lowbit_kernel

    return lowbit_kernel


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T", [100, 3000])
@pytest.mark.parametrize("E", [2, 8, 31, 32])
def test_both_softmaxes_are_one_where_every_expert_is_chosen(L, E, T, dtype):
    """top_k = E and logits in descending order: the sum over all experts has the terms of the sum over the chosen, on the same lanes in
    the same order, so the weights are equal bit for bit."""
    logits = (torch.randn(T, E, generator=torch.Generator(device="cuda").manual_seed(E), device="cuda") * 4).to(DT[dtype])
    logits = torch.sort(logits, dim=1, descending=True).values
    a, b = L.moe_route(logits, E, True), L.moe_route(logits, E, False)
    assert torch.equal(a[1], torch.arange(E, device="cuda").int().expand(T, E)) and torch.equal(a[1], b[1])
    assert torch.equal(a[0], b[0])
