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


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E", [40, 100, 257, 512, 1024])
@pytest.mark.parametrize("T", [20, 500])
def test_masks_and_ties(L, T, E, dtype):
    """Many equal logits, both zeros, -inf and NaN (never chosen), +inf (takes all the weight), the type's lowest number (chosen in order),
    at every number of logits a lane holds. Weights: expf is within 2 units and so is each difference it is taken of, at most 32 + 5 additions make
    a sum, a division: (2 |x| + 46) * 2^-24 with |x| the largest difference of logits whose exponential is a number."""
    g = torch.Generator(device="cuda").manual_seed(T + E)
    v = torch.randint(-2, 3, (T, E), generator=g, device="cuda").to(DT[dtype])
    v[v == 0] = -0.0
    v[::2][v[::2] == 0] = 0.0
    v[0, 1::2] *= -1.0
    v[3] = -math.inf
    v[T - 1] = -math.inf
    v[5, 2:] = -math.inf
    v[6, ::3] = math.nan
    v[7] = math.nan
    v[8, 4] = math.inf
    v[9, [4, 6]] = math.inf
    v[10] = torch.finfo(DT[dtype]).min
    v[11, :30] = torch.finfo(DT[dtype]).min
    v[12] = -math.inf
    v[12, E - 1] = torch.finfo(DT[dtype]).min
    v[13, E - 1] = torch.finfo(DT[dtype]).max
    v[14] = torch.arange(E, device="cuda").to(DT[dtype])                          # ascending: the last ones, backwards (ties in 16 bits)
    v[15] = torch.finfo(DT[dtype]).tiny * torch.where(torch.arange(E, device="cuda") % 2 == 0, 0.25, -0.25)      # subnormal numbers in order
    for top_k in (4, 32):
        for renormalize in (True, False):
            got = L.moe_route(v, top_k, renormalize)
            want = W.route(v, top_k, renormalize)
            for name, a, b in zip(("experts", "offsets", "rows", "slots"), got[1:], want[1:]):
                assert torch.equal(a.cpu(), b), name
            near = v[(v > -100) & (v < 1e4)].float()
            tol = (2 * float(near.max() - near.min()) + 46) * 2.0 ** -24
            assert bool(((got[0].double().cpu() - want[0]).abs() <= tol * want[0] + 1e-37).all())
            assert bool((got[1][3] == -1).all()) and bool((got[0][3] == 0).all()) and not bool(torch.isnan(got[0]).any())
