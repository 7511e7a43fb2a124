"""GPU tests of expert routing and combine against plain loops (oracle/w4_oracle.py). Choices, offsets, rows and slots have to be
equal; weights are 32-bit softmax values: expf is within 2 units in the last place and so is the difference it is taken of, the
sum of at most 1024 of them and the division add less than 1024 + 2 roundings in the worst case -- (2 |x| + 1030) * 2^-24
with |x| the largest difference of logits."""
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


def check_route(L, logits, top_k, renormalize):
    got = L.moe_route(logits, top_k, renormalize)
    want = W.route(logits, top_k, renormalize)
    for name, a, b in zip(("experts", "offsets", "rows", "slots"), got[1:], want[1:]):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name
    finite = logits[torch.isfinite(logits)].float()
    reach = float(finite.max() - finite.min()) if finite.numel() else 0.0
    tol = (2 * reach + min(logits.shape[1], 1024) + 6) * 2.0 ** -24
    assert got[0].dtype == torch.float32 and bool(((got[0].double().cpu() - want[0]).abs() <= tol * want[0] + 1e-37).all())
    return got


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 8), (2, 33, 3), (5, 64, 8), (31, 100, 4), (32, 256, 8), (33, 16, 2), (127, 65, 6), (128, 8, 2), (129, 128, 8),
                                   (300, 257, 5), (1000, 60, 6), (130, 1024, 32), (700, 513, 1), (4097, 8, 2)])
def test_route(L, T, E, k, dtype, renormalize):
    logits = (torch.randn(T, E, generator=torch.Generator(device="cuda").manual_seed(T + E), device="cuda") * 2).to(DT[dtype])
    check_route(L, logits, k, renormalize)


@pytest.mark.parametrize("T", [20, 500])
def test_route_masks_and_ties(L, T):
    g = torch.Generator(device="cuda").manual_seed(T)
    v = torch.randint(-2, 3, (T, 40), generator=g, device="cuda").float()          # many equal logits: the lowest index wins
    v[v == 0] = -0.0
    v[::2][v[::2] == 0] = 0.0
    v[0, 1::2] *= -1.0
    v[3] = -math.inf                                                               # padding rows
    v[T - 1] = -math.inf
    v[5, 2:] = -math.inf                                                           # fewer experts than choices
    v[6, ::3] = math.nan                                                           # never chosen
    v[7] = math.nan
    v[8, 4] = math.inf                                                             # takes all the weight
    v[9, [4, 6]] = math.inf
    v[10] = torch.finfo(torch.float32).min                                         # a mask value that is a number: chosen in order
    v[11, :30] = torch.finfo(torch.float32).min
    for renormalize in (True, False):
        got = check_route(L, v, 4, renormalize)
        assert bool((got[1][3] == -1).all()) and bool((got[0][3] == 0).all()) and not bool(torch.isnan(got[0]).any())
    empty = L.moe_route(torch.full((T, 40), -math.inf, device="cuda"), 4)
    assert bool((empty[2] == 0).all()) and bool((empty[3] == -1).all()) and bool((empty[4] == -1).all()) and bool((empty[0] == 0).all())


def test_route_strides_empty_and_refusals(L):
    wide = torch.randn(200, 77, device="cuda").half()
    check_route(L, wide[:, 3:60], 4, True)
    check_route(L, wide[:50, ::2], 4, True)
    check_route(L, wide.t()[:60, :33], 3, False)
    got = L.moe_route(wide[:0], 2)
    assert got[0].shape == (0, 2) and bool((got[2] == 0).all()) and got[2].shape == (78,) and got[3].shape == (0,)
    for call in (lambda: L.moe_route(wide, 0), lambda: L.moe_route(wide, 78), lambda: L.moe_route(wide.double(), 2), lambda: L.moe_route(wide[0], 2),
                 lambda: L.moe_route(torch.zeros(2, 1025, device="cuda"), 2), lambda: L.moe_route(wide.repeat(1, 2), 33),
                 lambda: L.moe_route(wide.clone().requires_grad_(True), 2)):
        with pytest.raises(RuntimeError):
            call()


def test_route_large_batch_against_sorts(L):
    """16000 tokens: the order against torch's stable sorts (whole numbers: equal)."""
    logits = torch.randn(16000, 256, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").bfloat16()
    logits[torch.rand(16000, device="cuda") < 0.1] = -math.inf
    weights, experts, offsets, rows, slots = L.moe_route(logits, 8, True)
    v, e = torch.sort(logits.float(), dim=-1, descending=True, stable=True)
    e = torch.where(v[:, :8] > -math.inf, e[:, :8], 256)
    key, order = torch.sort(e.reshape(-1), stable=True)
    n = int((key < 256).sum())
    assert torch.equal(experts.long(), torch.where(e < 256, e, -1))
    assert torch.equal(rows[:n].long(), order[:n] // 8) and bool((rows[n:] == -1).all()) and int(offsets[-1]) == n
    assert torch.equal(offsets.long(), torch.searchsorted(key, torch.arange(257, device="cuda")))
    place = torch.full((16000 * 8,), -1, dtype=torch.int64, device="cuda")
    place[order[:n]] = torch.arange(n, device="cuda")
    assert torch.equal(slots.reshape(-1).long(), place)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,M,k", [(1, 1, 1), (3, 8, 2), (7, 100, 4), (64, 4096, 8), (33, 1001, 5), (10, 64, 32), (500, 264, 3)])
def test_combine(L, T, M, k, dtype):
    """Off by one rounding of the result and k 32-bit additions of its parts."""
    g = torch.Generator(device="cuda").manual_seed(T + M)
    y = torch.randn(T * k, M, generator=g, device="cuda").to(DT[dtype])
    slots = torch.randperm(T * k, generator=g, device="cuda").int().view(T, k)
    weights = torch.rand(T, k, generator=g, device="cuda")
    slots[T // 2, 0] = -1
    if T > 2:
        slots[1] = -1
        slots[2, 0] = T * k                                                        # outside: adds nothing
    for src in (y, torch.cat([y, y], 1)[:, 3:3 + M] if M > 3 else y):
        got = L.moe_combine(src, slots, weights)
        want, mag = W.combine(src, slots, weights)
        tol = W.half_step(DT[dtype]) * want.abs() + 2.0 ** -25 + k * 2.0 ** -24 * mag
        assert got.dtype == DT[dtype] and bool(((got.double() - want).abs() <= tol).all())
    if T > 2:
        assert bool((got[1] == 0).all())


def test_combine_unused_rows_and_refusals(L):
    y = torch.ones(6, 16, dtype=torch.float16, device="cuda")
    y[4:] = float("nan")                                                           # rows no slot names
    slots = torch.tensor([[0, 1], [2, -1], [-1, -1]], dtype=torch.int32, device="cuda")
    weights = torch.tensor([[0.25, 0.5], [1.0, float("nan")], [0.0, 0.0]], device="cuda")
    got = L.moe_combine(y, slots, weights)
    assert got[:, 0].tolist() == [0.75, 1.0, 0.0]
    assert L.moe_combine(y, slots[:0], weights[:0]).shape == (0, 16)
    assert bool((L.moe_combine(y[:0], slots, weights) == 0).all())
    for call in (lambda: L.moe_combine(y.float(), slots, weights), lambda: L.moe_combine(y, slots.long(), weights), lambda: L.moe_combine(y, slots, weights.half()),
                 lambda: L.moe_combine(y, slots, weights[:, :1]), lambda: L.moe_combine(y[0], slots, weights), lambda: L.moe_combine(y, slots.cpu(), weights),
                 lambda: L.moe_combine(y.clone().requires_grad_(True), slots, weights)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M", [1, 7, 8, 9, 15, 16, 20, 22, 41, 1025])
def test_combine_any_alignment(L, M, dtype):
    """Rows on every even address, in and out (the result's rows follow one another, M values apart): the sums are those of
    16-byte aligned rows, bit for bit."""
    g = torch.Generator(device="cuda").manual_seed(M)
    T, k = 13, 5
    y = torch.randn(T * k, M, generator=g, device="cuda").to(DT[dtype])
    slots = torch.randperm(T * k, generator=g, device="cuda").int().view(T, k)
    weights = torch.rand(T, k, generator=g, device="cuda")
    room = torch.zeros(T * k, (M + 7) // 8 * 8, dtype=DT[dtype], device="cuda")
    room[:, :M] = y
    want = L.moe_combine(room, slots, weights)[:, :M]
    ref, mag = W.combine(y, slots, weights)
    assert bool(((want.double() - ref).abs() <= W.half_step(DT[dtype]) * ref.abs() + 2.0 ** -25 + k * 2.0 ** -24 * mag).all())
    for pitch in (M, M + 1, M + 2, M + 4, M + 8):
        for start in (0, 1, 2, 4):
            buf = torch.full((T * k * pitch + start + 8,), float("nan"), dtype=DT[dtype], device="cuda")
            src = buf[start:start + T * k * pitch].view(T * k, pitch)[:, :M]
            src.copy_(y)
            assert torch.equal(L.moe_combine(src, slots, weights), want)
