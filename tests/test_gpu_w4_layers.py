"""GPU tests of W4Linear and W4Experts: the operators run together as a model runs them. Each stage is held to its own 64-bit
oracle on the stage's own inputs (tolerances of w4_oracle), and the layer's result to the stages' bit for bit."""
import copy

import pytest
import torch

import w4_oracle as W

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def L():
    import lowbit_kernel

    return lowbit_kernel


@pytest.fixture(scope="module")
def N():
    import bgemm_linear

    return bgemm_linear


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check_linear(got, x, plane, scales, zeros, K, group):
    want = W.linear(x, W.values(plane, scales, zeros, K, group))
    assert bool(((got.double() - want).abs() <= W.linear_tolerance(x, want, plane, scales, zeros, K, group)).all())


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_w4_linear_layer(N, dtype, symmetric):
    g = gen(1)
    w = torch.randn(300, 520, generator=g, device="cuda").to(DT[dtype]) * 0.05
    bias = torch.randn(300, generator=g, device="cuda")
    layer = N.W4Linear(w, 64, symmetric, bias)
    assert (layer.zeros is None) == symmetric
    q, s, z = W.quantize(w, 64, symmetric, DT[dtype])
    assert torch.equal(layer.dequantized(), W.values(W.pack(q), s, z, 520, 64).to(DT[dtype]))
    for lead in ((3,), (2, 5), (2, 3, 20), (0,)):
        x = torch.randn(*lead, 520, generator=g, device="cuda").to(DT[dtype])
        got = layer(x)
        assert got.shape == lead + (300,) and got.dtype == DT[dtype]
        if x.numel():
            plain = N.W4Linear(w, 64, symmetric)(x)
            check_linear(plain.reshape(-1, 300), x.reshape(-1, 520), layer.plane, layer.scales, layer.zeros, 520, 64)
            assert torch.equal(got, plain + bias.to(DT[dtype]))
    other = N.W4Linear(torch.zeros_like(w), 64, symmetric, torch.zeros_like(bias))
    other.load_state_dict(copy.deepcopy(layer.state_dict()))
    x = torch.randn(4, 520, generator=g, device="cuda").to(DT[dtype])
    assert torch.equal(other(x), layer(x))
    with pytest.raises(RuntimeError):
        layer(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError):
        layer(x.float())
    with pytest.raises(ValueError):
        N.W4Linear(w[0])


def test_w4_linear_types(N):
    w = torch.randn(64, 128, generator=gen(2), device="cuda")
    assert N.W4Linear(w).scales.dtype == torch.float16
    assert N.W4Linear(w, dtype=torch.bfloat16).scales.dtype == torch.bfloat16
    half = N.W4Linear(w.half(), dtype=torch.bfloat16)
    assert half.scales.dtype == torch.bfloat16 and half(torch.ones(1, 128, device="cuda", dtype=torch.bfloat16)).dtype == torch.bfloat16
    with torch.no_grad():
        assert N.W4Linear(torch.nn.Parameter(w)).plane.shape == (64, 64)


def staged(L, layer, x, logits):
    weights, experts, offsets, rows, slots = L.moe_route(logits, layer.top_k, layer.renormalize)
    h = L.w4a16_grouped_forward(x, layer.gate_up_plane, layer.gate_up_scales, layer.gate_up_zeros, offsets, rows, layer.group_size)
    a = torch.nn.functional.silu(h[:, :layer.intermediate_size]) * h[:, layer.intermediate_size:]
    y = L.w4a16_grouped_forward(a, layer.down_plane, layer.down_scales, layer.down_zeros, offsets, None, layer.group_size)
    return (weights, experts, offsets, rows, slots), h, a, y, L.moe_combine(y, slots, weights)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,E,H,I,k", [(1, 8, 256, 192, 2), (5, 16, 520, 136, 4), (40, 8, 384, 256, 2), (150, 4, 256, 320, 3), (300, 33, 136, 64, 6)])
def test_w4_experts_layer(L, N, T, E, H, I, k, dtype):
    g = gen(T + E)
    gate_up = torch.randn(E, 2 * I, H, generator=g, device="cuda").to(DT[dtype]) * 0.06
    down = torch.randn(E, H, I, generator=g, device="cuda").to(DT[dtype]) * 0.06
    layer = N.W4Experts(gate_up, down, k, renormalize=T % 2 == 0, group_size=64)
    x = torch.randn(T, H, generator=g, device="cuda").to(DT[dtype])
    logits = torch.randn(T, E, generator=g, device="cuda")
    if T > 4:
        logits[T // 2] = -float("inf")                                # a padding row
        logits[1, 1:] = -float("inf")                                 # one expert left
    got = layer(x, logits)
    (weights, experts, offsets, rows, slots), h, a, y, out = staged(L, layer, x, logits)
    assert torch.equal(got, out)
    want = W.route(logits, k, T % 2 == 0)
    for have, ref in zip((experts, offsets, rows, slots), want[1:]):
        assert torch.equal(have.cpu(), ref)
    at = offsets.tolist()
    for e in range(E):
        if at[e + 1] > at[e]:
            sl = slice(at[e], at[e + 1])
            check_linear(h[sl], x[rows[sl].long()], layer.gate_up_plane[e], layer.gate_up_scales[e], layer.gate_up_zeros[e], H, 64)
            check_linear(y[sl], a[sl], layer.down_plane[e], layer.down_scales[e], layer.down_zeros[e], I, 64)
    ref, mag = W.combine(torch.where(torch.isfinite(y), y, 0), slots, weights)
    assert bool(((got.double() - ref).abs() <= W.half_step(DT[dtype]) * ref.abs() + 2.0 ** -25 + k * 2.0 ** -24 * mag).all())
    if T > 4:
        assert bool((got[T // 2] == 0).all())
    assert torch.equal(layer(x.reshape(1, T, H), logits.reshape(1, T, E))[0], got)
    assert layer(x[:0], logits[:0]).shape == (0, H)
    with pytest.raises(ValueError):
        layer(x, logits[:, :-1])


def test_w4_experts_captured_and_replayed(N):
    """A captured forward serves other tokens with another routing: nothing of the host's view of the first is kept."""
    g = gen(9)
    E, H, I, T = 8, 256, 128, 48
    layer = N.W4Experts(torch.randn(E, 2 * I, H, generator=g, device="cuda").bfloat16() * 0.06, torch.randn(E, H, I, generator=g, device="cuda").bfloat16() * 0.06, 2)
    xs = torch.randn(3, T, H, generator=g, device="cuda").bfloat16()
    ls = torch.randn(3, T, E, generator=g, device="cuda")
    ls[1, :, 1:3] += 9.0                                              # everybody to two experts
    ls[2, 10:] = -float("inf")                                        # mostly padding
    want = [layer(x, lg) for x, lg in zip(xs, ls)]
    sx, sl = xs[0].clone(), ls[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(sx, sl)
    for i in (1, 0, 2, 1):
        sx.copy_(xs[i])
        sl.copy_(ls[i])
        graph.replay()
        assert torch.equal(out, want[i])


def test_ctypes_binding_gives_the_same(L):
    import bgemm_b200 as B

    g = gen(4)
    w = torch.randn(3, 130, 264, generator=g, device="cuda").half() * 0.05
    for sym in (False, True):
        a, b = L.w4_quantize(w, 32, sym), B.w4_quantize(w, 32, sym)
        assert all(p is q is None or torch.equal(p, q) for p, q in zip(a, b))
        plane, scales, zeros = b
        assert torch.equal(L.w4_dequantize(plane, scales, zeros, 264, 32), B.w4_dequantize(plane, scales, zeros, 264, 32))
        for n in (3, 90):
            x = torch.randn(n, 264, generator=g, device="cuda").half()
            z0 = None if zeros is None else zeros[0]
            assert torch.equal(L.w4a16_linear_forward(x, plane[0], scales[0], z0, 32), B.w4a16_gemm(x, plane[0], scales[0], z0, 32))
            wide = torch.zeros(n, 140, dtype=torch.float16, device="cuda")
            B.w4a16_gemm(x, plane[0], scales[0], z0, 32, out=wide[:, 5:135])
            assert torch.equal(wide[:, 5:135], L.w4a16_linear_forward(x, plane[0], scales[0], z0, 32)) and bool((wide[:, :5] == 0).all())
            off = torch.tensor([0, n // 3, n // 2, n], dtype=torch.int32, device="cuda")
            rows = torch.randint(0, n, (n,), generator=g, device="cuda", dtype=torch.int32)
            for r in (None, rows):
                assert torch.equal(L.w4a16_grouped_forward(x, plane, scales, zeros, off, r, 32), B.w4a16_grouped_gemm(x, plane, scales, zeros, off, r, 32))
    for T in (5, 200):
        logits = torch.randn(T, 12, generator=g, device="cuda")
        assert all(torch.equal(p, q) for p, q in zip(L.moe_route(logits, 3, False), B.moe_route(logits, 3, False)))
        weights, _, _, _, slots = B.moe_route(logits, 3)
        y = torch.randn(T * 3, 24, generator=g, device="cuda").half()
        assert torch.equal(L.moe_combine(y, slots, weights), B.moe_combine(y, slots, weights))
    x = torch.randn(2, 264, device="cuda").half()
    for call in (lambda: B.w4a16_gemm(x.bfloat16(), plane[0], scales[0], None, 32), lambda: B.w4a16_gemm(x[:, :200], plane[0], scales[0], None, 32),
                 lambda: B.w4a16_grouped_gemm(x, plane, scales, None, torch.zeros(3, dtype=torch.int32, device="cuda"), None, 32), lambda: B.w4_quantize(w[0, 0]),
                 lambda: B.moe_combine(x, torch.zeros(1, 1, device="cuda"), torch.zeros(1, 1, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(B.BgemmError):
        B.moe_route(torch.zeros(2, 8, device="cuda"), 9)


def test_layers_refuse_other_widths_and_types(N):
    """[4, 2 H] is not taken for eight tokens of width H."""
    g = gen(15)
    H, I, E = 64, 32, 4
    gate_up, down = torch.randn(E, 2 * I, H, generator=g, device="cuda").half(), torch.randn(E, H, I, generator=g, device="cuda").half()
    layer, linear = N.W4Experts(gate_up, down, 2), N.W4Linear(gate_up[0])
    x, logits = torch.randn(4, 2 * H, generator=g, device="cuda").half(), torch.randn(4, E, generator=g, device="cuda")
    for call in (lambda: layer(x, logits), lambda: linear(x), lambda: linear(x[:, :32]), lambda: layer(x[:, :H], logits[:3]),
                 lambda: N.W4Linear(gate_up[0], dtype=torch.float32), lambda: N.W4Experts(gate_up, down, 2, dtype=torch.int8)):
        with pytest.raises(ValueError):
            call()
    assert layer(x[:, :H], logits).shape == (4, H) and linear(x[0, :H]).shape == (2 * I,)


def test_layers_saved_before_they_had_a_choice_of_arithmetic(N):
    """A pickled layer has the attributes of its time: without `exact` it behaves as it did."""
    import pickle

    g = gen(16)
    linear = N.W4Linear(torch.randn(64, 128, generator=g, device="cuda").half())
    experts = N.W4Experts(torch.randn(4, 64, 64, generator=g, device="cuda").half(), torch.randn(4, 64, 32, generator=g, device="cuda").half(), 2)
    x, logits = torch.randn(5, 128, generator=g, device="cuda").half(), torch.randn(5, 4, generator=g, device="cuda")
    want = linear(x), experts(x[:, :64], logits)
    for layer in (linear, experts):
        del layer.exact
    linear, experts = pickle.loads(pickle.dumps(linear)), pickle.loads(pickle.dumps(experts))
    assert torch.equal(linear(x), want[0]) and torch.equal(experts(x[:, :64], logits), want[1])
    with torch.inference_mode():
        assert torch.equal(linear(x), want[0]) and torch.equal(experts(x[:, :64], logits), want[1])


def test_the_first_call_of_a_process_may_be_a_captured_one():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import sys; sys.path[:0] = [sys.argv[1]]
import torch, lowbit_kernel as L
g = torch.Generator(device="cuda").manual_seed(0)
plane = torch.randint(0, 256, (4, 2048, 1024), generator=g, device="cuda", dtype=torch.uint8)
scales = torch.ones(4, 2048, 16, device="cuda", dtype=torch.bfloat16)
off, rows = torch.tensor([0, 100, 200, 300, 400], dtype=torch.int32, device="cuda"), torch.arange(400, device="cuda").int()
x, logits = torch.randn(400, 2048, generator=g, device="cuda").bfloat16(), torch.randn(400, 64, generator=g, device="cuda")
torch.cuda.synchronize()
def calls():
    r = L.moe_route(logits, 4)
    return [L.w4a16_grouped_forward(x, plane, scales, None, off, rows, 128), L.w4a16_linear_forward(x[:3], plane[0], scales[0], None, 128), *r, L.moe_combine(x, r[4][:100], r[0][:100]),
            *L.w4_quantize(x), L.w4_dequantize(plane, scales, None, 2048, 128)]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = calls()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, calls()))
"""
    root = Path(__file__).resolve().parent.parent / "bgemm-cuda_b200"
    subprocess.run([sys.executable, "-c", code, str(root)], check=True, timeout=240)
