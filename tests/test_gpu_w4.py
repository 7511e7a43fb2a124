"""GPU tests of the 4-bit weight operators against the plain 64-bit implementations of oracle/w4_oracle.py. Tolerances are
w4_oracle.linear_tolerance (roundings counted one by one) unless a test says exact."""
import os

import pytest
import torch

import w4_oracle as W

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def L():
    import lowbit_kernel

    return lowbit_kernel


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def matrix(lead, M, K, group, dtype, with_zeros, g, fill=0):
    """Random codes of the whole range with random padding behind K; scales of both signs' magnitude range."""
    shape = tuple(lead) + (M, K)
    plane = W.pack(torch.randint(0, 16, shape, generator=g, device="cuda"), fill)
    sshape = tuple(lead) + (M, -(-K // group))
    scales = (torch.randn(sshape, generator=g, device="cuda") * 0.5 - 4.5).exp().to(dtype)
    zeros = torch.randint(0, 16, sshape, generator=g, device="cuda", dtype=torch.uint8) if with_zeros else None
    return plane, scales, zeros


def check_linear(got, x, plane, scales, zeros, K, group):
    want = W.linear(x, W.values(plane, scales, zeros, K, group))
    tol = W.linear_tolerance(x, want, plane, scales, zeros, K, group)
    off = (got.double() - want).abs()
    assert got.dtype == x.dtype and bool((off <= tol).all()), f"largest error {float((off / tol).max()):.3g} of the tolerance"


# ---- quantize / dequantize -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("M,K,group", [(1, 1, 32), (3, 31, 32), (5, 128, 128), (7, 200, 64), (130, 1000, 32), (64, 4100, 128), (33, 257, 64), (256, 2048, 128)])
def test_quantize_bits(L, M, K, group, dtype, symmetric):
    w = (torch.randn(M, K, generator=gen(M + K), device="cuda") * 0.05).to(DT[dtype])
    w[M // 2] = 0                                                    # groups of zeros: scale 0
    plane, scales, zeros = L.w4_quantize(w, group, symmetric)
    kind = torch.float16 if dtype == "fp32" else DT[dtype]
    codes, s, z = W.quantize(w, group, symmetric, kind)
    assert plane.shape == (M, W.row_bytes(K)) and scales.dtype == kind
    assert torch.equal(scales, s) and torch.equal(W.unpack(plane, K), codes)
    assert (zeros is None) == symmetric and (symmetric or torch.equal(zeros, z))
    # every value within half a step of the weight, a step being the scale: the ends of the range are rounded with the scale
    # (half a step of 16 bits, times 15) and a zero point that is rounded clips by at most half a step more
    err = (W.values(plane, scales, zeros, K, group) - w.double()).abs()
    step = W.spread(scales.double(), K, group)
    slack = step * (0.5 if symmetric else 1.0) + step * 15 * W.half_step(kind) + step * 1e-5 + 2.0 ** -24
    assert bool((err <= slack).all())
    got = L.w4_dequantize(plane, scales, zeros, K, group)
    assert torch.equal(got, W.values(plane, scales, zeros, K, group).to(kind))     # products of 11 and 5 bits are exact in 64: one rounding


def test_quantize_ties_strides_and_stacks(L):
    g = gen(5)
    # w / s exactly on halves: s = 2^-4 in a group whose extremes are 15 s apart, elements k + 1/2 steps
    steps = torch.randint(0, 29, (64, 256), generator=g, device="cuda").float() / 2 - 7
    steps[:, ::32] = -7.5
    steps[:, 1::32] = 7.5
    w = (steps / 16).half()
    plane, scales, zeros = L.w4_quantize(w, 32, False)
    codes, s, z = W.quantize(w, 32, False, torch.float16)
    assert torch.equal(scales, s) and torch.equal(zeros, z) and torch.equal(W.unpack(plane, 256), codes)
    # rows of a wider matrix (not 16-byte aligned), a transposed one, a stack with a pitch of its own
    wide = torch.randn(3, 40, 333, generator=g, device="cuda").bfloat16()
    for v in (wide[:, :, 5:205], wide[:, ::2, :200], wide.transpose(1, 2)[:, :, :33]):
        plane, scales, zeros = L.w4_quantize(v, 64, False)
        for b in range(3):
            codes, s, z = W.quantize(v[b].contiguous(), 64, False, torch.bfloat16)
            assert torch.equal(scales[b], s) and torch.equal(zeros[b], z) and torch.equal(W.unpack(plane[b], v.shape[2]), codes)
    got = L.w4_dequantize(plane, scales, zeros, 33, 64)
    assert torch.equal(got, W.values(plane, scales, zeros, 33, 64).bfloat16())


# ---- linear ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,group", [(1, 1, 1, 32), (16, 128, 1, 128), (17, 129, 2, 32), (100, 1000, 7, 64), (128, 256, 8, 128), (33, 2056, 9, 32),
                                         (512, 4096, 1, 128), (300, 1111, 16, 64), (129, 640, 17, 128), (256, 1024, 33, 32), (130, 520, 64, 64),
                                         (1000, 2048, 100, 128), (257, 4104, 255, 64), (384, 1536, 300, 128), (128, 128, 513, 32), (5000, 264, 40, 128)])
def test_linear(L, M, K, N, group, dtype, with_zeros):
    g = gen(M * 7 + K + N)
    plane, scales, zeros = matrix((), M, K, group, DT[dtype], with_zeros, g, fill=15)
    x = torch.randn(N, K, generator=g, device="cuda").to(DT[dtype])
    check_linear(L.w4a16_linear_forward(x, plane, scales, zeros, group), x, plane, scales, zeros, K, group)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(200, 700, 5), (129, 1300, 70), (640, 384, 200)])
def test_linear_whole_numbers_are_exact(L, M, K, N, dtype):
    """Scales that are powers of two and small whole activations: every product and sum is exact in 32 bits and every weight
    in 16, so any kernel must return the rounded exact result bit for bit."""
    g = gen(3 + M)
    plane, scales, zeros = matrix((), M, K, 64, DT[dtype], True, g, fill=9)
    scales = (2.0 ** torch.randint(-2, 2, scales.shape, generator=g, device="cuda")).to(DT[dtype])
    x = torch.randint(-3, 4, (N, K), generator=g, device="cuda").to(DT[dtype])
    want = W.linear(x, W.values(plane, scales, zeros, K, 64)).to(DT[dtype])
    assert torch.equal(L.w4a16_linear_forward(x, plane, scales, zeros, 64), want)


@pytest.mark.parametrize("N", [1, 3, 40, 140])
def test_linear_strides(L, N):
    """x as a slice of a wider matrix whose rows start anywhere, and transposed; the result is a fresh contiguous tensor."""
    g = gen(N)
    M, K, group = 160, 392, 32
    plane, scales, zeros = matrix((), M, K, group, torch.bfloat16, True, g)
    wide = torch.randn(N, 811, generator=g, device="cuda").bfloat16()
    aligned = torch.randn(N, 800, generator=g, device="cuda").bfloat16()
    tall = torch.randn(K, N, generator=g, device="cuda").bfloat16()
    for x in (wide[:, 3:3 + K], wide[:, 8:8 + K], aligned[:, 8:8 + K], tall.t(), wide[:1, :K].expand(N, K)):
        got = L.w4a16_linear_forward(x, plane, scales, zeros, group)
        assert got.is_contiguous()
        check_linear(got, x, plane, scales, zeros, K, group)


@pytest.mark.parametrize("N", [1, 4, 20, 150])
def test_linear_rows_do_not_touch_each_other(L, N):
    """Inf and NaN in one row of x leave the other rows as they are, bit for bit; that row's results are not finite."""
    g = gen(N)
    plane, scales, zeros = matrix((), 130, 520, 128, torch.float16, True, g)
    x = torch.randn(N + 1, 520, generator=g, device="cuda").half()
    clean = L.w4a16_linear_forward(x, plane, scales, zeros, 128)
    x2 = x.clone()
    x2[N // 2, 7] = float("inf")
    x2[N // 2, 300] = float("nan")
    got = L.w4a16_linear_forward(x2, plane, scales, zeros, 128)
    keep = [n for n in range(N + 1) if n != N // 2]
    assert torch.equal(got[keep], clean[keep]) and not bool(torch.isfinite(got[N // 2]).any())


def test_linear_zero_point_uses_its_low_four_bits(L):
    g = gen(9)
    plane, scales, zeros = matrix((), 64, 256, 64, torch.bfloat16, True, g)
    for N in (2, 60):
        x = torch.randn(N, 256, generator=g, device="cuda").bfloat16()
        assert torch.equal(L.w4a16_linear_forward(x, plane, scales, zeros, 64), L.w4a16_linear_forward(x, plane, scales, zeros | 0xF0, 64))
    assert torch.equal(L.w4_dequantize(plane, scales, zeros, 256, 64), L.w4_dequantize(plane, scales, zeros | 0xF0, 256, 64))


def test_empty_and_refused_calls(L):
    g = gen(2)
    plane, scales, zeros = matrix((), 8, 64, 32, torch.float16, True, g)
    x = torch.randn(2, 64, generator=g, device="cuda").half()
    assert L.w4a16_linear_forward(x[:0], plane, scales, zeros, 32).shape == (0, 8)
    bad = [lambda: L.w4a16_linear_forward(x.bfloat16(), plane, scales, zeros, 32),                  # types differ
           lambda: L.w4a16_linear_forward(x.float(), plane, scales, zeros, 32),
           lambda: L.w4a16_linear_forward(x, plane, scales, zeros, 64),                             # scales of another group size
           lambda: L.w4a16_linear_forward(x, plane, scales, zeros[:, :1], 32),
           lambda: L.w4a16_linear_forward(x, plane, scales, zeros.int(), 32),
           lambda: L.w4a16_linear_forward(x, plane[:, ::2], scales, zeros, 32),
           lambda: L.w4a16_linear_forward(x[:, :40], plane, scales[:, :1], None, 128 + 32),
           lambda: L.w4a16_linear_forward(x[0], plane, scales, zeros, 32),
           lambda: L.w4a16_linear_forward(x.clone().requires_grad_(True), plane, scales, zeros, 32),
           lambda: L.w4_quantize(x.double(), 32), lambda: L.w4_quantize(x, 16), lambda: L.w4_quantize(x[0], 32), lambda: L.w4_quantize(x[:0], 32),
           lambda: L.w4_dequantize(plane, scales, zeros, 200, 32)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        L.w4a16_linear_forward(x.clone().requires_grad_(True), plane, scales, zeros, 32)


# ---- grouped by expert -----------------------------------------------------------------------------------------------
def ragged(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


COUNTS = [[1], [0, 3, 0], [8, 0, 1, 2], [0] * 40 + [5] + [0] * 30, [1] * 70, [40, 1, 0, 17, 16, 9], [300, 0, 5, 129], [64, 64, 65, 63], [700, 2]]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("counts", COUNTS, ids=[str(i) for i in range(len(COUNTS))])
def test_grouped(L, counts, dtype, gather):
    g = gen(len(counts) + sum(counts))
    E, M, K, group = len(counts), 150, 328, 64
    plane, scales, zeros = matrix((E,), M, K, group, DT[dtype], True, g, fill=3)
    offsets, slots = ragged(counts), sum(counts)
    T = 11 if gather else slots
    x = torch.randn(T, K, generator=g, device="cuda").to(DT[dtype])
    rows = torch.randint(0, T, (slots,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, offsets, rows, group)
    src = x[rows.long()] if gather else x
    at = offsets.tolist()
    for e in range(E):
        if counts[e]:
            check_linear(got[at[e]:at[e + 1]], src[at[e]:at[e + 1]], plane[e], scales[e], zeros[e], K, group)


@pytest.mark.parametrize("slots", [7, 30, 400])
def test_grouped_leaves_other_rows_alone(L, slots):
    """Rows behind offsets[E] keep what the buffer held, also in a buffer with a row pitch of its own; an index outside x is
    a row of zeros; a repeated index is read twice."""
    g = gen(slots)
    E, M, K, group = 3, 70, 256, 128
    plane, scales, zeros = matrix((E,), M, K, group, torch.float16, True, g)
    n = slots - 3
    offsets = torch.tensor([0, n // 3, n // 3, n], dtype=torch.int32, device="cuda")
    x = torch.randn(5, K, generator=g, device="cuda").half()
    rows = torch.randint(0, 5, (slots,), generator=g, device="cuda", dtype=torch.int32)
    rows[0], rows[n - 1], rows[1] = -1, 5, rows[2]
    buf = torch.full((slots, M + 9), 77.0, dtype=torch.float16, device="cuda")
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, offsets, rows, group, buf[:, 4:4 + M])
    assert got.data_ptr() == buf[:, 4:].data_ptr()
    assert bool((buf[n:] == 77).all()) and bool((buf[:, :4] == 77).all()) and bool((buf[:, 4 + M:] == 77).all())
    assert bool((got[0] == 0).all()) and bool((got[n - 1] == 0).all())
    src = torch.where(((rows >= 0) & (rows < 5))[:, None], x[rows.clamp(0, 4).long()], 0)
    for e, (a, b) in enumerate(((0, n // 3), (n // 3, n // 3), (n // 3, n))):
        if b > a:
            check_linear(got[a:b], src[a:b], plane[e], scales[e], zeros[e], K, group)


@pytest.mark.parametrize("slots", [6, 200])
def test_grouped_offsets_that_make_no_sense_stay_in_bounds(L, slots):
    """The host cannot look at the offsets: whatever they hold, nothing outside the buffers is read or written (the ranges are
    clamped), and the rows around the result keep their values."""
    g = gen(1)
    E, M, K = 4, 64, 128
    plane, scales, zeros = matrix((E,), M, K, 128, torch.bfloat16, False, g)
    x = torch.randn(slots, K, generator=g, device="cuda").bfloat16()
    buf = torch.full((slots + 16, M), 5.0, dtype=torch.bfloat16, device="cuda")
    for bad in ([0, 1 << 30, 3, -7, 9], [-5, -4, -3, -2, -1], [slots + 1] * 5, [0, 2, 1, slots + 90, slots + 100], [2 ** 31 - 1, -2 ** 31, 0, 2 ** 31 - 1, 1]):
        L.w4a16_grouped_forward(x, plane, scales, zeros, torch.tensor(bad, dtype=torch.int32, device="cuda"), None, 128, buf[8:8 + slots])
        torch.cuda.synchronize()
        assert bool((buf[:8] == 5).all()) and bool((buf[8 + slots:] == 5).all())


def test_grouped_refusals(L):
    g = gen(4)
    plane, scales, zeros = matrix((2,), 16, 64, 64, torch.float16, True, g)
    x = torch.randn(4, 64, generator=g, device="cuda").half()
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    rows = torch.zeros(4, dtype=torch.int32, device="cuda")
    bad = [lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off[:2], None, 64), lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off.long(), None, 64),
           lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off.cpu(), None, 64), lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off, rows.long(), 64),
           lambda: L.w4a16_grouped_forward(x, plane[0], scales[0], zeros[0], off, None, 64), lambda: L.w4a16_grouped_forward(x, plane, scales[:1], None, off, None, 64),
           lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, 64, torch.empty(3, 16, dtype=torch.float16, device="cuda")),
           lambda: L.w4a16_grouped_forward(x[:0], plane, scales, zeros, off, rows, 64)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    assert L.w4a16_grouped_forward(x[:0], plane, scales, zeros, off * 0, None, 64).shape == (0, 16)


def test_two_streams_and_graphs(L):
    """The same call on two streams at once, and captured into two graphs that are replayed in turn with new inputs: the
    results are those of plain calls, bit for bit."""
    g = gen(6)
    E, M, K, group = 6, 512, 1024, 128
    plane, scales, zeros = matrix((E,), M, K, group, torch.bfloat16, True, g)
    xs = [torch.randn(96, K, generator=g, device="cuda").bfloat16() for _ in range(4)]
    off = ragged([30, 0, 1, 40, 20, 5])
    single = lambda x: L.w4a16_linear_forward(x, plane[0], scales[0], zeros[0], group)      # noqa: E731
    stacked = lambda x: L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, group)  # noqa: E731
    want = [(single(x), single(x[:3]), stacked(x)) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for x, st in zip(xs, streams):
        with torch.cuda.stream(st):
            got.append((single(x), single(x[:3]), stacked(x)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, o in zip(want, got) for a, b in zip(w, o))
    static, graphs = [x.clone() for x in xs[:2]], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = (single(x), single(x[:3]), stacked(x))
        graphs.append((graph, out))
    for turn in range(2):
        for i, (graph, out) in enumerate(graphs):
            static[i].copy_(xs[2 * turn + i])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want[2 * turn + i], out))


def test_rows_of_a_stack_beyond_32_bits(L):
    """Expert planes whose byte offset passes 2^32 (and 2^31): the last expert is computed like the first."""
    E, M, K, group = 600, 4096, 4096, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    g = gen(8)
    plane = torch.zeros(E, M, K // 2, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(E, M, K // group, dtype=torch.bfloat16, device="cuda")
    one, s, _ = matrix((), M, K, group, torch.bfloat16, False, g)
    for e in (0, 257, E - 1):
        plane[e], scales[e] = one, s
    x = torch.randn(40, K, generator=g, device="cuda").bfloat16()
    for per in (2, 40):
        counts = [0] * E
        for e in (0, 257, E - 1):
            counts[e] = per
        got = L.w4a16_grouped_forward(x[:per].repeat(3, 1), plane, scales, None, ragged(counts), None, group)
        assert torch.equal(got[:per], got[per:2 * per]) and torch.equal(got[:per], got[2 * per:])
        check_linear(got[:per], x[:per], one, s, None, K, group)


def test_more_groups_of_eight_rows_than_one_grid_holds():
    """Rows that TMA cannot take stay on the kernel that gives every eight rows a grid row of their own, of which a launch has
    65535: half a million rows go in several launches, dense and by expert."""
    import bgemm_b200 as B

    g = gen(12)
    M, K, N, group = 3, 9, 65535 * 8 + 4100, 32                            # rows 18 bytes apart
    plane, scales, zeros = matrix((2,), M, K, group, torch.float16, True, g)
    x = torch.randn(N, K, generator=g, device="cuda").half()
    got = B.w4a16_gemm(x, plane[0], scales[0], zeros[0], group)
    check_linear(got, x, plane[0], scales[0], zeros[0], K, group)
    cut = 65535 * 8 - 13
    got = B.w4a16_grouped_gemm(x, plane, scales, zeros, torch.tensor([0, cut, N], dtype=torch.int32, device="cuda"), None, group)
    check_linear(got[:cut], x[:cut], plane[0], scales[0], zeros[0], K, group)
    check_linear(got[cut:], x[cut:], plane[1], scales[1], zeros[1], K, group)


def test_one_expert_with_an_index_is_the_dense_product(L):
    """The workspace asked for a single matrix serves the grouped call too: its rows are put together first, and the result is
    that of the dense call on those rows."""
    import bgemm_b200 as B

    g = gen(13)
    M, K, n, group = 4096, 4096, 320, 128
    plane, scales, zeros = matrix((1,), M, K, group, torch.bfloat16, True, g)
    x = torch.randn(200, K, generator=g, device="cuda").bfloat16()
    rows = torch.randint(0, 200, (n,), generator=g, device="cuda", dtype=torch.int32)
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, ragged([n]), rows, group)
    if os.environ.get("BGEMM_W4_TENSOR") != "0":                            # (the other kernel wants no workspace, and adds in another order)
        assert B.lib.bgemm_w4a16_workspace_bytes(1, M, K, n) >= n * K * 2
        assert torch.equal(got, L.w4a16_linear_forward(x[rows.long()], plane[0], scales[0], zeros[0], group))
    check_linear(got, x[rows.long()], plane[0], scales[0], zeros[0], K, group)


def test_a_gradient_is_refused_wherever_it_is_asked(L):
    g = gen(14)
    plane, scales, zeros = matrix((2,), 16, 64, 64, torch.float16, True, g)
    x = torch.randn(4, 64, generator=g, device="cuda").half()
    learnt = scales.clone().requires_grad_(True)
    out = torch.zeros(4, 16, dtype=torch.float16, device="cuda", requires_grad=True)
    off = ragged([2, 2])
    for call in (lambda: L.w4a16_linear_forward(x, plane[0], learnt[0], zeros[0], 64), lambda: L.w4_dequantize(plane, learnt, zeros, 64, 64),
                 lambda: L.w4a16_grouped_forward(x, plane, learnt, zeros, off, None, 64),
                 lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, 64, out)):
        with pytest.raises(RuntimeError):
            call()
    with torch.no_grad():
        want = L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, 64)
        assert torch.equal(L.w4a16_grouped_forward(x, plane, learnt, zeros, off, None, 64, out), want)


@pytest.mark.parametrize("M", [256, 300, 257])
@pytest.mark.parametrize("pitch,start", [(320, 0), (320, 1), (320, 2), (320, 4), (324, 0), (322, 2), (321, 0), (321, 3)])
def test_results_at_any_alignment(L, M, pitch, start):
    """Many rows (tensor cores) into a buffer with that pitch from that element: the values of a plain call, and nothing else written."""
    g = gen(M + pitch + start)
    K, n, group, E = 1024, 700, 64, 3
    plane, scales, zeros = matrix((E,), M, K, group, torch.bfloat16, True, g)
    x = torch.randn(n, K, generator=g, device="cuda").bfloat16()
    off = ragged([100, 0, 500])
    want = L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, group)
    check_linear(want[:100], x[:100], plane[0], scales[0], zeros[0], K, group)
    check_linear(want[100:600], x[100:600], plane[2], scales[2], zeros[2], K, group)
    buf = torch.full((n * pitch + start,), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = buf[start:].view(n, pitch)
    L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, group, rows[:, :M])
    assert torch.equal(rows[:600, :M], want[:600])
    assert bool((rows[600:] == 7).all()) and bool((rows[:, M:] == 7).all()) and bool((buf[:start] == 7).all())
