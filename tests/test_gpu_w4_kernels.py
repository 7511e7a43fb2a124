"""GPU tests of the two kernels behind the 4-bit products, each forced in turn (bgemm_debug_set_w4_kernel; the library's own rule
sends everything small to the streaming kernel). Every test also checks, by the library's counts, which kernel ran.
Real values: w4_oracle.linear_bound of the kernel under test, the tensor-core kernel against weights rounded as it rounds them. Whole
numbers: scales that are powers of two and activations of -3..3 make every product and sum exact in 32 bits, so a result
is the rounded exact one bit for bit and a single missing or misread column shows."""
import pytest
import torch

import w4_oracle as W

pytestmark = pytest.mark.gpu
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def L():
    import lowbit_kernel

    return lowbit_kernel


@pytest.fixture(params=["stream", "tensor"])
def kernel(request):
    yield from forced(request.param == "tensor")


@pytest.fixture()
def tensor():
    yield from forced(True)


def forced(on_tensor):
    """Every product of the test runs on that kernel, and at least one did."""
    import bgemm_b200 as B

    before = [B.lib.bgemm_debug_w4_calls(i) for i in (0, 1)]
    B.lib.bgemm_debug_set_w4_kernel(1 if on_tensor else 0)
    yield on_tensor
    B.lib.bgemm_debug_set_w4_kernel(-1)
    ran = [B.lib.bgemm_debug_w4_calls(i) - before[i] for i in (0, 1)]
    assert ran[on_tensor] > 0 and ran[not on_tensor] == 0, ran
    torch.cuda.synchronize()
    assert B.lib.bgemm_device_status(1) == 0                      # no wait ran out


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ragged(counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")


def matrix(lead, M, K, group, dtype, with_zeros, g, fill=0, whole=False):
    shape = tuple(lead) + (M, K)
    plane = W.pack(torch.randint(0, 16, shape, generator=g, device="cuda"), fill)
    sshape = tuple(lead) + (M, -(-K // group))
    if whole:
        scales = (2.0 ** torch.randint(-2, 2, sshape, generator=g, device="cuda")).to(dtype)
    else:
        scales = (torch.randn(sshape, generator=g, device="cuda") * 0.5 - 4.5).exp().to(dtype)
    zeros = torch.randint(0, 16, sshape, generator=g, device="cuda", dtype=torch.uint8) if with_zeros else None
    return plane, scales, zeros


def rows(N, K, dtype, g, whole=False, off=0):
    """Activations whose rows start on 16-byte boundaries (off elements behind one)."""
    wide = torch.empty(N, (K + 7) // 8 * 8 + 16, dtype=dtype, device="cuda").fill_(float("nan"))
    x = wide[:, 8 + off:8 + off + K]
    x.copy_(torch.randint(-3, 4, (N, K), generator=g, device="cuda") if whole else torch.randn(N, K, generator=g, device="cuda"))
    return x


def check(got, x, plane, scales, zeros, K, group, on_tensor):
    want = W.linear(x, (W.rounded if on_tensor else W.values)(plane, scales, zeros, K, group))
    off, tol = (got.double() - want).abs(), W.linear_bound(x, want, plane, scales, zeros, K, group, on_tensor)
    assert got.dtype == x.dtype and bool((off <= tol).all()), f"largest error {float((off / tol).max()):.3g} of the bound"


# ---- dense -----------------------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1, 32), (16, 128, 1, 128), (17, 129, 2, 32), (100, 1000, 7, 64), (128, 256, 8, 128), (33, 2056, 9, 32), (512, 4096, 1, 128), (300, 1111, 16, 64),
          (129, 640, 17, 128), (256, 1024, 33, 32), (130, 520, 64, 64), (1000, 2048, 100, 128), (257, 4104, 255, 64), (384, 1536, 300, 128), (128, 128, 513, 32),
          (5000, 264, 40, 128), (2, 31, 257, 64)]


@pytest.mark.parametrize("whole", [True, False], ids=["whole", "real"])
@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,group", SHAPES)
def test_linear(L, kernel, M, K, N, group, dtype, with_zeros, whole):
    g = gen(M * 7 + K + N)
    plane, scales, zeros = matrix((), M, K, group, DT[dtype], with_zeros, g, 15, whole)
    x = rows(N, K, DT[dtype], g, whole)
    got = L.w4a16_linear_forward(x, plane, scales, zeros, group)
    if whole:
        assert torch.equal(got, W.linear(x, W.values(plane, scales, zeros, K, group)).to(DT[dtype]))
    else:
        check(got, x, plane, scales, zeros, K, group, kernel)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N", [(40, 8193, 3), (150, 8320, 70), (2400, 14336, 2), (640, 14336, 160), (5000, 28680, 1), (6000, 8200, 1), (12000, 8200, 2), (17000, 8200, 1), (300, 28680, 300)])
def test_long_rows_are_exact(L, kernel, M, K, N, dtype, group):
    """More than 64 blocks of 128 columns, where the streaming kernel comes round to a second set of scales, on 12, 8 and 4 warps and
    every tile height. |sums| stay below 2^24 quarter units: 28680 x 3 x 15 x 2 < 2^22."""
    g = gen(M + K)
    plane, scales, zeros = matrix((), M, K, group, DT[dtype], True, g, 5, True)
    x = rows(N, K, DT[dtype], g, True)
    assert torch.equal(L.w4a16_linear_forward(x, plane, scales, zeros, group), W.linear(x, W.values(plane, scales, zeros, K, group)).to(DT[dtype]))


@pytest.mark.parametrize("N", [1, 3, 40, 140])
def test_linear_strides(L, kernel, N):
    """x as a slice of a wider matrix whose rows start on 16-byte boundaries, transposed, and one row for all."""
    g = gen(N)
    M, K, group = 160, 392, 32
    plane, scales, zeros = matrix((), M, K, group, torch.bfloat16, True, g)
    aligned = torch.randn(N, 800, generator=g, device="cuda").bfloat16()
    tall = torch.randn(K, N, generator=g, device="cuda").bfloat16()
    for x in (aligned[:, 8:8 + K], tall.t(), aligned[:1, :K].expand(N, K)):
        got = L.w4a16_linear_forward(x, plane, scales, zeros, group)
        assert got.is_contiguous()
        check(got, x, plane, scales, zeros, K, group, kernel)


@pytest.mark.parametrize("N", [1, 4, 20, 150, 300])
def test_rows_do_not_touch_each_other(L, kernel, N):
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


@pytest.mark.parametrize("group", [32, 64, 128])
def test_zero_point_uses_its_low_four_bits(L, kernel, group):
    g = gen(9)
    plane, scales, zeros = matrix((), 64, 256, group, torch.bfloat16, True, g)
    x = torch.randn(60, 256, generator=g, device="cuda").bfloat16()
    assert torch.equal(L.w4a16_linear_forward(x, plane, scales, zeros, group), L.w4a16_linear_forward(x, plane, scales, zeros | 0xF0, group))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("K", [1, 31, 127, 130, 200, 257, 1000, 4095])
def test_codes_behind_k_are_ignored(L, kernel, K, dtype, group):
    """Whatever they hold, also where (q - z) s of such a code is beyond the type's numbers: fp16 scales of 6000, codes 0..2, padding 15."""
    g = gen(K)
    M, N = 130, 70
    codes = torch.randint(0, 3, (M, K), generator=g, device="cuda")
    scales = torch.full((M, -(-K // group)), 6000.0 if dtype == "fp16" else 2.0 ** 126, dtype=DT[dtype], device="cuda")
    zeros = torch.zeros(scales.shape, dtype=torch.uint8, device="cuda")
    x = rows(N, K, DT[dtype], g, True).zero_()
    x[torch.arange(N, device="cuda"), torch.randint(0, K, (N,), generator=g, device="cuda")] = 0.5 if dtype == "fp16" else 2.0 ** -30
    want = W.linear(x, W.values(W.pack(codes), scales, zeros, K, group)).to(DT[dtype])
    assert bool(torch.isfinite(want).all())
    assert torch.equal(L.w4a16_linear_forward(x, W.pack(codes, 15), scales, zeros, group), want)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,N,group", [(300, 2048, 40, 64), (256, 4096, 200, 32), (1001, 4100, 17, 128), (1300, 4096, 300, 128)])
def test_divided_k(L, tensor, M, K, N, group, dtype):
    """Few tiles: K is divided and a second kernel adds the parts up. With less workspace than asked for, or none, K stays whole."""
    import bgemm_b200 as B

    g = gen(M + N)
    plane, scales, zeros = matrix((), M, K, group, DT[dtype], True, g, 7)
    x = rows(N, K, DT[dtype], g)
    need = B.lib.bgemm_w4a16_workspace_bytes(1, M, K, N)
    assert need >= 2 * N * M * 4
    before = B.launch_count()
    check(L.w4a16_linear_forward(x, plane, scales, zeros, group), x, plane, scales, zeros, K, group, True)
    assert B.launch_count() - before == 2
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    for give in (0, N * M * 4):
        out = torch.zeros(N, M, dtype=DT[dtype], device="cuda")
        before = B.launch_count()
        assert B.lib.bgemm_w4a16_gemm(torch.cuda.current_stream().cuda_stream, plane.data_ptr(), M, K, group, scales.data_ptr(), zeros.data_ptr(), x.data_ptr(), x.stride(0),
                                      B.dtype_code(x), N, out.data_ptr(), M, ws.data_ptr() if give else None, give) == 0
        assert B.launch_count() - before == 1
        check(out, x, plane, scales, zeros, K, group, True)


# ---- grouped by expert -----------------------------------------------------------------------------------------------
COUNTS = [[1], [0, 3, 0], [8, 0, 1, 2], [0] * 40 + [5] + [0] * 30, [1] * 70, [40, 1, 0, 17, 16, 9], [300, 0, 5, 129], [64, 64, 65, 63], [700, 2], [0, 0, 0, 515],
          [33, 97, 161, 225, 31, 95, 159, 223], [1] * 200 + [90]]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype,group", [("fp16", 32), ("fp16", 64), ("fp16", 128), ("bf16", 32), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("counts", COUNTS, ids=[str(i) for i in range(len(COUNTS))])
def test_grouped(L, kernel, counts, dtype, group, gather):
    """Whole numbers: ragged, empty and single-row experts, by index (tile::gather4 or rows put together first) and in order; several
    divide K. A width off 8 takes the unaligned stores."""
    g = gen(len(counts) + sum(counts))
    E, M, K = len(counts), 150, 328
    plane, scales, zeros = matrix((E,), M, K, group, DT[dtype], True, g, 3, True)
    offsets, slots = ragged(counts), sum(counts)
    T = 11 if gather else slots
    x = rows(T, K, DT[dtype], g, True)
    index = torch.randint(0, T, (slots,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, offsets, index, group)
    src = x[index.long()] if gather else x
    at = offsets.tolist()
    for e in range(E):
        sl = slice(at[e], at[e + 1])
        assert torch.equal(got[sl], W.linear(src[sl], W.values(plane[e], scales[e], zeros[e], K, group)).to(DT[dtype])), e


@pytest.mark.parametrize("M,K", [(1000, 2056), (1001, 1024)])
@pytest.mark.parametrize("per", [5, 20, 50])
def test_grouped_rows_by_index(L, kernel, per, M, K):
    """Real values on 16 experts of uneven counts: on the tensor cores up to 24 slots an expert on average are read by tile::gather4, more
    are put together first; one launch more."""
    import bgemm_b200 as B

    g = gen(per + M)
    E, group = 16, 64
    counts = [per * 2 if e % 4 == 0 else (0 if e % 4 == 1 else per) for e in range(E)]
    plane, scales, zeros = matrix((E,), M, K, group, torch.bfloat16, True, g, 1)
    x = rows(30, K, torch.bfloat16, g)
    index = torch.randint(0, 30, (sum(counts),), generator=g, device="cuda", dtype=torch.int32)
    before = B.launch_count()
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, ragged(counts), index, group)
    if kernel:
        assert B.launch_count() - before == (2 if per > 24 else 1)
    at = 0
    for e, c in enumerate(counts):
        if c:
            check(got[at:at + c], x[index[at:at + c].long()], plane[e], scales[e], zeros[e], K, group, kernel)
        at += c


@pytest.mark.parametrize("K", [256, 6000])
@pytest.mark.parametrize("slots", [7, 30, 400])
def test_grouped_leaves_other_rows_alone(L, kernel, slots, K):
    """With the longer rows the tensor cores divide K, and the kernel that adds the parts up keeps to the experts' rows too."""
    g = gen(slots)
    E, M, group = 3, 70, 128
    plane, scales, zeros = matrix((E,), M, K, group, torch.float16, True, g, 0, True)
    n = slots - 3
    offsets = torch.tensor([0, n // 3, n // 3, n], dtype=torch.int32, device="cuda")
    x = torch.randint(-3, 4, (5, K), generator=g, device="cuda").half()
    index = torch.randint(0, 5, (slots,), generator=g, device="cuda", dtype=torch.int32)
    index[0], index[n - 1], index[1] = -1, 5, index[2]
    buf = torch.full((slots, M + 9), 77.0, dtype=torch.float16, device="cuda")
    L.w4a16_grouped_forward(x, plane, scales, zeros, offsets, index, group, buf[:, 4:4 + M])
    assert bool((buf[n:] == 77).all()) and bool((buf[:, :4] == 77).all()) and bool((buf[:, 4 + M:] == 77).all())
    src = torch.where(((index >= 0) & (index < 5))[:, None], x[index.clamp(0, 4).long()], 0)
    for e, (a, b) in enumerate(((0, n // 3), (n // 3, n // 3), (n // 3, n))):
        assert torch.equal(buf[a:b, 4:4 + M], W.linear(src[a:b], W.values(plane[e], scales[e], zeros[e], K, group)).half())


@pytest.mark.parametrize("K", [128, 2048])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("slots", [6, 200])
def test_offsets_that_make_no_sense_stay_in_bounds(L, kernel, slots, gather, K):
    g = gen(1)
    E, M = 4, 64
    plane, scales, zeros = matrix((E,), M, K, 128, torch.bfloat16, False, g)
    x = torch.randn(slots, K, generator=g, device="cuda").bfloat16()
    index = torch.randint(-5, slots + 5, (slots,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    buf = torch.full((slots + 16, M), 5.0, dtype=torch.bfloat16, device="cuda")
    for bad in ([0, 1 << 30, 3, -7, 9], [-5, -4, -3, -2, -1], [slots + 1] * 5, [0, 2, 1, slots + 90, slots + 100], [2 ** 31 - 1, -2 ** 31, 0, 2 ** 31 - 1, 1]):
        L.w4a16_grouped_forward(x, plane, scales, zeros, torch.tensor(bad, dtype=torch.int32, device="cuda"), index, 128, buf[8:8 + slots])
        torch.cuda.synchronize()
        assert bool((buf[:8] == 5).all()) and bool((buf[8 + slots:] == 5).all())


def test_two_streams_and_graphs(L, kernel):
    g = gen(6)
    E, M, K, group = 6, 512, 1024, 128
    plane, scales, zeros = matrix((E,), M, K, group, torch.bfloat16, True, g)
    xs = [torch.randn(196, K, generator=g, device="cuda").bfloat16() for _ in range(4)]
    off, index = ragged([30, 0, 101, 40, 20, 5]), torch.randint(0, 196, (196,), generator=g, device="cuda", dtype=torch.int32)
    calls = lambda x: (L.w4a16_linear_forward(x, plane[0], scales[0], zeros[0], group), L.w4a16_linear_forward(x[:3], plane[0], scales[0], zeros[0], group),      # noqa: E731
                       L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, group), L.w4a16_grouped_forward(x, plane, scales, zeros, off, index, group))
    want = [calls(x) for x in xs]
    torch.cuda.synchronize()
    got = []
    for x, st in zip(xs, [torch.cuda.Stream() for _ in range(4)]):
        with torch.cuda.stream(st):
            got.append(calls(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for w, o in zip(want, got) for a, b in zip(w, o))
    static, graphs = [x.clone() for x in xs[:2]], []
    for x in static:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = calls(x)
        graphs.append((graph, out))
    for turn in range(2):
        for i, (graph, out) in enumerate(graphs):
            static[i].copy_(xs[2 * turn + i])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want[2 * turn + i], out))


def test_rows_of_a_stack_beyond_32_bits(L, kernel):
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
        check(got[:per], x[:per], one, s, None, K, group, kernel)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M", [256, 257])
@pytest.mark.parametrize("pitch,start", [(320, 0), (320, 1), (320, 2), (320, 4), (324, 0), (322, 2), (321, 0), (321, 3)])
def test_results_at_any_alignment(L, kernel, M, pitch, start, dtype, group, gather):
    g = gen(M + pitch + start)
    K, n, E = 512, 420, 20 if gather else 3                        # 21 slots an expert: by tile::gather4
    plane, scales, zeros = matrix((E,), M, K, group, DT[dtype], True, g, 2, True)
    x = rows(n, K, DT[dtype], g, True)
    index = torch.randperm(n, generator=g, device="cuda").int() if gather else None
    src = x[index.long()] if gather else x
    buf = torch.full((n * pitch + start,), 7.0, dtype=DT[dtype], device="cuda")
    out = buf[start:].view(n, pitch)
    L.w4a16_grouped_forward(x, plane, scales, zeros, ragged([60] + [0] * (E - 2) + [300]), index, group, out[:, :M])
    for e, sl in ((0, slice(0, 60)), (E - 1, slice(60, 360))):
        assert torch.equal(out[sl, :M], W.linear(src[sl], W.values(plane[e], scales[e], zeros[e], K, group)).to(DT[dtype]))
    assert bool((out[360:] == 7).all()) and bool((out[:, M:] == 7).all()) and bool((buf[:start] == 7).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_both_bindings_and_the_layers(L, kernel, dtype):
    """The extension, the ctypes binding and W4Experts call the same thing: equal bits; a captured layer serves other tokens."""
    import bgemm_b200 as B
    import bgemm_linear as N

    g = gen(21)
    E, H, I, T = 8, 264, 136, 150
    layer = N.W4Experts(torch.randn(E, 2 * I, H, generator=g, device="cuda").to(DT[dtype]) * 0.06, torch.randn(E, H, I, generator=g, device="cuda").to(DT[dtype]) * 0.06, 2,
                        group_size=64)
    xs = torch.randn(2, T, H, generator=g, device="cuda").to(DT[dtype])
    ls = torch.randn(2, T, E, generator=g, device="cuda")
    ls[1, 40:] = -float("inf")
    want = []
    for x, lg in zip(xs, ls):
        weights, _, off, index, slots = L.moe_route(lg, 2, True)
        h = B.w4a16_grouped_gemm(x, layer.gate_up_plane, layer.gate_up_scales, layer.gate_up_zeros, off, index, 64)
        assert torch.equal(h[:int(off[-1])], L.w4a16_grouped_forward(x, layer.gate_up_plane, layer.gate_up_scales, layer.gate_up_zeros, off, index, 64)[:int(off[-1])])
        at = off.tolist()
        for e in range(E):
            if at[e + 1] > at[e]:
                sl = slice(at[e], at[e + 1])
                check(h[sl], x[index[sl].long()], layer.gate_up_plane[e], layer.gate_up_scales[e], layer.gate_up_zeros[e], H, 64, kernel)
        want.append(layer(x, lg))
        assert bool(torch.isfinite(want[-1]).all())
    assert bool((want[1][40:] == 0).all())
    sx, sl = xs[0].clone(), ls[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(sx, sl)
    for i in (1, 0, 1):
        sx.copy_(xs[i])
        sl.copy_(ls[i])
        graph.replay()
        assert torch.equal(out, want[i])


# ---- which kernel a call takes -----------------------------------------------------------------------------------------
def calls():
    import bgemm_b200 as B

    return [B.lib.bgemm_debug_w4_calls(i) for i in (0, 1)]


def telling(E, M, K, group, n, dtype):
    """Two weights of a row, 15 s with a scale of many bits and 15, and activations 1 and -1 for them: 15 s - 15 where no weight is rounded
    (a number of 4 bits); 15 s rounded to the type is another."""
    s = 1 + (2.0 ** -10 if dtype == torch.float16 else 2.0 ** -7)
    plane = torch.full((E, M, W.row_bytes(K)), 255, dtype=torch.uint8, device="cuda")
    scales = torch.ones(E, M, -(-K // group), dtype=dtype, device="cuda")
    scales[..., 0] = s
    x = torch.zeros(n, K, dtype=dtype, device="cuda")
    x[:, 0], x[:, group] = 1, -1
    exact, off = 15 * s - 15, float(torch.tensor(15 * s).to(dtype)) - 15
    assert exact != off
    return plane, scales, torch.zeros(scales.shape, dtype=torch.uint8, device="cuda"), x, exact, off


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("E,M,K,per", [(1, 28672, 8192, 7), (1, 28672, 8192, 8), (64, 2048, 4096, 7), (64, 2048, 4096, 8)])
def test_up_to_eight_slots_an_expert_meet_unrounded_weights(L, E, M, K, per, dtype):
    n = E * per
    plane, scales, zeros, x, exact, _ = telling(E, M, K, 128, n, DT[dtype])
    before = calls()
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, ragged([per] * E), None, 128)
    assert bool((got == exact).all())
    assert bool((L.w4a16_linear_forward(x[:per], plane[0], scales[0], zeros[0], 128) == exact).all())
    assert [b - a for a, b in zip(before, calls())] == [2, 0]


@pytest.mark.parametrize("n", [8, 9, 16, 17, 40])
@pytest.mark.parametrize("M,K", [(28672, 8192), (8192, 8192), (1024, 4096)])
def test_one_expert_takes_the_kernel_of_the_dense_product(L, M, K, n):
    plane, scales, zeros, x, exact, off = telling(1, M, K, 64, n, torch.bfloat16)
    before = calls()
    dense = L.w4a16_linear_forward(x, plane[0], scales[0], zeros[0], 64)
    middle = calls()
    assert torch.equal(L.w4a16_grouped_forward(x, plane, scales, zeros, ragged([n]), None, 64), dense)
    assert [b - a for a, b in zip(before, middle)] == [b - a for a, b in zip(middle, calls())]
    assert bool((dense == (exact if middle[0] > before[0] else off)).all())


def test_a_tangent_is_refused(L):
    """Forward-mode: the results carry no tangent, which autograd would take for zero."""
    import bgemm_linear as N
    from torch.autograd import forward_ad as F

    g = gen(31)
    plane, scales, zeros = matrix((2,), 64, 64, 64, torch.float16, True, g)
    x = torch.randn(4, 64, generator=g, device="cuda").half()
    off, logits = ragged([2, 2]), torch.randn(4, 2, generator=g, device="cuda")
    weights, _, _, _, slots = L.moe_route(logits, 1)
    out = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    linear, experts = N.W4Linear(x.repeat(16, 1)), N.W4Experts(torch.randn(2, 64, 64, device="cuda").half(), torch.randn(2, 64, 32, device="cuda").half(), 1)
    with F.dual_level(), torch.no_grad():
        dual = lambda t: F.make_dual(t, torch.ones_like(t))      # noqa: E731
        for call in (lambda: L.w4_quantize(dual(x), 64), lambda: L.w4_dequantize(plane, dual(scales), zeros, 64, 64),
                     lambda: L.w4a16_linear_forward(dual(x), plane[0], scales[0], zeros[0], 64), lambda: L.w4a16_linear_forward(x, plane[0], dual(scales[0]), zeros[0], 64),
                     lambda: L.w4a16_grouped_forward(dual(x), plane, scales, zeros, off, None, 64), lambda: L.w4a16_grouped_forward(x, plane, scales, zeros, off, None, 64, dual(out)),
                     lambda: L.moe_route(dual(logits), 1), lambda: L.moe_combine(dual(x), slots, weights), lambda: L.moe_combine(x, slots, dual(weights)),
                     lambda: linear(dual(x)), lambda: experts(dual(x), logits), lambda: experts(x, dual(logits))):
            with pytest.raises(RuntimeError):
                call()
        assert linear(x).shape == experts(x, logits).shape == (4, 64)      # inputs without one are served


def test_the_ctypes_binding_refuses_gradients_too(L):
    import bgemm_b200 as B
    from torch.autograd import forward_ad as F

    g = gen(32)
    plane, scales, zeros = matrix((2,), 64, 64, 64, torch.float16, True, g)
    x = torch.randn(4, 64, generator=g, device="cuda").half()
    off, logits = ragged([2, 2]), torch.randn(4, 2, generator=g, device="cuda")
    weights, _, _, _, slots = B.moe_route(logits, 1)
    out = torch.zeros(4, 64, dtype=torch.float16, device="cuda")
    calls = lambda v: [lambda: B.w4_quantize(v(x), 64), lambda: B.w4_dequantize(plane, v(scales), zeros, 64, 64),      # noqa: E731
                       lambda: B.w4a16_gemm(v(x), plane[0], scales[0], zeros[0], 64), lambda: B.w4a16_gemm(x, plane[0], v(scales[0]), zeros[0], 64),
                       lambda: B.w4a16_gemm(x, plane[0], scales[0], zeros[0], 64, v(out)), lambda: B.w4a16_grouped_gemm(v(x), plane, scales, zeros, off, None, 64),
                       lambda: B.w4a16_grouped_gemm(x, plane, scales, zeros, off, None, 64, v(out)), lambda: B.moe_route(v(logits), 1), lambda: B.moe_combine(v(x), slots, weights),
                       lambda: B.moe_combine(x, slots, v(weights))]
    learnt = lambda t: t.clone().requires_grad_(True)            # noqa: E731
    for call in calls(learnt):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        for call in calls(learnt):
            call()
        with F.dual_level():
            for call in calls(lambda t: F.make_dual(t, torch.ones_like(t))):
                with pytest.raises(ValueError):
                    call()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,n", [(28672, 8192, 17), (4096, 4096, 200), (1000, 1024, 2000)])
def test_exact_weights_at_any_number_of_rows(L, M, K, n, dtype):
    """Without the flag these sizes meet rounded weights; with it none is rounded, in both bindings, dense and by expert."""
    import bgemm_b200 as B

    plane, scales, zeros, x, exact, off = telling(1, M, K, 128, n, DT[dtype])
    index = torch.arange(n, device="cuda").int()
    assert bool((L.w4a16_linear_forward(x, plane[0], scales[0], zeros[0], 128) == off).all())
    before = calls()
    for got in (L.w4a16_linear_forward(x, plane[0], scales[0], zeros[0], 128, exact=True), B.w4a16_gemm(x, plane[0], scales[0], zeros[0], 128, exact=True),
                L.w4a16_grouped_forward(x, plane, scales, zeros, ragged([n]), None, 128, exact=True), B.w4a16_grouped_gemm(x, plane, scales, zeros, ragged([n]), index, 128, exact=True)):
        assert bool((got == exact).all())
    assert [b - a for a, b in zip(before, calls())] == [4, 0]


def test_exact_layers(L):
    """W4Linear and W4Experts with exact: real values within the bound that rounds no weight; the default takes the other kernel."""
    import bgemm_linear as N

    g = gen(41)
    w = torch.randn(2048, 2048, generator=g, device="cuda").half() * 0.05
    x = torch.randn(600, 2048, generator=g, device="cuda").half()
    before = calls()
    layer = N.W4Linear(w, exact=True)
    check(layer(x), x, layer.plane, layer.scales, layer.zeros, 2048, 128, False)
    assert [b - a for a, b in zip(before, calls())] == [1, 0]
    N.W4Linear(w)(x)
    assert [b - a for a, b in zip(before, calls())] == [1, 1]
    gate_up, down = torch.randn(4, 1024, 1024, generator=g, device="cuda").half() * 0.05, torch.randn(4, 1024, 512, generator=g, device="cuda").half() * 0.05
    logits = torch.randn(600, 4, generator=g, device="cuda")
    before = calls()
    N.W4Experts(gate_up, down, 2, exact=True)(x[:, :1024], logits)
    assert [b - a for a, b in zip(before, calls())] == [2, 0]
    N.W4Experts(gate_up, down, 2)(x[:, :1024], logits)
    assert [b - a for a, b in zip(before, calls())] == [2, 2]


@pytest.mark.parametrize("n", [1, 9, 40])
def test_a_few_rows_of_a_large_x_are_not_paid_for_by_all_of_it(L, n):
    """Rows off 16-byte boundaries, named by index: read where they lie, no copy of x."""
    g = gen(n)
    M, K, T = 4096, 4095, 20000
    plane, scales, zeros = matrix((4,), M, K, 128, torch.bfloat16, True, g)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    index = torch.randint(0, T, (n,), generator=g, device="cuda", dtype=torch.int32)
    off = ragged([n - n // 2, 0, n // 2, 0])
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    got = L.w4a16_grouped_forward(x, plane, scales, zeros, off, index, 128)
    assert torch.cuda.max_memory_allocated() - held < x.numel() // 4
    at = off.tolist()
    for e in range(4):
        if at[e + 1] > at[e]:
            sl = slice(at[e], at[e + 1])
            check(got[sl], x[index[sl].long()], plane[e], scales[e], zeros[e], K, 128, False)
