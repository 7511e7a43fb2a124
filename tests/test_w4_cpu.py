"""CPU tests of the 4-bit weight and routing entry points: the storage format, and the refusals of the C ABI and of the
extension, which all come before anything is launched."""
import ctypes

import pytest
import torch

import w4_oracle as W
from test_abi_cpu import LIB


@pytest.fixture(scope="module")
def lib():
    import bgemm_b200

    assert LIB.exists()
    return bgemm_b200.lib


def test_format_helpers(lib):
    for K in (1, 31, 128, 129, 4096, 4100):
        assert lib.bgemm_w4_row_bytes(K) == W.row_bytes(K)
    assert lib.bgemm_w4_row_bytes(0) == 0
    seen = {W.position(k) for k in range(256)}
    assert len(seen) == 256 and max(b for b, _ in seen) == 127          # every nibble of two blocks exactly once
    codes = torch.randint(0, 16, (3, 200), generator=torch.Generator().manual_seed(1))
    assert torch.equal(W.unpack(W.pack(codes), 200).long(), codes)


def test_quantize_refusals(lib):
    fake = 0x1000
    q = lib.bgemm_w4_quantize
    ok = dict(src=fake, dt=0, M=4, K=64, ld=64, group=32, sym=0, sdt=0, plane=fake, scales=fake, zeros=fake, batch=1, stride=0)

    def call(**kw):
        a = {**ok, **kw}
        return q(None, a["src"], a["dt"], a["M"], a["K"], a["ld"], a["group"], a["sym"], a["sdt"], a["plane"], a["scales"], a["zeros"], a["batch"], a["stride"])

    before = lib.bgemm_launch_count()
    assert call(src=None) == -1 and call(plane=None) == -1 and call(scales=None) == -1 and call(zeros=None) == -1
    assert call(dt=3) == -4 and call(sdt=2) == -4 and call(group=16) == -4 and call(group=256) == -4
    assert call(M=0) == -2 and call(K=0) == -2 and call(ld=63) == -2 and call(batch=0) == -2 and call(batch=2, stride=-1) == -2
    assert call(plane=fake + 8) == -3 and call(src=fake + 1) == -3 and call(dt=2, src=fake + 2) == -3
    assert lib.bgemm_launch_count() == before


def test_gemm_refusals(lib):
    fake = 0x1000
    before = lib.bgemm_launch_count()

    def gemm(plane=fake, M=8, K=64, group=32, scales=fake, zeros=None, x=fake, x_ld=64, dt=0, N=2, out=fake, out_ld=8, ws=None):
        return lib.bgemm_w4a16_gemm(None, plane, M, K, group, scales, zeros, x, x_ld, dt, N, out, out_ld, ws, 0)

    assert gemm(plane=None) == -1 and gemm(scales=None) == -1 and gemm(x=None) == -1 and gemm(out=None) == -1
    assert gemm(dt=2) == -4 and gemm(dt=3) == -4 and gemm(group=48) == -4
    assert gemm(M=0) == -2 and gemm(N=0) == -2 and gemm(K=0) == -2 and gemm(x_ld=63) == -2 and gemm(out_ld=7) == -2 and gemm(M=(1 << 24) + 1) == -2
    assert gemm(plane=fake + 4) == -3 and gemm(x=fake + 1) == -3 and gemm(out=fake + 1) == -3 and gemm(ws=fake + 16) == -3

    def grouped(E=4, x_rows=2, slots=2, offsets=fake, rows=None, x_ld=64, ws=None):
        return lib.bgemm_w4a16_grouped_gemm(None, fake, E, 8, 64, 32, fake, None, fake, x_rows, x_ld, 0, offsets, rows, slots, fake, 8, ws, 0)

    assert grouped(offsets=None) == -1 and grouped(E=0) == -2 and grouped(E=1025) == -2 and grouped(slots=0) == -2 and grouped(x_rows=0) == -2
    assert grouped(x_rows=1) == -2                                        # without an index every slot needs its row
    assert grouped(offsets=fake + 2) == -3 and grouped(rows=fake + 2) == -3 and grouped(x_ld=1) == -2 and grouped(ws=fake + 128) == -3
    assert lib.bgemm_w4_dequantize(None, None, 8, 64, 32, fake, None, 0, fake) == -1
    assert lib.bgemm_w4_dequantize(None, fake, 8, 64, 33, fake, None, 0, fake) == -4
    assert lib.bgemm_w4_dequantize(None, fake, 8, 64, 32, fake, None, 2, fake) == -4
    assert lib.bgemm_w4_dequantize(None, fake, 0, 64, 32, fake, None, 0, fake) == -2
    assert lib.bgemm_launch_count() == before


def test_routing_refusals(lib):
    fake = 0x1000
    before = lib.bgemm_launch_count()

    def route(logits=fake, dt=2, T=4, E=8, ld=8, k=2, weights=fake, ws=None, nbytes=0):
        return lib.bgemm_moe_route(None, logits, dt, T, E, ld, k, 1, weights, fake, fake, fake, fake, ws, nbytes)

    assert route(logits=None) == -1 and route(weights=None) == -1 and route(dt=3) == -4
    assert route(T=0) == -2 and route(E=0) == -2 and route(E=1025, ld=1025) == -2 and route(ld=7) == -2
    assert route(k=0) == -2 and route(k=9) == -2 and route(E=64, ld=64, k=33) == -2
    assert route(logits=fake + 2) == -3 and route(dt=0, logits=fake + 1) == -3
    assert lib.bgemm_moe_route_workspace_bytes(128, 64) == 0 and lib.bgemm_moe_route_workspace_bytes(129, 64) > 0
    assert route(T=1000) == -5 and route(T=1000, ws=fake, nbytes=16) == -5

    def combine(y=fake, dt=0, S=8, M=16, ld=16, T=4, k=2, out_ld=16):
        return lib.bgemm_moe_combine(None, y, dt, S, M, ld, fake, fake, T, k, fake, out_ld)

    assert combine(y=None) == -1 and combine(dt=2) == -4 and combine(S=0) == -2 and combine(M=0) == -2 and combine(ld=15) == -2
    assert combine(T=0) == -2 and combine(k=0) == -2 and combine(k=33) == -2 and combine(out_ld=8) == -2 and combine(y=fake + 1) == -3
    assert lib.bgemm_launch_count() == before


def test_extension_refuses_host_tensors():
    import lowbit_kernel

    x, plane, scales = torch.zeros(1, 64).half(), torch.zeros(8, 64, dtype=torch.uint8), torch.zeros(8, 1).half()
    for call in (lambda: lowbit_kernel.w4_quantize(torch.zeros(4, 64)), lambda: lowbit_kernel.w4a16_linear_forward(x, plane, scales),
                 lambda: lowbit_kernel.w4_dequantize(plane, scales, None, 64), lambda: lowbit_kernel.moe_route(torch.zeros(4, 8), 2),
                 lambda: lowbit_kernel.moe_combine(x, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1))):
        with pytest.raises(RuntimeError):
            call()
