"""The wait-expiry path of the tensor-core kernel of the 4-bit products, in the form of test_gpu_wait_expiry.py: with a budget of 0.1 ms
of SM clock and one block of codes withheld (bgemm_debug_set_wait_test) the unpack warps' wait runs out; the launch has to return, the status word to
name one of the kernel's barriers (51-59), and the next normal launch to be exact. Nothing faults or hangs."""
import pytest
import torch

import w4_oracle as W

pytestmark = pytest.mark.gpu


@pytest.fixture()
def B():
    import bgemm_b200

    bgemm_b200.lib.bgemm_debug_set_w4_kernel(1)
    yield bgemm_b200
    bgemm_b200.lib.bgemm_debug_set_wait_test(0, -1)          # never leave the hooks armed
    bgemm_b200.lib.bgemm_debug_set_w4_kernel(-1)


@pytest.mark.parametrize("M,K,counts,gather", [(256, 4096, [64], False),              # few pairs, tiles in one accumulator half, K divided
                                               (10240, 4096, [300, 256], False),      # every pair, tiles of both halves
                                               (512, 2048, [20] * 40, True),          # rows by index
                                               (300, 24576, [300], True)])            # rows put together first
def test_withheld_codes_make_the_wait_run_out_and_the_kernel_return(B, M, K, counts, gather):
    g = torch.Generator(device="cuda").manual_seed(M)
    E, n, group = len(counts), sum(counts), 128
    plane = W.pack(torch.randint(0, 16, (E, M, K), generator=g, device="cuda"))
    scales = torch.ones(E, M, K // group, dtype=torch.bfloat16, device="cuda")
    x = torch.randint(-3, 4, (n, K), generator=g, device="cuda").bfloat16()
    rows = torch.randint(0, n, (n,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    off = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device="cuda")
    src = x[rows.long()] if gather else x
    want = torch.cat([W.linear(src[int(off[e]):int(off[e + 1])], W.values(plane[e], scales[e], None, K, group)) for e in range(E)]).bfloat16()
    run = lambda: B.w4a16_grouped_gemm(x, plane, scales, None, off, rows, group)      # noqa: E731
    assert torch.equal(run(), want) and B.lib.bgemm_device_status(1) == 0
    B.lib.bgemm_debug_set_wait_test(200_000, 1)              # 0.1 ms budget; the second block of every tile never arrives
    run()
    torch.cuda.synchronize()                                 # the launch ends by itself
    status = B.lib.bgemm_device_status(1)
    assert status in range(51, 60), status
    assert B.lib.bgemm_device_status(0) == 0                 # reading with reset cleared the word
    B.lib.bgemm_debug_set_wait_test(0, -1)
    for _ in range(2):                                       # the context is intact: normal launches are exact again
        assert torch.equal(run(), want)
    assert B.lib.bgemm_device_status(1) == 0
