"""CPU tests of the ctypes binding's checks that need no GPU: stand-ins for tensors that say where they are."""
import types

import pytest
import torch


@pytest.fixture(scope="module")
def B():
    import bgemm_b200

    return bgemm_b200


def on(index, **more):
    return types.SimpleNamespace(is_cuda=True, device=torch.device("cuda", index), **more)


def test_tensors_of_two_devices_are_refused(B):
    B._require_cuda(on(0), None, on(0))
    B._require_cuda(None, on(1), on(1))
    for mixed in ((on(0), on(1)), (None, on(1), None, on(0)), (on(0), on(0), on(1))):
        with pytest.raises(ValueError, match="one device"):
            B._require_cuda(*mixed)
    with pytest.raises(ValueError, match="CUDA tensor"):
        B._require_cuda(on(0), torch.zeros(1))


def test_every_product_and_routing_call_checks_its_tensors_together(B):
    """One tensor on another device than the others, in every place."""
    here, there = on(0, shape=(2, 64)), on(1, shape=(2, 64))
    for call in (lambda: B.w4a16_gemm(there, here, here), lambda: B.w4a16_gemm(here, there, there), lambda: B.w4a16_gemm(here, here, there), lambda: B.w4a16_gemm(here, here, here, there),
                 lambda: B.w4a16_grouped_gemm(there, here, here, None, here), lambda: B.w4a16_grouped_gemm(here, here, here, None, there),
                 lambda: B.w4a16_grouped_gemm(here, here, here, None, here, there), lambda: B.w4a16_grouped_gemm(here, here, there, None, here),
                 lambda: B.w4_dequantize(here, there, None, 64), lambda: B.moe_combine(here, there, here), lambda: B.moe_combine(here, here, there)):
        with pytest.raises(ValueError, match="one device"):
            call()


def test_unknown_flags_are_refused_before_any_launch(B):
    fake = 0x1000
    before = B.launch_count()
    for flags in (1, 2, 4, 16, 8 | 1, -1):
        assert B.lib.bgemm_w4a16_gemm_ex(None, fake, 8, 64, 32, fake, None, fake, 64, 0, 2, fake, 8, None, 0, flags) == -4
        assert B.lib.bgemm_w4a16_grouped_gemm_ex(None, fake, 4, 8, 64, 32, fake, None, fake, 2, 64, 0, fake, None, 2, fake, 8, None, 0, flags) == -4
    assert B.lib.bgemm_w4a16_gemm_ex(None, None, 8, 64, 32, fake, None, fake, 64, 0, 2, fake, 8, None, 0, 8) == -1
    assert B.lib.bgemm_w4a16_grouped_gemm_ex(None, fake, 0, 8, 64, 32, fake, None, fake, 2, 64, 0, fake, None, 2, fake, 8, None, 0, 8) == -2
    assert B.launch_count() == before
