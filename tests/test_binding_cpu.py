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
