"""The 8-bit path and the experts' layer are for inference: no gradients flow,
on the CPU as on the GPU, also from inputs that ask for them."""

import pytest
import torch


def _outputs(device):
    import rotalabs_accel_b200 as ra
    g = torch.Generator().manual_seed(1)
    x, r = (torch.randn(3, 32, generator=g).half().to(device).requires_grad_() for _ in range(2))
    w = torch.nn.Parameter(torch.ones(32, device=device))
    q = torch.randint(-9, 9, (3, 32), generator=g, dtype=torch.int8).to(device)
    sx, sw = (torch.ones(n, device=device).requires_grad_() for n in (3, 3))
    bias = torch.zeros(3, device=device).half().requires_grad_()
    router = torch.randn(4, 32, generator=g).half().to(device).requires_grad_()
    we = torch.randint(-9, 9, (4, 32, 32), generator=g, dtype=torch.int8).to(device)
    se = (torch.ones(4, 32, device=device) * 1e-2).requires_grad_()
    return (*ra.add_rmsnorm(x, r, w), *ra.add_rmsnorm_int8(x, r, w), *ra.swiglu_int8(x, r),
            ra.int8_gemm_w8a8(q, sx, q, sw, bias), ra.int8_moe(x, router, we, se, we, se, we, se, top_k=2))


def test_cpu():
    assert not any(t.requires_grad for t in _outputs("cpu"))


@pytest.mark.gpu
def test_gpu(cuda_lib):
    assert not any(t.requires_grad for t in _outputs("cuda"))
