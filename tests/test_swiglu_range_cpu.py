"""SwiGLU's CPU form where silu alone leaves fp32's range (see the GPU tests of
the same name): one rounding of the 64-bit product."""

import torch


def test_far_gates():
    import rotalabs_accel_b200 as ra
    gate = torch.tensor([[-88.0, 0.5], [-96.0, 1.0], [-100.0, -120.0]]).bfloat16()
    up = torch.tensor([[1e38, 1.0], [-3e38, 0.25], [2e38, 3e38]]).bfloat16()
    q, s = ra.swiglu_int8(gate, up)
    v = gate.double() * torch.sigmoid(gate.double()) * up.double()
    top = v.abs().amax(-1)
    assert bool(((s.double() - top / 127).abs() <= top / 127 * 2.0 ** -23).all())
    assert bool(((q - v / (top / 127)[:, None]).abs() <= 0.5 + 2.0 ** -14).all())


def test_experts_on_far_gates():
    import rotalabs_accel_b200 as ra
    one = torch.ones(1, 1)
    y = ra.int8_moe(torch.ones(1, 1), torch.zeros(1, 1), torch.full((1, 1, 1), -95, dtype=torch.int8), one,
                    torch.full((1, 1, 1), 100, dtype=torch.int8), one * 1e36, torch.ones(1, 1, 1, dtype=torch.int8), one, top_k=1)
    g = torch.tensor(-95.0, dtype=torch.float64)
    want = (g * torch.sigmoid(g) * 1e38).item()
    assert abs(y.item() - want) <= abs(want) * 2.0 ** -21
