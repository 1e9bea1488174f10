"""SwiGLU where silu alone leaves fp32's range: gates below -87 times large ups,
rows of strongly negative gates only, against the formula in 64 bits.

Tolerance: silu's relative error is at most 2^-20, and for negative gates |gate| * 2^-23.5
more (the rounding of gate * log2(e), and of log2(e)); below -87 the exponential is the
square of a rounded one, the same bound.  q is off by half a step and that
error of itself and of the scale.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _check(gate, up):
    import rotalabs_accel_b200 as ra
    q, s = ra.swiglu_int8(gate, up)
    d, u = gate.double(), up.double()
    v = d * torch.sigmoid(d) * u
    rel = 2.0 ** -20 + (-d).clamp(min=0) * 2.0 ** -23.5
    top = v.abs().amax(-1)
    err = (v.abs() * rel).amax(-1)
    s64 = torch.where(top > 127 * 2.0 ** -149, top / 127, torch.ones_like(top))
    # (a subnormal scale is a multiple of 2^-149)
    assert bool(((s.double() - s64).abs() <= err / 127 * (1 + 2.0 ** -10) + s64 * 2.0 ** -22 + 2.0 ** -150).all())
    normal = s64 > 2.0 ** -126
    off = (q.double() - v / s64.unsqueeze(-1)).abs()
    assert bool((off <= 0.5 + 127 * (rel + (err / top).unsqueeze(-1)) + 127 * 2.0 ** -20)[normal].all())
    return q, s


# widths of the vector, 4-wide and single-element forms, few rows and the many
# that run through the ring
@pytest.mark.parametrize("M,N", [(3, 64), (5, 4100), (4, 255), (700, 2048), (601, 4104), (600, 4100)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_strongly_negative_gates(cuda_lib, M, N, dtype):
    g = torch.Generator(device="cuda").manual_seed(M + N)
    u01 = lambda: torch.rand(M, N, generator=g, device="cuda")  # noqa: E731
    sign = torch.where(u01() < 0.5, -1.0, 1.0)
    most = 60000.0 if dtype == torch.float16 else 3e38
    for low, high in ((-87, -16), (-104, -60), (-170, -86)):
        gate = (low + (high - low) * u01()).to(dtype)
        _check(gate, (sign * most * (0.1 + 0.9 * u01())).to(dtype))
    # one far gate beside ordinary ones, its product the row's largest
    gate = torch.randn(M, N, generator=g, device="cuda").clamp(-8, 8).to(dtype)
    up = torch.randn(M, N, generator=g, device="cuda").to(dtype)
    if dtype == torch.bfloat16:
        gate[:, N // 3], up[:, N // 3] = -88.0, 1e38
        q, s = _check(gate, up)
        assert bool((q[:, N // 3] == -127).all())
        assert bool(((s.double() * 127 / 53 - 1).abs() < 0.01).all())
    _check(gate, up)


def test_limits(cuda_lib):
    import rotalabs_accel_b200 as ra
    inf = float("inf")
    for dtype in (torch.float16, torch.bfloat16):
        gate = torch.tensor([[-inf, 1.0], [-torch.finfo(dtype).max, 1.0], [inf, 1.0], [-200.0, 1.0]], device="cuda").to(dtype)
        up = torch.ones_like(gate)
        q, s = ra.swiglu_int8(gate, up)
        assert torch.isnan(s[0]) and torch.isnan(s[2]) and not q[0].any() and not q[2].any()
        assert q[1].tolist() == [0, 127] and q[3].tolist() == [0, 127]


def test_far_gates_in_the_experts(cuda_lib):
    """silu(-95) is 5e-40, its product with 1e38 is not."""
    import rotalabs_accel_b200 as ra
    H, I = 64, 16
    for T in (1, 7, 30):
        x = torch.zeros(T, H, device="cuda").half()
        x[:, 0] = 1.0
        wg = torch.zeros(1, I, H, dtype=torch.int8, device="cuda")
        wu, wd = torch.zeros_like(wg), torch.zeros(1, H, I, dtype=torch.int8, device="cuda")
        wg[0, :, 0], wu[0, :, 0] = -torch.arange(80, 96, device="cuda").to(torch.int8), 100
        wd[0, :I] = 100 * torch.eye(I, device="cuda").to(torch.int8)
        su = torch.full((1, I), 1e36, device="cuda")
        one = torch.ones(1, I, device="cuda")
        sd = torch.full((1, H), 1e-3, device="cuda")
        p = (x, torch.zeros(1, H, device="cuda").half(), wg, one, wu, su, wd, sd)
        y = ra.int8_moe(*p, top_k=1)
        gate = wg[0, :, 0].double()
        ref = gate * torch.sigmoid(gate) * 1e38 * 0.1
        ref = torch.where(ref.abs() > 65519, torch.sign(ref) * inf_like(ref), ref)
        tol = ref.abs().nan_to_num(posinf=0.0) * (2.0 ** -11 + 2.0 ** -16 + (4 + 1.2 * gate.abs()) * 2.0 ** -23) + 2.0 ** -25
        assert bool(((y[:, :I].double() == ref) | ((y[:, :I].double() - ref).abs() <= tol)).all())
        cpu = ra.int8_moe(*(t.cpu().float() if t.dtype == torch.float16 else t.cpu() for t in p), top_k=1)
        assert bool(((cpu[:, :I].double() - gate.cpu() * torch.sigmoid(gate.cpu()) * 1e37).abs()
                     <= (gate.cpu() * torch.sigmoid(gate.cpu()) * 1e37).abs() * 2.0 ** -20).all())


def inf_like(t):
    return torch.full_like(t, float("inf"))
