"""The experts' activation between gate/up and down keeps fp32's range and more
than 16 bits: against the layer's formula in 64 bits.

Tolerance, element by element.  A tensor-core sum of n products is off by at
most (n / 8 + 16) * 2^-23 of the sum of their absolute values (an addition for
each instruction and one for each warp, truncated; twice the instructions in
the down product, whose operand has two terms).  a = silu(g) * u carries g's
error (|silu'| <= 1.1) and u's.  The exponential's intrinsic is off by 2 + 1.173 |g|
ulp and the quotient by 2: (4 + 1.2 |g|) * 2^-23, the |g| for negative g only
(the exponential vanishes beside 1 otherwise, up to 8: 2^-18).  The two bf16 terms of a lose half a
step of half a step, 2^-8 * 2^-8.  The coefficients are off by 2^-18; the
result by one fp16 rounding, 2^-11, or 2^-25 where it is subnormal.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -18


def _problem(T, H, I, E, seed, gate, up, down):
    """An int8 layer whose gates, ups and down products are about this large."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").half()
    router = (torch.randn(E, H, generator=g, device="cuda") * 1.5 / H ** 0.5).half()

    def weight(rows, cols, size):
        w = torch.randint(-127, 128, (E, rows, cols), generator=g, device="cuda", dtype=torch.int8)
        s = (torch.rand(E, rows, generator=g, device="cuda") + 0.5) * (size / (73 * cols ** 0.5))
        return w, s

    return x, router, *weight(I, H, gate), *weight(I, H, up), *weight(H, I, down)


def _reference(x, router, wg, sg, wu, su, wd, sd, k):
    """(y, tolerance) in 64 bits, and max |a|."""
    T, H = x.shape
    I = wg.shape[1]
    logits = x.double() @ router.double().t()
    top, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    assert k == router.shape[0] or (top[:, k - 1] - top[:, k]).min().item() > 1e-4, "a tie: another seed"
    c = torch.softmax(top[:, :k], -1)
    y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    tol, most = torch.zeros_like(y), 0.0
    n1, n2 = (H / 8 + 16) * 2.0 ** -23, (2 * I / 8 + 16) * 2.0 ** -23
    for t in range(T):
        xt = x[t].double()
        for j in range(k):
            e = int(ids[t, j])
            Wg, Wu = wg[e].double() * sg[e].double()[:, None], wu[e].double() * su[e].double()[:, None]
            Wd = wd[e].double() * sd[e].double()[:, None]
            gate, up = Wg @ xt, Wu @ xt
            dg, du = n1 * (Wg.abs() @ xt.abs()), n1 * (Wu.abs() @ xt.abs())
            silu = gate * torch.sigmoid(gate)
            a = silu * up
            da = 1.1 * dg * (up.abs() + du) + silu.abs() * du
            da = da + a.abs() * (EPS + 1.2 * 2.0 ** -23 * (-gate).clamp(min=0) + 2.0 ** -16)
            part = Wd @ a
            y[t] += c[t, j] * part
            tol[t] += c[t, j] * (Wd.abs() @ (da + n2 * (a.abs() + da)) + EPS * part.abs())
            most = max(most, a.abs().max().item())
    return y, tol * (1 + 2.0 ** -10) + y.abs() * 2.0 ** -11 + 2.0 ** -25, most


# one to few tokens of an expert (two columns a token), up to 8, 16 and 32 of them
SHAPES = [(1, 64, 48, 2, 1), (3, 256, 272, 3, 2), (9, 128, 144, 6, 2), (8, 256, 128, 1, 1), (5, 128, 1296, 1, 1),
          (14, 144, 400, 1, 1), (16, 128, 528, 2, 1), (32, 256, 272, 2, 1), (29, 272, 128, 1, 1), (32, 512, 144, 40, 4)]


@pytest.mark.parametrize("T,H,I,E,k", SHAPES)
@pytest.mark.parametrize("gate,up,down", [
    (300.0, 300.0, 1e-5),     # |a| far above 65504
    (1.0, 1e15, 1e-15),       # ... and far beyond 2^32
    (2e-5, 2e-5, 1e8),        # |a| about 1e-10, most of it below fp16's smallest subnormal
    (1e-3, 0.1, 1e3),         # |a| in fp16's subnormal range
    (1.5, 1.5, 1.0)])         # ordinary values: no 2^-11 of a is lost
def test_range_of_the_activation(cuda_lib, T, H, I, E, k, gate, up, down):
    import rotalabs_accel_b200 as ra
    p = _problem(T, H, I, E, T + H + I, gate, up, down)
    y = ra.int8_moe(*p, top_k=k)
    ref, tol, most = _reference(*p, k)
    if gate == 300.0:
        assert most > 65504
    assert torch.isfinite(y).all()
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} wrong, first at {bad.nonzero()[0].tolist()}"


@pytest.mark.parametrize("T", [2, 6, 12, 24])
def test_every_weight_and_special_activations(cuda_lib, T):
    """All 256 weights exactly, and an infinite or largest finite activation:
    one channel's activation alone (the others are 0) times its column of the
    down weights."""
    import rotalabs_accel_b200 as ra
    H, I = 256, 64
    x = torch.zeros(T, H, device="cuda").half()
    x[:, 0] = 1.0
    router = torch.zeros(1, H, device="cuda").half()
    wg = torch.zeros(1, I, H, dtype=torch.int8, device="cuda")
    wu = torch.zeros_like(wg)
    wd = torch.zeros(1, H, I, dtype=torch.int8, device="cuda")
    sg = torch.ones(1, I, device="cuda")
    values = torch.arange(-128, 128, device="cuda")
    for channel in (0, 1, 2, 3, 13, 31, 63):
        wg.zero_(), wu.zero_(), wd.zero_()
        wg[0, channel, 0], wu[0, channel, 0] = 100, 1
        wd[0, :, channel] = values.to(torch.int8)
        for size, down in ((0.01, 1.0), (3.0e36, 1e-38), (3.395e36, 1e-37)):   # (bf16(3.395e38) is infinite)
            su, sd = torch.full((1, I), size, device="cuda"), torch.full((1, H), down, device="cuda")
            a = 100 * size                       # silu(100) is 100
            y = ra.int8_moe(x, router, wg, sg, wu, su, wd, sd, top_k=1)
            ref = values.double() * a * down
            # sums beyond fp32's range (a term alone may be 2^-8 larger)
            ref = torch.where(values.abs() * a > 3.40e38, torch.sign(values) * float("inf"), ref)
            sure = ((values.abs() * a - 3.40e38).abs() > 0.03e38) | (values.abs() == 1)
            tol = ref.abs().nan_to_num(posinf=0.0) * (2.0 ** -11 + 2.0 ** -16 + 2 * EPS) + 2.0 ** -25
            same = (y.double() == ref) | ((y.double() - ref).abs() <= tol)
            assert bool(same[:, sure].all()), (channel, size)
        su = torch.full((1, I), float("inf"), device="cuda")
        y = ra.int8_moe(x, router, wg, sg, wu, su, wd, torch.ones(1, H, device="cuda"), top_k=1)
        # (inf * 0 in the other ups makes every sum NaN, as the formula has it)
        assert torch.isnan(y).all()
