"""The mixture-of-experts layer without a GPU: the torch form against a loop
over tokens in 64 bits, the module, refusals and the C ABI's argument checks
(nothing is launched)."""

import ctypes

import pytest
import torch


def _problem(T, H, I, E, seed=0):
    from rotalabs_accel_b200 import quantize_weight_per_channel
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g)
    router = (torch.randn(E, H, generator=g) * 1.5 / H ** 0.5).half()

    def weight(*shape):
        q, s = quantize_weight_per_channel(torch.randn(shape[0] * shape[1], shape[2], generator=g) * 0.05)
        return q.view(shape), s.view(shape[:2])

    return x, router, *weight(E, I, H), *weight(E, I, H), *weight(E, H, I)


def _loop64(x, router, wg, sg, wu, su, wd, sd, k, renorm):
    y = torch.zeros(x.shape, dtype=torch.float64)
    for t in range(x.shape[0]):
        p = torch.softmax(router.double() @ x[t].double(), 0).tolist()
        best = sorted(range(len(p)), key=lambda e: (-p[e], e))[:k]
        total = sum(p[e] for e in best) if renorm else 1.0
        for e in best:
            gate = (wg[e].double() @ x[t].double()) * sg[e].double()
            up = (wu[e].double() @ x[t].double()) * su[e].double()
            y[t] += p[e] / total * ((wd[e].double() @ (gate * torch.sigmoid(gate) * up)) * sd[e].double())
    return y


@pytest.mark.parametrize("k,renorm", [(1, True), (1, False), (3, True), (6, False)])
def test_cpu_layer(k, renorm):
    import rotalabs_accel_b200 as ra
    p = _problem(7, 40, 24, 6)
    y = ra.int8_moe(*p, top_k=k, renormalize=renorm)
    ref = _loop64(*p, k, renorm)
    assert y.dtype == torch.float32 and bool(((y - ref).abs() <= 1e-5 * ref.abs().max()).all())
    y3 = ra.int8_moe(p[0].view(1, 7, 40), *p[1:], top_k=k, renormalize=renorm)
    assert y3.shape == (1, 7, 40) and torch.equal(y3[0], y)
    assert ra.int8_moe(p[0][:0], *p[1:], top_k=k).shape == (0, 40)


def test_ties_take_the_lower_index():
    import rotalabs_accel_b200 as ra
    x, router, *w = _problem(4, 32, 16, 5)
    router[1] = router[4]                                  # equal logits, different experts
    router[[0, 2, 3]] = 0
    x = x * torch.sign(x @ router[1].float()).unsqueeze(1)     # the pair has the largest
    y = ra.int8_moe(x, router, *w, top_k=1)
    only = [t[1:2] for t in w]
    assert torch.equal(y, ra.int8_moe(x, router[1:2], *only, top_k=1))


def test_module():
    import rotalabs_accel_b200 as ra
    g = torch.Generator().manual_seed(3)
    m = ra.Int8MoE(32, 16, 4, 2)
    assert list(m.state_dict()) == ["router_weight", "w_gate", "w_up", "w_down", "scale_gate", "scale_up", "scale_down"]
    with pytest.raises(RuntimeError, match="Weights not quantized"):
        m(torch.randn(2, 32))
    w = [torch.randn(4, *s, generator=g) * 0.1 for s in ((16, 32), (16, 32), (32, 16))]
    m.quantize_weights(torch.randn(4, 32, generator=g), *w)
    x = torch.randn(3, 32, generator=g)
    # one expert alone is the framework's SwiGLU block with that expert's weights
    one = ra.Int8MoE(32, 16, 1, 1)
    one.quantize_weights(torch.zeros(1, 32), *[t[2:3] for t in w])
    block = ra.Int8SwiGLU(32, 16)
    block.quantize_weights(*[t[2] for t in w])
    assert torch.allclose(one(x), block(x), rtol=1e-4, atol=1e-5)
    assert torch.equal(one.w_gate[0], block.w_gate.weight_int8) and torch.equal(one.scale_gate[0], block.w_gate.scale)
    m2 = ra.Int8MoE(32, 16, 4, 2)
    m2.load_state_dict(m.state_dict())
    m2.mark_quantized()
    assert torch.equal(m2(x), m(x))
    assert "num_experts=4, top_k=2" in repr(m)
    with pytest.raises(ValueError, match="top_k"):
        ra.Int8MoE(32, 16, 4, 5)


def test_python_refusals():
    import rotalabs_accel_b200 as ra
    p = list(_problem(2, 32, 16, 4))
    bad = lambda i, t: p[:i] + [t] + p[i + 1:]  # noqa: E731
    with pytest.raises(AssertionError, match="Weight must be INT8"):
        ra.int8_moe(*bad(2, p[2].float()), top_k=2)
    with pytest.raises(AssertionError, match="Hidden dim mismatch"):
        ra.int8_moe(*bad(0, p[0][:, :16]), top_k=2)
    with pytest.raises(AssertionError, match="Weight shape mismatch"):
        ra.int8_moe(*bad(6, p[6].transpose(1, 2)), top_k=2)
    with pytest.raises(AssertionError, match="Scale shape mismatch"):
        ra.int8_moe(*bad(7, p[7][:, :5]), top_k=2)
    for k in (0, 5):
        with pytest.raises(ValueError, match="top_k"):
            ra.int8_moe(*p, top_k=k)


@pytest.fixture(scope="module")
def lib():
    from rotalabs_accel_b200 import build, _capi
    build.build()
    return _capi.load_library()


def test_capi_rejects_bad_arguments(lib):
    n0 = lib.rla_launch_count()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)   # never dereferenced: validation fails first

    def moe(x=p, ldx=64, r=p, wg=p, sg=p, wu=p, su=p, wd=p, sd=p, sdt=2, ren=1, y=p, ldy=64, T=4, H=64, I=32, E=8, k=2,
            ws=p, wsb=1 << 20):
        return lib.rla_moe(x, ldx, r, wg, sg, wu, su, wd, sd, sdt, ren, y, ldy, T, H, I, E, k, ws, wsb, None)

    assert moe(T=-1) == 1 and moe(H=0) == 1 and moe(I=0) == 1 and moe(E=0) == 1
    assert moe(k=0) == 1 and moe(k=9) == 1
    assert moe(T=33) == 2 and moe(E=257) == 2 and moe(E=64, k=33) == 2
    assert moe(H=72, ldx=72, ldy=72) == 2 and moe(I=40) == 2
    assert moe(H=1 << 18, ldx=1 << 18, ldy=1 << 18) == 1 and moe(I=1 << 18) == 1
    assert moe(sdt=0) == 1 and moe(sdt=3) == 1
    for name in ("x", "r", "wg", "sg", "wu", "su", "wd", "sd", "y"):
        assert moe(**{name: None}) == 1
    assert moe(ldx=63) == 1 and moe(ldy=63) == 1
    assert moe(x=odd) == 2 and moe(r=odd) == 2 and moe(wg=odd) == 2 and moe(wu=odd) == 2 and moe(wd=odd) == 2
    assert moe(ldx=68) == 2
    need = lib.rla_moe_workspace_size(4, 32, 2)
    assert need >= 4 * 2 * 32 * 2 and need % 256 == 0      # fp16 activations of 8 (token, expert) pairs, and the routing
    assert moe(ws=None) == 4 and moe(wsb=need - 1) == 4 and moe(ws=ctypes.c_void_p(4096 + 128)) == 4
    assert b"workspace" in lib.rla_last_error()
    assert moe(T=0) == 0
    assert lib.rla_moe_workspace_size(33, 32, 2) == 0 and lib.rla_moe_workspace_size(0, 32, 2) == 0
    assert lib.rla_launch_count() == n0
