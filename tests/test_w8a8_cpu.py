"""The 8-bit activation path without a GPU: the CPU forms against the formulas
in 64 bits, the module path, and the C ABI's argument checks (nothing is
launched)."""

import ctypes

import pytest
import torch


def _rows64(v):
    top = v.abs().amax(-1)
    s = torch.where(top > 0, top / 127, torch.ones_like(top))
    return v / s.unsqueeze(-1), s


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [True, False])
def test_add_rmsnorm_cpu(dtype, residual):
    import rotalabs_accel_b200 as ra
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 5, 72, generator=g).to(dtype)
    r = torch.randn(3, 5, 72, generator=g).to(dtype) if residual else None
    w = torch.rand(72, generator=g) + 0.5
    y, h = ra.add_rmsnorm(x, r, w, 1e-5)
    assert y.dtype == dtype and y.shape == x.shape
    assert torch.equal(h, (x.float() + r.float()).to(dtype)) if residual else h is x
    d = h.double()
    v = d / (d.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    half = torch.finfo(dtype).eps / 2
    assert bool(((y.double() - v).abs() <= v.abs() * (half + 2 ** -19) + 1e-7).all())
    q, s, h2 = ra.add_rmsnorm_int8(x, r, w, 1e-5)
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and s.shape == (3, 5) and torch.equal(h, h2)
    t, s64 = _rows64(v)
    assert bool(((s.double() - s64).abs() <= s64 * 2 ** -18).all())
    assert bool(((q.double() - t).abs() <= 0.5 + 127 * 2 ** -18).all())


def test_zero_and_nonfinite_rows_cpu():
    import rotalabs_accel_b200 as ra
    x = torch.randn(4, 16).half()
    x[0] = 0
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    q, s, _ = ra.add_rmsnorm_int8(x, None, torch.ones(16))
    assert s[0] == 1 and not q[0].any()
    assert torch.isnan(s[1:3]).all() and not q[1:3].any()
    assert torch.isfinite(s[3]) and q[3].abs().max() == 127
    q, s = ra.swiglu_int8(x, torch.ones_like(x))
    assert s[0] == 1 and torch.isnan(s[1:3]).all() and not q[:3].any()
    q, s, _ = ra.add_rmsnorm_int8(torch.zeros(2, 0).half(), None, torch.ones(0))
    assert q.shape == (2, 0) and torch.equal(s, torch.ones(2))


def test_w8a8_cpu_is_exact_and_module_path():
    import rotalabs_accel_b200 as ra
    g = torch.Generator().manual_seed(2)
    q = torch.randint(-128, 128, (2, 3, 100), generator=g, dtype=torch.int8)
    w = torch.randint(-128, 128, (7, 100), generator=g, dtype=torch.int8)
    sx, sw = torch.rand(2, 3, generator=g), torch.rand(7, generator=g)
    b = torch.randn(7, generator=g)
    y = ra.int8_gemm_w8a8(q, sx * 1e-3, w, sw * 1e-2, b)
    ref = (q.double() @ w.double().t()) * (sw * 1e-2).double() * (sx * 1e-3).double().unsqueeze(-1) + b.double()
    assert y.shape == (2, 3, 7) and y.dtype == torch.float16
    assert bool(((y.double() - ref).abs() <= ref.abs() * 2 ** -11 + 2 ** -20).all())
    m = ra.Int8SwiGLU(64, 96)
    with pytest.raises(RuntimeError, match="Weights not quantized"):
        m.forward_w8a8(q, sx)
    m.quantize_weights(torch.randn(96, 64, generator=g) * 0.1, torch.randn(96, 64, generator=g) * 0.1,
                       torch.randn(64, 96, generator=g) * 0.1)
    x = torch.randn(5, 64, generator=g)
    xq, xs, _ = ra.add_rmsnorm_int8(x, None, torch.ones(64))
    y = m.forward_w8a8(xq, xs)
    ref = m(ra.rmsnorm(x, torch.ones(64)))
    # two more 8-bit roundings (half a step of 127 each way) than the 16-bit path
    assert (y.float() - ref).abs().max() < 0.05 * ref.abs().max()


def test_python_refusals():
    import rotalabs_accel_b200 as ra
    x = torch.zeros(2, 8).half()
    q = torch.zeros(2, 8, dtype=torch.int8)
    w = torch.zeros(4, 8, dtype=torch.int8)
    with pytest.raises(AssertionError, match="Hidden dim mismatch"):
        ra.add_rmsnorm(x, x, torch.ones(9))
    with pytest.raises(AssertionError, match="Residual shape mismatch"):
        ra.add_rmsnorm_int8(x, x[:1], torch.ones(8))
    with pytest.raises(AssertionError, match="Gate and up shape"):
        ra.swiglu_int8(x, x[:, :4])
    with pytest.raises(AssertionError, match="Activations must be INT8"):
        ra.int8_gemm_w8a8(x, torch.ones(2), w, torch.ones(4))
    with pytest.raises(AssertionError, match="Weight must be INT8"):
        ra.int8_gemm_w8a8(q, torch.ones(2), w.half(), torch.ones(4))
    with pytest.raises(AssertionError, match="Weight shape mismatch"):
        ra.int8_gemm_w8a8(q[:, :4], torch.ones(2), w, torch.ones(4))
    with pytest.raises(AssertionError, match="Activation scale shape"):
        ra.int8_gemm_w8a8(q, torch.ones(3), w, torch.ones(4))
    with pytest.raises(AssertionError, match="Scale shape mismatch"):
        ra.int8_gemm_w8a8(q, torch.ones(2), w, torch.ones(5))


@pytest.fixture(scope="module")
def lib():
    from rotalabs_accel_b200 import build, _capi
    build.build()
    return _capi.load_library()


def test_capi_rejects_bad_arguments(lib):
    n0 = lib.rla_launch_count()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)   # never dereferenced: validation fails first

    def norm(x=p, ldx=64, r=p, ldr=64, dt=1, w=p, wdt=2, eps=1e-6, h=p, ldh=64, y=p, ldy=64, M=4, K=64):
        return lib.rla_add_rmsnorm(x, ldx, r, ldr, dt, w, wdt, eps, h, ldh, y, ldy, M, K, None)

    def norm8(x=p, ldx=64, r=p, ldr=64, dt=1, w=p, wdt=2, eps=1e-6, h=p, ldh=64, q=p, ldq=64, s=p, M=4, K=64):
        return lib.rla_add_rmsnorm_int8(x, ldx, r, ldr, dt, w, wdt, eps, h, ldh, q, ldq, s, M, K, None)

    for f in (norm, norm8):
        assert f(M=-1) == 1 and f(K=-1) == 1 and f(K=(1 << 30) + 1) == 1
        assert f(dt=2) == 1 and f(dt=0) == 1 and f(wdt=0) == 1 and f(wdt=7) == 1
        assert f(eps=-1.0) == 1 and f(eps=float("nan")) == 1
        assert f(x=None) == 1 and f(w=None) == 1 and f(h=None) == 1
        assert f(ldx=63) == 1 and f(ldr=63) == 1 and f(ldh=63) == 1
        assert f(M=0) == 0
    assert norm(y=None) == 1 and norm(ldy=63) == 1 and norm(K=0) == 0
    assert norm8(q=None) == 1 and norm8(ldq=63) == 1 and norm8(s=None) == 1 and norm8(K=0, s=None) == 1

    def swiglu(g=p, ldg=64, u=p, ldu=64, dt=1, q=p, ldq=64, s=p, M=4, N=64):
        return lib.rla_swiglu_int8(g, ldg, u, ldu, dt, q, ldq, s, M, N, None)

    assert swiglu(g=None) == 1 and swiglu(u=None) == 1 and swiglu(q=None) == 1 and swiglu(s=None) == 1
    assert swiglu(dt=2) == 1 and swiglu(ldg=63) == 1 and swiglu(ldu=63) == 1 and swiglu(ldq=63) == 1
    assert swiglu(M=-1) == 1 and swiglu(M=0) == 0

    def gemm(x=p, ldx=64, sx=p, w=p, ldw=64, s=p, sdt=2, b=None, bdt=0, y=p, ldy=64, M=4, N=64, K=64, ws=None, wsb=0):
        return lib.rla_w8a8_gemm(x, ldx, sx, w, ldw, s, sdt, b, bdt, y, ldy, M, N, K, ws, wsb, None)

    assert gemm(M=-1) == 1 and gemm(N=-1) == 1 and gemm(K=-1) == 1
    assert gemm(K=131072, ldx=131072, ldw=131072) == 2
    assert gemm(sdt=3) == 1 and gemm(sdt=0) == 1 and gemm(bdt=3, b=p) == 1 and gemm(bdt=1) == 1
    assert gemm(x=None) == 1 and gemm(sx=None) == 1 and gemm(w=None) == 1 and gemm(s=None) == 1 and gemm(y=None) == 1
    assert gemm(ldx=63) == 1 and gemm(ldw=63) == 1 and gemm(ldy=63) == 1
    assert gemm(M=0) == 0 and gemm(N=0) == 0
    # unaligned rows need the workspace
    assert gemm(x=odd) == 4 and gemm(w=odd) == 4 and gemm(ldx=65) == 4 and gemm(ldw=72) == 4
    assert gemm(x=odd, ws=p, wsb=4 * 64 - 1) == 4 and gemm(x=odd, ws=odd, wsb=1 << 20) == 4
    assert b"workspace" in lib.rla_last_error()
    assert lib.rla_launch_count() == n0


def test_workspace_size(lib):
    assert lib.rla_w8a8_workspace_size(3, 5, 17) == 8 * 32
    assert lib.rla_w8a8_workspace_size(0, 5, 17) == 0 and lib.rla_w8a8_workspace_size(3, 5, -1) == 0


def test_ops_on_meta_tensors(lib):
    """Shapes and types for tracing, without computing."""
    from rotalabs_accel_b200 import _capi
    _capi.torch_ops()
    e = lambda *s, dt=torch.float16: torch.empty(*s, dtype=dt, device="meta")  # noqa: E731
    i8, f32 = torch.int8, torch.float32
    y, h = torch.ops.rla.add_rmsnorm(e(3, 8), e(3, 8), e(8, dt=f32))
    assert y.shape == h.shape == (3, 8) and y.dtype == h.dtype == torch.float16
    q, s, h = torch.ops.rla.add_rmsnorm_int8(e(3, 8, dt=torch.bfloat16), e(3, 8, dt=torch.bfloat16), e(8, dt=f32))
    assert (q.dtype, s.dtype, h.dtype) == (i8, f32, torch.bfloat16) and s.shape == (3,)
    q, s = torch.ops.rla.swiglu_int8(e(3, 8), e(3, 8))
    assert (q.dtype, s.dtype) == (i8, f32) and q.shape == (3, 8)
    y = torch.ops.rla.w8a8_gemm(e(3, 8, dt=i8), e(3, dt=f32), e(5, 8, dt=i8), e(5, dt=f32))
    assert y.shape == (3, 5) and y.dtype == torch.float16
    y = torch.ops.rla.moe(e(3, 16), e(4, 16), e(4, 32, 16, dt=i8), e(4, 32), e(4, 32, 16, dt=i8), e(4, 32),
                          e(4, 16, 32, dt=i8), e(4, 16), 2)
    assert y.shape == (3, 16) and y.dtype == torch.float16
    with pytest.raises(RuntimeError, match="Weight shape mismatch"):
        torch.ops.rla.w8a8_gemm(e(3, 8, dt=i8), e(3, dt=f32), e(5, 9, dt=i8), e(5, dt=f32))
