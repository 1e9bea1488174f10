"""The 8-bit activation path on the GPU against its formulas in 64 bits.

Tolerances.  eps-half of the output type for its one rounding (fp16 2^-11,
bf16 2^-8, half a step of q), plus the fp32 arithmetic before it:

* norm: the sum of squares adds at most 64 terms a thread and then two trees
  (10 levels), each addition off by 2^-24 of the sum: 74 * 2^-24, half of it in
  the root; rsqrt 2 ulp, the division, products: under 2^-18 in all (EPS).
* SwiGLU: expf's intrinsic is off by at most 2 + 1.173 |x| ulp, 12 for
  |x| <= 8; with the quotient (2 ulp) and the product under 2^-18.
* product: the sum is exact; its conversion, two products and the addition of
  the bias are off by 2^-24 each of the larger of the two addends.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -18
TYPES = [torch.float16, torch.bfloat16]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rand(shape, g, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _check_rows(q, s, v, what=""):
    """int8 rows q * s against the 64-bit rows v."""
    top = v.abs().amax(-1)
    s64 = torch.where(top > 0, top / 127, torch.ones_like(top))
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and q.shape == v.shape and s.shape == v.shape[:-1]
    assert bool(((s.double() - s64).abs() <= s64 * EPS).all()), what
    assert bool(((q.double() - v / s64.unsqueeze(-1)).abs() <= 0.5 + 127 * EPS).all()), what
    assert bool((q.abs().amax(-1)[top > 0] == 127).all()), what


def _norm64(h, w, eps):
    d = h.double()
    return d / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()


# K: one element, less than a vector, odd, one warp's share and around it, the
# widths of the configurations, more than 8 * 1024 (32 elements a thread), more
# than 32 * 1024 (the row is read twice)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (5, 255), (4, 256), (9, 257), (2, 264), (1, 4096), (7, 4100),
                                 (16, 4097), (3, 8192), (2, 8200), (2, 8193), (3, 11008), (1, 28672), (2, 32768),
                                 (2, 33000), (1, 33001), (1, 65540), (1029, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_add_rmsnorm(cuda_lib, M, K, dtype):
    import rotalabs_accel_b200 as ra
    g = _gen(M * 31 + K)
    x, r = _rand((M, K), g, dtype), _rand((M, K), g, dtype, 2.0)
    for wdt in (torch.float32, torch.float16, torch.bfloat16):
        w = (torch.rand(K, generator=g, device="cuda") + 0.5).to(wdt)
        for res in (r, None):
            y, h = ra.add_rmsnorm(x, res, w, 1e-5)
            assert h is x if res is None else torch.equal(h, (x.float() + r.float()).to(dtype))
            v = _norm64(h, w, 1e-5)
            assert y.dtype == dtype
            assert bool(((y.double() - v).abs() <= v.abs() * (_half(dtype) + EPS) + 2 ** -25).all())
            q, s, h8 = ra.add_rmsnorm_int8(x, res, w, 1e-5)
            assert torch.equal(h8, h)
            _check_rows(q, s, v, f"{M}x{K} {dtype} {wdt}")


@pytest.mark.parametrize("M,N", [(1, 1), (3, 7), (5, 255), (9, 257), (16, 11008), (2, 28672), (3, 4100), (1, 33001),
                                 (1029, 64)])
@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_int8(cuda_lib, M, N, dtype):
    import rotalabs_accel_b200 as ra
    g = _gen(M * 17 + N)
    gate, up = _rand((M, N), g, dtype, 1.5).clamp(-8, 8), _rand((M, N), g, dtype, 1.5)
    q, s = ra.swiglu_int8(gate, up)
    d = gate.double()
    _check_rows(q, s, d * torch.sigmoid(d) * up.double())


def test_swiglu_large_gates(cuda_lib):
    """e^-gate overflows or vanishes: the limits 0 and gate."""
    import rotalabs_accel_b200 as ra
    gate = torch.tensor([[-60000.0, -100.0, -88.0, 0.0, 88.0, 100.0, 300.0, 60000.0]], device="cuda").half()
    up = torch.ones_like(gate)
    q, s = ra.swiglu_int8(gate, up)
    assert torch.equal(q, torch.tensor([[0, 0, 0, 0, 0, 0, 1, 127]], dtype=torch.int8, device="cuda"))
    assert abs(s.item() * 127 / 60000 - 1) < 1e-6
    q, s = ra.swiglu_int8(gate[:, :3].contiguous(), up[:, :3].contiguous())
    assert torch.isfinite(s).all() and bool(((q * s[:, None]).abs() <= 1e-30).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [16, 40, 4096, 33000])
def test_special_rows(cuda_lib, dtype, K):
    import rotalabs_accel_b200 as ra
    g = _gen(K)
    x = _rand((8, K), g, dtype)
    x[0] = 0
    x[1, K // 2] = float("inf")
    x[2, K - 1] = float("nan")
    x[3, 0] = float("-inf")
    x[4] = 0
    x[4, K - 1] = torch.finfo(dtype).smallest_normal / 8   # a subnormal of the type
    x[5] = torch.finfo(dtype).max if dtype == torch.float16 else 1e17
    w = torch.ones(K, device="cuda")
    w[K // 2 + 1] = 0
    q, s, _ = ra.add_rmsnorm_int8(x, None, w)
    assert s[0] == 1 and not q[0].any()
    assert torch.isnan(s[1:4]).all() and not q[1:4].any()
    assert q[4, K - 1] == 127 and s[4] > 0
    assert bool((q[5][w != 0] == 127).all()) and q[5, K // 2 + 1] == 0
    _check_rows(q[6:], s[6:], _norm64(x[6:], w, 1e-6))
    # an infinity under a zero weight is NaN in the product
    x[1, K // 2], x[1, K // 2 + 1] = 0, float("inf")
    q, s, _ = ra.add_rmsnorm_int8(x[1:2], None, w)
    assert torch.isnan(s).all() and not q.any()
    y, _ = ra.add_rmsnorm(x, None, w)
    assert torch.isnan(y[2]).any() and not y[0].any()
    # the addition overflows the type: as T(x + residual)
    big = torch.full((1, K), torch.finfo(dtype).max, dtype=dtype, device="cuda")
    q, s, h = ra.add_rmsnorm_int8(big, big, w)
    assert torch.isinf(h).all() and torch.isnan(s).all() and not q.any()
    # products below 1e-30 (the reciprocal of the maximum would overflow)
    tiny = torch.full((K,), 1e-36, device="cuda")
    q, s, _ = ra.add_rmsnorm_int8(x[6:] * 0.01, None, tiny, 0.0)
    _check_rows(q, s, _norm64(x[6:] * 0.01, tiny, 0.0))
    q, s = ra.swiglu_int8(x, torch.ones_like(x))
    assert s[0] == 1 and torch.isnan(s[2]) and not q[:3].any()


def test_norm_strides_and_shapes(cuda_lib):
    import rotalabs_accel_b200 as ra
    g = _gen(3)
    w = torch.rand(72, generator=g, device="cuda")
    wide = _rand((6, 101), g, torch.float16)
    for x, r in ((wide[:, :72], wide[:, 29:]),                      # odd row stride, odd start
                 (wide[::2, 1:73], wide[::2, 5:77]),
                 (_rand((72, 6), g, torch.float16).t(), wide[:, :72]),   # no unit inner stride
                 (wide[:1, :72].expand(6, 72), wide[:, :72])):       # broadcast rows
        q, s, h = ra.add_rmsnorm_int8(x, r, w)
        assert torch.equal(h, (x.float() + r.float()).half())
        _check_rows(q, s, _norm64(h, w, 1e-6))
    x3 = _rand((2, 3, 72), g, torch.float16)
    q, s, h = ra.add_rmsnorm_int8(x3, x3, w)
    assert q.shape == x3.shape and s.shape == (2, 3) and h.shape == x3.shape
    y, h = ra.add_rmsnorm(x3, None, w)
    assert y.shape == x3.shape and h is x3
    q, s = ra.swiglu_int8(x3, x3)
    assert q.shape == x3.shape and s.shape == (2, 3)
    q1, s1, _ = ra.add_rmsnorm_int8(x3[0, 0], None, w)   # one row, no batch dimension
    assert q1.shape == (72,) and s1.shape == ()
    # gate and up as the two halves of one buffer
    both = _rand((5, 144), g, torch.float16)
    q, s = ra.swiglu_int8(both[:, :72], both[:, 72:])
    d = both[:, :72].double()
    _check_rows(q, s, d * torch.sigmoid(d) * both[:, 72:].double())
    for shape in ((0, 72), (2, 0, 72)):
        q, s, h = ra.add_rmsnorm_int8(torch.empty(shape, device="cuda").half(), None, w)
        assert q.shape == shape and s.shape == shape[:-1]
    q, s, _ = ra.add_rmsnorm_int8(torch.empty(3, 0, device="cuda").half(), None, w[:0])
    assert q.shape == (3, 0) and torch.equal(s, torch.ones(3, device="cuda"))


def _gemm64(q, sx, w, sw, b=None):
    p = (q.double() @ w.double().t()) * sw.double() * sx.double().unsqueeze(1)
    y = p if b is None else p + b.double()
    tol = y.abs() * 2.0 ** -11 + 2.0 ** -22 * (p.abs() + (0 if b is None else b.double().abs())) + 2.0 ** -25
    return y, tol


def _gemm_case(M, N, K, g, sdt=torch.float32, bias=None):
    q = torch.randint(-128, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    sx = torch.rand(M, generator=g, device="cuda") * 0.02 + 1e-3
    sw = (torch.rand(N, generator=g, device="cuda") * 1e-3 + 1e-4).to(sdt)
    b = None if bias is None else torch.randn(N, generator=g, device="cuda").to(bias)
    return q, sx, w, sw, b


def _gemm_check(q, sx, w, sw, b=None):
    import rotalabs_accel_b200 as ra
    y = ra.int8_gemm_w8a8(q, sx, w, sw, b)
    ref, tol = _gemm64(q, sx, w, sw, b)
    assert y.dtype == torch.float16 and y.shape == ref.shape
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} wrong, first at {bad.nonzero()[0].tolist()}"
    return y


# tokens around every tile width, channels and K around a tile and a k block
@pytest.mark.parametrize("M", [1, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 256, 257, 600])
@pytest.mark.parametrize("N,K", [(1, 16), (127, 112), (129, 128), (256, 144), (1000, 2064)])
def test_w8a8_sizes(cuda_lib, M, N, K):
    g = _gen(M * 7 + N * 3 + K)
    _gemm_check(*_gemm_case(M, N, K, g))
    _gemm_check(*_gemm_case(M, N, K, g, torch.float16, torch.float16 if M % 2 else torch.float32))


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (16, 14336, 4096), (8, 4096, 11008), (333, 1001, 4112),
                                   (2048, 4096, 1024), (5, 1024, 28672), (100, 128, 28672)])
def test_w8a8_configurations(cuda_lib, M, N, K):
    from rotalabs_accel_b200 import _capi
    _gemm_check(*_gemm_case(M, N, K, _gen(M + N + K), torch.float32, torch.float16))
    assert _capi.device_error() == 0


# many tiles: the persistent CTA pairs, ragged on every side, one to some tiles
# a pair, one k block, more tokens than a group of tiles holds
@pytest.mark.parametrize("M,N,K", [(2000, 3001, 272), (300, 9500, 144), (20000, 130, 1040), (1025, 5000, 16),
                                   (4097, 2049, 128), (700, 20000, 4112), (9000, 1500, 4096)])
def test_w8a8_many_tiles(cuda_lib, M, N, K):
    from rotalabs_accel_b200 import _capi
    _gemm_check(*_gemm_case(M, N, K, _gen(M + N + K), torch.float16, torch.float32 if M % 2 else None))
    assert _capi.device_error() == 0


# one tile and several of each kernel, with the slices of K joined and not; the
# width of a store follows the alignment of y and of its rows
@pytest.mark.parametrize("M,N,K", [(33, 261, 144), (20, 203, 4112), (130, 5003, 272), (700, 9999, 2064),
                                   (2049, 6001, 1040)])
def test_w8a8_output_alignments(cuda_lib, M, N, K):
    lib = cuda_lib
    q, sx, w, sw, b = _gemm_case(M, N, K, _gen(M + N), torch.float32, torch.float16)
    ref, tol = _gemm64(q, sx, w, sw, b)
    stream = torch.cuda.current_stream().cuda_stream
    width = (N + 7) // 8 * 8 + 16
    outs = []
    for pad, start in ((0, 0), (8, 8), (0, 4), (4, 0), (4, 4), (2, 0), (0, 2), (1, 0), (0, 1), (3, 3)):
        ld = width + pad
        buf = torch.full((M + 2, ld), 3.0, dtype=torch.float16, device="cuda")
        st = lib.rla_w8a8_gemm(q.data_ptr(), K, sx.data_ptr(), w.data_ptr(), K, sw.data_ptr(), 2, b.data_ptr(), 1,
                               buf.data_ptr() + 2 * (ld + start), ld, M, N, K, None, 0, stream)
        torch.cuda.synchronize()
        assert st == 0
        outs.append(buf[1:1 + M, start:start + N].clone())
        buf[1:1 + M, start:start + N] = 3.0
        assert bool((buf == 3.0).all()), (pad, start)
    assert bool(((outs[0].double() - ref).abs() <= tol).all())
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_w8a8_very_many_tokens(cuda_lib):
    """More token tiles than a grid has rows."""
    import rotalabs_accel_b200 as ra
    M, N, K = 8_400_001, 8, 16
    q, sx, w, sw, _ = _gemm_case(M, N, K, _gen(1))
    y = ra.int8_gemm_w8a8(q, sx, w, sw)
    for part in (slice(0, 1000), slice(65535 * 128 - 500, 65535 * 128 + 500), slice(M - 1000, M)):
        ref, tol = _gemm64(q[part], sx[part], w, sw)
        assert bool(((y[part].double() - ref).abs() <= tol).all())


# rows that TMA cannot address: odd K, odd strides, odd starts
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (3, 5, 15), (17, 130, 257), (70, 33, 4099), (300, 64, 31)])
def test_w8a8_unaligned(cuda_lib, M, N, K):
    g = _gen(M + N + K)
    q, sx, w, sw, b = _gemm_case(M, N, K, g, torch.float32, torch.float32)
    y = _gemm_check(q, sx, w, sw, b)
    import rotalabs_accel_b200 as ra

    def placed(t, stride, start):
        buf = torch.full((t.shape[0] * stride + start + 16,), 77, dtype=torch.int8, device="cuda")
        v = buf[start:start + t.shape[0] * stride].view(t.shape[0], stride)[:, :t.shape[1]]
        v.copy_(t)
        return v

    for qs, ws in ((placed(q, K + 3, 5), w), (q, placed(w, K + 1, 1)), (placed(q, K + 16, 3), placed(w, K + 2, 7)),
                   (placed(q, (K + 31) // 16 * 16, 16), placed(w, (K + 31) // 16 * 16, 32)),
                   (q.t().contiguous().t(), w.t().contiguous().t())):
        assert torch.equal(ra.int8_gemm_w8a8(qs, sx, ws, sw, b), y)
    # a broadcast row
    assert torch.equal(ra.int8_gemm_w8a8(q[:1].expand(M, K), sx, w, sw, b),
                       ra.int8_gemm_w8a8(q[:1].repeat(M, 1), sx, w, sw, b))


def test_w8a8_extremes(cuda_lib):
    import rotalabs_accel_b200 as ra
    for M in (1, 40, 300):
        for a, b in ((-128, -128), (-128, 127), (127, 127)):
            K = 131071
            q = torch.full((M, K), a, dtype=torch.int8, device="cuda")
            w = torch.full((3, K), b, dtype=torch.int8, device="cuda")
            sx = torch.full((M,), 2.0 ** -20, device="cuda")
            _gemm_check(q, sx, w, torch.full((3,), 2.0 ** -4, device="cuda"))
    with pytest.raises(RuntimeError, match="131072"):
        ra.int8_gemm_w8a8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), torch.ones(1, device="cuda"),
                          torch.zeros(2, 131072, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    # NaN rows stay NaN, others untouched; results above fp16's range are infinite
    q, sx, w, sw, _ = _gemm_case(20, 140, 256, _gen(9))
    sx[3] = float("nan")
    sx[7] = 1e30
    y = ra.int8_gemm_w8a8(q, sx, w, sw)
    assert torch.isnan(y[3]).all() and torch.isinf(y[7]).any()
    keep = [i for i in range(20) if i not in (3, 7)]
    assert torch.isfinite(y[keep]).all()


def test_w8a8_empty(cuda_lib):
    import rotalabs_accel_b200 as ra
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device="cuda")
    o = lambda *s: torch.ones(*s, device="cuda")
    assert ra.int8_gemm_w8a8(z(0, 64), o(0), z(8, 64), o(8)).shape == (0, 8)
    assert ra.int8_gemm_w8a8(z(3, 64), o(3), z(0, 64), o(0)).shape == (3, 0)
    y = ra.int8_gemm_w8a8(z(3, 0), o(3), z(8, 0), o(8), torch.arange(8, device="cuda").half())
    assert torch.equal(y, torch.arange(8, device="cuda").half().expand(3, 8))
    assert not ra.int8_gemm_w8a8(z(3, 0), o(3), z(8, 0), o(8)).any()
    x = torch.randint(-9, 9, (2, 3, 32), dtype=torch.int8, device="cuda")
    w = torch.randint(-9, 9, (5, 32), dtype=torch.int8, device="cuda")
    y = ra.int8_gemm_w8a8(x, o(2, 3), w, o(5))
    assert torch.equal(y.long(), (x.double() @ w.double().t()).long())
    assert torch.equal(ra.int8_gemm_w8a8(x[0, 0], o(1)[0], w, o(5)), y[0, 0])


def test_gpu_refusals(cuda_lib):
    import rotalabs_accel_b200 as ra
    x = torch.zeros(2, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ra.add_rmsnorm(x, None, w)
    with pytest.raises(TypeError, match="x's dtype"):
        ra.add_rmsnorm_int8(x.half(), x.bfloat16(), w)
    with pytest.raises(TypeError, match="weight dtype"):
        ra.add_rmsnorm(x.half(), None, w.double())
    with pytest.raises(TypeError, match="gate's dtype"):
        ra.swiglu_int8(x.half(), x.bfloat16())
    with pytest.raises(RuntimeError, match="same CUDA device"):
        ra.add_rmsnorm(x.half(), None, w.cpu())
    with pytest.raises(RuntimeError, match="same CUDA device"):
        ra.add_rmsnorm(x.half(), x.half().cpu(), w)
    with pytest.raises(RuntimeError, match="eps"):
        ra.add_rmsnorm(x.half(), None, w, -1.0)
    with pytest.raises(AssertionError, match="Hidden dim mismatch"):
        ra.add_rmsnorm(x.half(), None, w[:5])
    with pytest.raises(AssertionError, match="Residual shape mismatch"):
        ra.add_rmsnorm_int8(x.half(), x.half()[:1], w)
    with pytest.raises(AssertionError, match="Gate and up shape"):
        ra.swiglu_int8(x.half(), x.half()[:, :5])
    q, s = torch.zeros(2, 64, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda")
    for args, what in (((x, s, q, s), "Activations must be INT8"), ((q, s, x, s), "Weight must be INT8"),
                       ((q, s, q[:, :5], s), "Weight shape mismatch"), ((q, s[:1], q, s), "Activation scale shape"),
                       ((q, s, q, s[:1]), "Scale shape mismatch")):
        with pytest.raises(AssertionError, match=what):
            ra.int8_gemm_w8a8(*args)
    with pytest.raises(RuntimeError, match="same CUDA device"):
        ra.int8_gemm_w8a8(q, s, q.cpu(), s)
    with pytest.raises(TypeError, match="x_scale must be float32"):
        ra.int8_gemm_w8a8(q, s.half(), q, s)
    with pytest.raises(TypeError, match="float32 or float16"):
        ra.int8_gemm_w8a8(q, s, q, s.bfloat16())


def _layer(hidden, inter, g):
    import rotalabs_accel_b200 as ra
    mlp = ra.Int8SwiGLU(hidden, inter).cuda()
    mlp.quantize_weights(_rand((inter, hidden), g, scale=0.02), _rand((inter, hidden), g, scale=0.02),
                         _rand((hidden, inter), g, scale=0.02))
    return mlp


@pytest.mark.parametrize("M", [1, 16, 200])
def test_layer(cuda_lib, M):
    """add_rmsnorm_int8 -> gate/up -> swiglu_int8 -> down, as a layer runs
    them, against the same roundings in 64 bits."""
    import rotalabs_accel_b200 as ra
    g = _gen(M)
    mlp = _layer(512, 1376, g)
    x, r = _rand((M, 512), g, torch.float16), _rand((M, 512), g, torch.float16)
    w = torch.rand(512, generator=g, device="cuda") + 0.5
    q, s, h = ra.add_rmsnorm_int8(x, r, w)
    y = mlp.forward_w8a8(q, s)
    gate, tg = _gemm64(q, s, mlp.w_gate.weight_int8, mlp.w_gate.scale)
    up, tu = _gemm64(q, s, mlp.w_up.weight_int8, mlp.w_up.scale)
    a = gate * torch.sigmoid(gate) * up
    # |silu'| <= 1.1: the error of a from gate's and up's, and half a step of q
    ta = 1.1 * tg * up.abs() + (gate * torch.sigmoid(gate)).abs() * tu + a.abs() * EPS
    step = (a.abs() + ta).amax(-1, keepdim=True) / 127
    ta = ta + 0.5 * step * (1 + 254 * EPS) + a.abs() * EPS
    wd = mlp.w_down.weight_int8.double() * mlp.w_down.scale.double()[:, None]
    ref, tol = a @ wd.t(), ta @ wd.abs().t()
    assert bool(((y.double() - ref).abs() <= (tol + ref.abs()) * 2.0 ** -10 + tol + 2.0 ** -25).all())
    # and close to the 16-bit path as a whole: the steps of two quantizations
    # (max / 127 / sqrt(12) each, the maximum some ten times the mean square)
    ref16 = mlp(ra.add_rmsnorm(x, r, w)[0]).float()
    assert (y.float() - ref16).norm() < 0.1 * ref16.norm()


def test_streams_graph_and_ops(cuda_lib):
    """Another stream than the default, a captured and replayed layer, the
    registered ops, and results that do not change from run to run."""
    import rotalabs_accel_b200 as ra
    g = _gen(5)
    mlp = _layer(256, 768, g)
    w = torch.rand(256, generator=g, device="cuda") + 0.5
    xs = [_rand((24, 256), g, torch.float16) for _ in range(3)]
    r = _rand((24, 256), g, torch.float16)
    odd = torch.randint(-99, 99, (33, 257), generator=g, device="cuda", dtype=torch.int8)   # scratch inside the graph
    so = torch.rand(33, generator=g, device="cuda") * 1e-3

    def run(x):
        q, s, h = ra.add_rmsnorm_int8(x, r, w)
        return mlp.forward_w8a8(q, s), h, ra.int8_gemm_w8a8(odd, so, odd, so)

    want = [run(x) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [run(x) for x in xs]
    side.synchronize()
    for a, b in zip(want, other):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(x)
    for k in (1, 2, 0):
        x.copy_(xs[k])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(u, v) for u, v in zip(out, want[k]))
    q, s, h = torch.ops.rla.add_rmsnorm_int8(xs[0], r, w, 1e-6)
    q2, s2, h2 = ra.add_rmsnorm_int8(xs[0], r, w)
    assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h, h2)
    y, h = torch.ops.rla.add_rmsnorm(xs[0], r, w, 1e-6)
    assert torch.equal(y, ra.add_rmsnorm(xs[0], r, w)[0])
    gate = torch.ops.rla.w8a8_gemm(q, s, mlp.w_gate.weight_int8, mlp.w_gate.scale)
    up = torch.ops.rla.w8a8_gemm(q, s, mlp.w_up.weight_int8, mlp.w_up.scale)
    q, s = torch.ops.rla.swiglu_int8(gate, up)
    assert torch.equal(torch.ops.rla.w8a8_gemm(q, s, mlp.w_down.weight_int8, mlp.w_down.scale), want[0][0])


def test_two_streams_at_once(cuda_lib):
    """Products of both kernels (CTA pairs and split clusters down to one k
    block a CTA), norms and SwiGLU on two streams at the same time, from two
    host threads."""
    import threading
    import rotalabs_accel_b200 as ra
    from rotalabs_accel_b200 import _capi
    g = _gen(21)
    cases = [_gemm_case(M, N, K, g) for M, N, K in ((1024, 8192, 1024), (16, 1024, 512), (32, 2048, 1024), (80, 512, 2048),
                                                    (128, 4096, 512), (2048, 4096, 256))]
    x = _rand((2048, 4096), g, torch.float16)
    w = torch.rand(4096, generator=g, device="cuda")

    def all_of(order):
        out = {}
        for i in order:
            out[i] = ra.int8_gemm_w8a8(*cases[i][:4])
        out["n"] = ra.add_rmsnorm_int8(x, x, w)
        out["s"] = ra.swiglu_int8(x, x)
        return out

    want = all_of(range(len(cases)))
    torch.cuda.synchronize()
    got, streams = {}, [torch.cuda.Stream() for _ in range(2)]

    def work(k):
        with torch.cuda.stream(streams[k]):
            for _ in range(30):
                got[k] = all_of(range(len(cases)) if k else reversed(range(len(cases))))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        for i in range(len(cases)):
            assert torch.equal(got[k][i], want[i])
        assert all(torch.equal(a, b) for n in ("n", "s") for a, b in zip(got[k][n], want[n]))
    assert _capi.device_error() == 0


def test_first_call_inside_a_capture(cuda_lib):
    """Nothing of a first call (attributes, occupancy) disturbs a capture."""
    import subprocess
    import sys
    code = """
import torch, rotalabs_accel_b200 as ra
x = torch.randn(700, 4096, device="cuda").half(); w = torch.ones(4096, device="cuda")
wt = torch.randint(-9, 9, (512, 4096), dtype=torch.int8, device="cuda"); sw = torch.ones(512, device="cuda") * 1e-3
r = torch.randn(4, 4096, device="cuda").half()
wg = torch.randint(-9, 9, (4, 32, 4096), dtype=torch.int8, device="cuda"); sg = torch.ones(4, 32, device="cuda") * 1e-3
wd = torch.randint(-9, 9, (4, 4096, 32), dtype=torch.int8, device="cuda"); sd = torch.ones(4, 4096, device="cuda") * 1e-3
torch.cuda.synchronize()
def run():
    q, s, h = ra.add_rmsnorm_int8(x, x, w)
    return (ra.int8_gemm_w8a8(q, s, wt, sw), ra.int8_gemm_w8a8(q[:3], s[:3], wt, sw), *ra.swiglu_int8(x, h),
            ra.int8_moe(h[:9], r, wg, sg, wg, sg, wd, sd, top_k=2))
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = run()
g.replay(); torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(out, run()))
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_rows_around_the_outputs_stay(cuda_lib):
    """Through the C ABI, with outputs inside larger buffers: nothing beside
    the [M, N] outputs is written."""
    lib = cuda_lib
    g = _gen(11)
    M, N, K = 21, 150, 272
    q, sx, w, sw, _ = _gemm_case(M, N, K, g)
    buf = torch.full((M + 4, N + 7), 3.0, dtype=torch.float16, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    st = lib.rla_w8a8_gemm(q.data_ptr(), K, sx.data_ptr(), w.data_ptr(), K, sw.data_ptr(), 2, None, 0,
                           buf.data_ptr() + 2 * ((N + 7) * 2 + 3), N + 7, M, N, K, None, 0, stream)
    torch.cuda.synchronize()
    assert st == 0
    ref, tol = _gemm64(q, sx, w, sw)
    assert bool(((buf[2:2 + M, 3:3 + N].double() - ref).abs() <= tol).all())
    buf[2:2 + M, 3:3 + N] = 3.0
    assert bool((buf == 3.0).all())
    x = _rand((M, K), g, torch.float16)
    wn = torch.ones(K, device="cuda")
    qb = torch.full((M + 2, K + 5), 55, dtype=torch.int8, device="cuda")
    hb = torch.full((M + 2, K + 5), 3.0, dtype=torch.float16, device="cuda")
    sb = torch.full((M + 2,), 3.0, device="cuda")
    st = lib.rla_add_rmsnorm_int8(x.data_ptr(), K, x.data_ptr(), K, 1, wn.data_ptr(), 2, 1e-6,
                                  hb.data_ptr() + 2 * (K + 5), K + 5, qb.data_ptr() + K + 5, K + 5, sb.data_ptr() + 4,
                                  M, K, stream)
    torch.cuda.synchronize()
    assert st == 0
    assert torch.equal(hb[1:1 + M, :K], (x.float() * 2).half())
    _check_rows(qb[1:1 + M, :K], sb[1:1 + M], _norm64(hb[1:1 + M, :K], wn, 1e-6))
    qb[1:1 + M, :K], hb[1:1 + M, :K], sb[1:1 + M] = 55, 3.0, 3.0
    assert bool((qb == 55).all()) and bool((hb == 3.0).all()) and bool((sb == 3.0).all())
