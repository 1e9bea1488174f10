"""Row kernels with many rows -- the ring of bulk copies (16-byte aligned rows
of 2048 to 16384 elements, four rows for each SM and more) and the forms beside
it -- against their formulas in 64 bits, row by row.

Tolerances: half a step of the output's type for its one rounding (fp16 2^-11,
bf16 2^-8, half a step of q), and for the fp32 arithmetic before it 2^-18 as in the
tests of few rows (at most 74 additions, a root, a division and products); SwiGLU's
exponential 2^-20 and |gate| 2^-23.5 for negative gates.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -18
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _rows(M, K, pad, start, g, dtype, scale=1.0):
    """M rows of K values, K + pad elements apart, `start` elements into a
    buffer of 77 everywhere else."""
    buf = torch.full((M * (K + pad) + start + 8,), 77.0, device="cuda", dtype=dtype)
    v = buf[start:start + M * (K + pad)].view(M, K + pad)[:, :K]
    v.copy_(torch.randn(M, K, generator=g, device="cuda") * scale)
    return v


def _check_int8(q, s, v, rel, what):
    top = v.abs().amax(-1)
    s64 = torch.where(top > 0, top / 127, torch.ones_like(top))
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert bool(((s.double() - s64).abs() <= s64 * rel).all()), what
    assert bool(((q.double() - v / s64.unsqueeze(-1)).abs() <= 0.5 + 127 * 2 * rel).all()), what
    assert bool((q.abs().amax(-1)[top > 0] == 127).all()), what


def _norm64(h, w, eps):
    d = h.double()
    return d / (d.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()


# every width class of the ring (2 and 4 vectors a thread, 256 and 512 threads,
# 1 to 3 CTAs an SM, the weight held or read again), its ends, ragged in a
# thread's vectors; beyond it; rows that 4 and 1 elements divide; strided rows
SIZES = [(600, 2048, 0), (1000, 2056, 0), (2048, 4096, 0), (601, 4104, 8), (700, 8192, 0), (593, 8200, 0), (1000, 11008, 16),
         (600, 13824, 0), (700, 13832, 0), (600, 16384, 0), (610, 16392, 0), (700, 2040, 0), (600, 2044, 0),
         (600, 12300, 4), (600, 3001, 0), (600, 4096, 4), (600, 4096, 1), (4097, 2048, 0)]


@pytest.mark.parametrize("M,K,pad", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_norms(cuda_lib, M, K, pad, dtype):
    import rotalabs_accel_b200 as ra
    g = torch.Generator(device="cuda").manual_seed(M + K + pad)
    x, r = _rows(M, K, pad, 0, g, dtype), _rows(M, K, pad, 0, g, dtype, 2.0)
    x0, r0 = x.clone(), r.clone()
    for i, wdt in enumerate((F32, F16, BF16)):
        w = (torch.rand(K, generator=g, device="cuda") + 0.5).to(wdt)
        for res in (r, None):
            if res is None and i != (M + K) % 3:
                continue
            h64 = (x.float() + r.float()).to(dtype) if res is not None else x
            v = _norm64(h64, w, 1e-5)
            y, h = ra.add_rmsnorm(x, res, w, 1e-5)
            assert torch.equal(h, h64) and y.dtype == dtype
            assert bool(((y.double() - v).abs() <= v.abs() * (_half(dtype) + EPS) + 2.0 ** -25).all())
            q, s, h = ra.add_rmsnorm_int8(x, res, w, 1e-5)
            assert torch.equal(h, h64)
            _check_int8(q, s, v, EPS, (M, K, pad, dtype, wdt))
    assert torch.equal(x, x0) and torch.equal(r, r0)


@pytest.mark.parametrize("M,K,pad", SIZES)
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_swiglu(cuda_lib, M, K, pad, dtype):
    import rotalabs_accel_b200 as ra
    g = torch.Generator(device="cuda").manual_seed(M + K + pad + 1)
    gate, up = _rows(M, K, pad, 0, g, dtype, 1.5), _rows(M, K, pad, 0, g, dtype, 1.5)
    q, s = ra.swiglu_int8(gate, up)
    d = gate.double()
    _check_int8(q, s, d * torch.sigmoid(d) * up.double(), 2.0 ** -20 + 9 * 2.0 ** -23.5, (M, K, pad, dtype))


@pytest.mark.parametrize("K", [2048, 4096, 8192, 11008, 16384])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_special_rows_late_in_a_run(cuda_lib, K, dtype):
    """Infinite, NaN and zero rows among ordinary ones, after the ring has
    wrapped and at the last row: they spoil no other row."""
    import rotalabs_accel_b200 as ra
    g = torch.Generator(device="cuda").manual_seed(K)
    M = 4000
    x, r = _rows(M, K, 0, 0, g, dtype), _rows(M, K, 0, 0, g, dtype)
    w = torch.rand(K, generator=g, device="cuda") + 0.5
    inf, nan = [5, 1501, 2900, M - 1], [444, 3001]
    zero = [0, 1777, 3999 - 148, M - 2]
    x[inf, K - 1], x[nan, K // 2] = float("inf"), float("nan")
    x[zero], r[zero] = 0, 0
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[inf + nan] = True
    h = (x.float() + r.float()).to(dtype)
    v = _norm64(h, w, 1e-6)
    q, s, h2 = ra.add_rmsnorm_int8(x, r, w)
    assert torch.equal(h2.nan_to_num(nan=99.0), h.nan_to_num(nan=99.0))
    assert torch.isnan(s[bad]).all() and not q[bad].any()
    _check_int8(q[~bad], s[~bad], v[~bad], EPS, K)
    assert bool((s[zero] == 1).all()) and not q[zero].any()
    y, _ = ra.add_rmsnorm(x, r, w)
    assert bool(((y.double() - v).abs() <= v.abs() * (_half(dtype) + EPS) + 2.0 ** -25)[~bad].all())
    assert torch.isnan(y[nan]).all() and torch.isnan(y[inf, K - 1]).all()
    q, s = ra.swiglu_int8(x, r)
    assert torch.isnan(s[bad]).all() and not q[bad].any()
    d = x.double()
    _check_int8(q[~bad], s[~bad], (d * torch.sigmoid(d) * r.double())[~bad], 2.0 ** -20 + 9 * 2.0 ** -23.5, K)


@pytest.mark.parametrize("K,pad", [(2048, 16), (4096, 8), (8192, 24), (11008, 16), (16384, 8), (4096, 3)])
def test_nothing_beside_the_outputs_is_written(cuda_lib, K, pad):
    """Through the C ABI, with outputs inside larger buffers (rows 8-byte and,
    where pad allows, 16-byte aligned)."""
    lib, M = cuda_lib, 650
    g = torch.Generator(device="cuda").manual_seed(K)
    x, r = _rows(M, K, 0, 0, g, F16), _rows(M, K, 0, 0, g, F16)
    w = torch.rand(K, generator=g, device="cuda") + 0.5
    ld = K + pad
    stream = torch.cuda.current_stream().cuda_stream

    def outputs():
        return (torch.full((M + 2, ld), 55, dtype=torch.int8, device="cuda"), torch.full((M + 2, ld), 3.0, device="cuda").half(),
                torch.full((M + 2, ld), 3.0, device="cuda").half(), torch.full((M + 2,), 3.0, device="cuda"))

    q, h, y, s = outputs()
    h64 = (x.float() + r.float()).half()
    st = lib.rla_add_rmsnorm_int8(x.data_ptr(), K, r.data_ptr(), K, 1, w.data_ptr(), 2, 1e-6, h.data_ptr() + 2 * ld, ld,
                                  q.data_ptr() + ld, ld, s.data_ptr() + 4, M, K, stream)
    torch.cuda.synchronize()
    assert st == 0 and torch.equal(h[1:1 + M, :K], h64)
    _check_int8(q[1:1 + M, :K], s[1:1 + M], _norm64(h64, w, 1e-6), EPS, K)
    h[1:1 + M, :K] = 3.0
    st = lib.rla_add_rmsnorm(x.data_ptr(), K, r.data_ptr(), K, 1, w.data_ptr(), 2, 1e-6, h.data_ptr() + 2 * ld, ld,
                             y.data_ptr() + 2 * ld, ld, M, K, stream)
    torch.cuda.synchronize()
    v = _norm64(h64, w, 1e-6)
    assert st == 0 and torch.equal(h[1:1 + M, :K], h64)
    assert bool(((y[1:1 + M, :K].double() - v).abs() <= v.abs() * (2.0 ** -11 + EPS) + 2.0 ** -25).all())
    q2, _, _, s2 = outputs()
    st = lib.rla_swiglu_int8(x.data_ptr(), K, r.data_ptr(), K, 1, q2.data_ptr() + ld, ld, s2.data_ptr() + 4, M, K, stream)
    torch.cuda.synchronize()
    d = x.double()
    assert st == 0
    _check_int8(q2[1:1 + M, :K], s2[1:1 + M], d * torch.sigmoid(d) * r.double(), 2.0 ** -20 + 9 * 2.0 ** -23.5, K)
    for b, fill in ((q, 55), (h, 3.0), (y, 3.0), (q2, 55)):
        b[1:1 + M, :K] = fill
        assert bool((b == fill).all())
    for b in (s, s2):
        b[1:1 + M] = 3.0
        assert bool((b == 3.0).all())


def test_two_streams_every_result(cuda_lib):
    """Products of both kernels, norms and SwiGLU on two streams at once, each
    iteration's results compared (with 64-bit-checked ones of a call alone)."""
    import rotalabs_accel_b200 as ra
    from rotalabs_accel_b200 import _capi
    g = torch.Generator(device="cuda").manual_seed(3)
    cases = []
    for M, N, K in ((1024, 8192, 1024), (16, 1024, 512), (80, 512, 2048), (2048, 4096, 256)):
        q = torch.randint(-128, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
        wt = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        cases.append((q, torch.rand(M, generator=g, device="cuda"), wt, torch.rand(N, generator=g, device="cuda") * 1e-4))
    xs = [_rows(1000, K, 0, 0, g, F16) for K in (4096, 11008)]
    ws = [torch.rand(x.shape[1], generator=g, device="cuda") for x in xs]

    def all_of(reverse):
        out = {}
        for i in (reversed(range(4)) if reverse else range(4)):
            out["g%d" % i] = (ra.int8_gemm_w8a8(*cases[i]),)
            x, w = xs[i % 2], ws[i % 2]
            out["n%d" % i] = ra.add_rmsnorm_int8(x, x, w)
            out["s%d" % i] = ra.swiglu_int8(x, x)
        return out

    want = all_of(False)
    for x, w, i in zip(xs, ws, (0, 1)):
        _check_int8(want["n%d" % i][0], want["n%d" % i][1], _norm64((2 * x.float()).half(), w, 1e-6), EPS, i)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    same = torch.zeros(2, dtype=torch.int64, device="cuda")
    count = 0
    for _ in range(12):
        got = []
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got.append(all_of(bool(k)))
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                for name, parts in want.items():
                    for a, b in zip(got[k][name], parts):
                        same[k] += (a != b).any()
                        count += 1
        torch.cuda.synchronize()
    assert count > 500 and same.tolist() == [0, 0] and _capi.device_error() == 0
