"""The mixture-of-experts layer on the GPU against its formula in 64 bits.

Tolerance, element by element, from the sums that each element is made of.  A
tensor-core sum of n products is off by at most (n / 8 + 16) * 2^-23 of the sum
of their absolute values (an addition for each instruction and one for each
warp, truncated); a = silu(g) * u carries g's error (|silu'| <= 1.1), u's, one
fp16 rounding and 2^-18 for the exponential and the quotient; the coefficients
2^-18; the result one fp16 rounding.  Inputs are checked to have no two
experts closer than 1e-5 at the border of the choice, where fp32 logits could
choose otherwise.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -18


def _problem(T, H, I, E, seed=0, sdt=torch.float32):
    from rotalabs_accel_b200 import quantize_weight_per_channel
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, H, generator=g, device="cuda").half()
    router = (torch.randn(E, H, generator=g, device="cuda") * 1.5 / H ** 0.5).half()

    def weight(*shape):
        w = torch.randn(shape[0] * shape[1], shape[2], generator=g, device="cuda") * 0.05
        q, s = quantize_weight_per_channel(w)
        return q.view(shape), s.view(shape[:2]).to(sdt)

    return x, router, *weight(E, I, H), *weight(E, I, H), *weight(E, H, I)


def _reference(x, router, wg, sg, wu, su, wd, sd, k, renorm):
    """(y, tolerance) in 64 bits, and the smallest distance at the border."""
    T, H = x.shape
    E, I = sg.shape
    logits = x.double() @ router.double().t()
    p = torch.softmax(logits, -1)
    top, ids = torch.sort(logits, dim=-1, descending=True, stable=True)
    gap = (top[:, k - 1] - top[:, k]).min().item() if k < E else 1.0
    ids = ids[:, :k]
    c = p.gather(1, ids)
    if renorm:
        c = c / c.sum(-1, keepdim=True)
    y = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(y)
    n1, n2 = (H / 8 + 16) * 2.0 ** -23, (I / 8 + 16) * 2.0 ** -23
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
            da = 1.1 * dg * (up.abs() + du) + silu.abs() * du + a.abs() * (2.0 ** -11 + EPS) + 2.0 ** -25
            part = Wd @ a
            y[t] += c[t, j] * part
            tol[t] += c[t, j] * (Wd.abs() @ (da + n2 * (a.abs() + da)) + EPS * part.abs())
    return y, tol * (1 + 2.0 ** -10) + y.abs() * 2.0 ** -11 + 2.0 ** -25, gap


def _check(p, k, renorm=True):
    import rotalabs_accel_b200 as ra
    y = ra.int8_moe(*p, top_k=k, renormalize=renorm)
    ref, tol, gap = _reference(*p, k, renorm)
    assert gap > 1e-5, "the inputs have a tie: another seed"
    assert y.dtype == torch.float16 and y.shape == ref.shape
    bad = (y.double() - ref).abs() > tol
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} wrong, first at {bad.nonzero()[0].tolist()}"
    return y


# tokens around the 8-token tiles, widths of one 16-element piece up, E around a warp
@pytest.mark.parametrize("T,H,I,E,k", [
    (1, 16, 16, 1, 1), (1, 64, 32, 2, 1), (2, 80, 48, 3, 3), (7, 256, 128, 8, 2), (8, 128, 272, 31, 4),
    (9, 528, 64, 33, 2), (16, 512, 256, 64, 8), (17, 144, 96, 60, 4), (24, 96, 80, 128, 32), (20, 1040, 528, 2, 1), (23, 272, 1296, 3, 2), (31, 272, 48, 255, 3),
    (32, 256, 128, 256, 8), (32, 512, 512, 4, 4), (5, 4096, 1024, 4, 2), (3, 1024, 4112, 5, 1)])
@pytest.mark.parametrize("renorm", [True, False])
def test_sizes(cuda_lib, T, H, I, E, k, renorm):
    from rotalabs_accel_b200 import _capi
    n0 = _capi.launch_count()
    p = _problem(T, H, I, E, seed=T + H + E + 1, sdt=torch.float32 if renorm else torch.float16)
    n0 = _capi.launch_count()
    _check(p, k, renorm)
    assert _capi.launch_count() == n0 + 2


def test_all_tokens_one_expert(cuda_lib):
    """Every token chooses the same expert; then none but the first does."""
    p = list(_problem(32, 256, 128, 16, seed=4))
    p[0] = p[0].abs()
    p[1][5] = p[1][5].abs() + 0.05
    _check(p, 1)
    p[0][1:] = -p[0][1:]
    _check(p, 1)


def test_longer_batches(cuda_lib):
    import rotalabs_accel_b200 as ra
    p = _problem(75, 256, 128, 16, seed=6)
    y = ra.int8_moe(*p, top_k=3)
    for t0 in (0, 32, 64):
        part = ra.int8_moe(p[0][t0:t0 + 32], *p[1:], top_k=3)
        assert torch.equal(y[t0:t0 + 32], part)
    _check([p[0][64:]] + list(p[1:]), 3)
    assert ra.int8_moe(p[0][:0], *p[1:], top_k=3).shape == (0, 256)


def test_ties_take_the_lower_index(cuda_lib):
    import rotalabs_accel_b200 as ra
    x, router, *w = _problem(9, 256, 64, 40, seed=7)
    router[3], router[36], router[7] = router[20], router[20], router[20]
    p = [x, router, *w]
    logits = x.double() @ router.double().t()
    # tokens for which the four equal experts are the largest
    best = (logits.amax(-1) == logits[:, 20]).nonzero().flatten()
    x = torch.cat([x, (router[20].float() * 40).half().unsqueeze(0)])
    logits = x.double() @ router.double().t()
    assert logits[-1].argmax() in (3, 7, 20, 36) and len(best) < 9
    for k, chosen in ((1, [3]), (2, [3, 7]), (3, [3, 7, 20])):
        y = ra.int8_moe(x[-1:], router, *w, top_k=k)
        sub = [t[chosen].contiguous() for t in w]
        want = ra.int8_moe(x[-1:], router[chosen], *sub, top_k=k)
        # (p / (p + p) is exactly 1/2; a third may round either way)
        assert torch.equal(y, want) if k < 3 else torch.allclose(y, want, rtol=2 ** -9, atol=1e-5)


def test_router_of_zeros_and_nan_tokens(cuda_lib):
    import rotalabs_accel_b200 as ra
    x, router, *w = _problem(6, 128, 64, 12, seed=8)
    router.zero_()
    y = ra.int8_moe(x, router, *w, top_k=2)
    sub = [t[:2].contiguous() for t in w]
    assert torch.equal(y, ra.int8_moe(x, router[:2], *sub, top_k=2))
    _, router, *w = _problem(6, 128, 64, 12, seed=9)
    want, tol, gap = _reference(x, router, *w, 2, True)
    assert gap > 1e-5
    for bad in (float("nan"), float("inf"), float("-inf")):
        xb = x.clone()
        xb[2, 17] = bad
        y = ra.int8_moe(xb, router, *w, top_k=2)
        assert torch.isnan(y[2]).all()
        keep = [0, 1, 3, 4, 5]
        assert bool(((y.double() - want).abs() <= tol)[keep].all())   # a bad token spoils no other
    y = ra.int8_moe(torch.zeros_like(x), router, *w, top_k=2)
    assert not y.any()


def test_types_strides_and_refusals(cuda_lib):
    import rotalabs_accel_b200 as ra
    p = _problem(10, 128, 64, 12, seed=10)
    x = p[0]
    y = _check(p, 2)
    wide = torch.zeros(10, 139, device="cuda").half()
    wide[:, 3:131] = x
    assert torch.equal(ra.int8_moe(wide[:, 3:131], *p[1:], top_k=2), y)           # odd stride and start
    assert torch.equal(ra.int8_moe(x.t().contiguous().t(), *p[1:], top_k=2), y)
    assert torch.equal(ra.int8_moe(x.float().view(2, 5, 128), *p[1:], top_k=2), y.view(2, 5, 128))
    r = torch.zeros(12 * 128 + 1, device="cuda").half()
    r[1:] = p[1].flatten()
    assert torch.equal(ra.int8_moe(x, r[1:].view(12, 128), *p[2:], top_k=2), y)
    assert torch.equal(torch.ops.rla.moe(*p, 2, True), y)
    wd_t = p[6].transpose(1, 2).contiguous().transpose(1, 2)
    with pytest.raises(RuntimeError, match="contiguous"):
        ra.int8_moe(*p[:6], wd_t, p[7], top_k=2)
    with pytest.raises(TypeError, match="router_weight"):
        ra.int8_moe(x, p[1].float(), *p[2:], top_k=2)
    with pytest.raises(TypeError, match="one dtype"):
        ra.int8_moe(*p[:7], p[7].half(), top_k=2)
    with pytest.raises(RuntimeError, match="same CUDA device"):
        ra.int8_moe(x, p[1].cpu(), *p[2:], top_k=2)
    with pytest.raises(AssertionError, match="Weight must be INT8"):
        ra.int8_moe(*p[:2], p[2].float(), *p[3:], top_k=2)
    with pytest.raises(AssertionError, match="Scale shape mismatch"):
        ra.int8_moe(*p[:3], p[3][:, :5], *p[4:], top_k=2)
    with pytest.raises(ValueError, match="top_k"):
        ra.int8_moe(*p, top_k=13)
    odd = _problem(3, 72, 40, 4)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        ra.int8_moe(*odd, top_k=2)
    many = _problem(1, 16, 16, 257)
    with pytest.raises(RuntimeError, match="256 experts"):
        ra.int8_moe(*many, top_k=2)
    shifted = torch.zeros(p[2].numel() + 8, dtype=torch.int8, device="cuda")[8:].view(p[2].shape)
    with pytest.raises(RuntimeError, match="16-byte aligned"):
        ra.int8_moe(x, p[1], shifted, *p[3:], top_k=2)


def test_streams_and_graphs(cuda_lib):
    """Another stream, two captured graphs replayed at once on two streams
    (each has its own scratch), results that do not change from run to run."""
    import rotalabs_accel_b200 as ra
    p = _problem(20, 512, 256, 32, seed=11)
    xs = [torch.randn(20, 512, generator=torch.Generator(device="cuda").manual_seed(s), device="cuda").half()
          for s in range(4)]
    want = [ra.int8_moe(x, *p[1:], top_k=4) for x in xs]
    assert all(torch.equal(ra.int8_moe(x, *p[1:], top_k=4), w) for x, w in zip(xs, want))
    graphs, ins, outs = [], [], []
    for _ in range(2):
        ins.append(xs[0].clone())
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            y = ins[-1]
            outs.append([ra.int8_moe(y, *p[1:], top_k=4) for _ in range(3)])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for a, b in ((0, 1), (2, 3), (1, 2)):
        ins[0].copy_(xs[a])
        ins[1].copy_(xs[b])
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[a]) for o in outs[0]) and all(torch.equal(o, want[b]) for o in outs[1])


def test_two_streams_at_once(cuda_lib):
    """Eager calls on two streams at the same time, from two host threads,
    each call with other inputs than the one before it."""
    import threading
    import rotalabs_accel_b200 as ra
    from rotalabs_accel_b200 import _capi
    problems = [_problem(T, 512, 256, E, seed=T) for T, E in ((1, 8), (12, 32), (30, 16), (70, 8))]
    want = [ra.int8_moe(*p, top_k=3) for p in problems]
    torch.cuda.synchronize()
    wrong, streams = [], [torch.cuda.Stream() for _ in range(2)]

    def work(k):
        with torch.cuda.stream(streams[k]):
            for i in range(40):
                j = (i * (k + 1) + k) % 4
                if not torch.equal(ra.int8_moe(*problems[j], top_k=3), want[j]):
                    wrong.append((k, i, j))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and _capi.device_error() == 0
    # back to back without a wait between: every call's scratch is its own
    outs = [ra.int8_moe(*problems[i % 4], top_k=3) for i in range(40)]
    assert all(torch.equal(o, want[i % 4]) for i, o in enumerate(outs))


def test_layers_together(cuda_lib):
    """h, xn = add_rmsnorm; the experts and a shared W8A8 block; next norm."""
    import rotalabs_accel_b200 as ra
    g = torch.Generator(device="cuda").manual_seed(12)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    H, I, E = 256, 160, 8
    m = ra.Int8MoE(H, I, E, 2).cuda()
    m.quantize_weights(rnd(E, H) * 0.1, rnd(E, I, H) * 0.05, rnd(E, I, H) * 0.05, rnd(E, H, I) * 0.05)
    shared = ra.Int8SwiGLU(H, I).cuda()
    shared.quantize_weights(rnd(I, H) * 0.05, rnd(I, H) * 0.05, rnd(H, I) * 0.05)
    w = torch.rand(H, generator=g, device="cuda") + 0.5
    for T in (1, 13, 40):
        x, r = rnd(T, H).half(), rnd(T, H).half()
        xn, h = ra.add_rmsnorm(x, r, w)
        y = m(xn)
        q, s, h2 = ra.add_rmsnorm_int8(x, r, w)
        y2 = shared.forward_w8a8(q, s)
        out, h3 = ra.add_rmsnorm((y.float() + y2.float()).half(), h, w)
        assert torch.equal(h, h2)
        p = [xn[:32], m.router_weight, m.w_gate, m.scale_gate, m.w_up, m.scale_up, m.w_down, m.scale_down]
        assert torch.equal(_check(p, 2), y[:32])
        assert torch.equal(h3, ((y.float() + y2.float()).half().float() + h.float()).half())
        v = h3.double()
        v = v / (v.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        assert bool(((out.double() - v).abs() <= v.abs() * (2.0 ** -11 + EPS) + 2.0 ** -25).all())
