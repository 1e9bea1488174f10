"""The choice of the experts where the logits are sums of very different or very
close values: the fp32 sums that a tensor-core instruction is added to are at
most 128 products (8 instructions) long, and joined without loss.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _experts(E, H, I, g):
    def weight(rows, cols):
        return (torch.randint(-127, 128, (E, rows, cols), generator=g, device="cuda", dtype=torch.int8),
                torch.full((E, rows), 0.02 / cols ** 0.5, device="cuda"))

    return (*weight(I, H), *weight(I, H), *weight(H, I))


def _only(w, ids):
    return [t[ids].contiguous() for t in w]


# (more experts: longer sums of a warp; more tokens: fewer warps)
@pytest.mark.parametrize("T", [1, 9, 32])
@pytest.mark.parametrize("E", [16, 64, 128, 256])
def test_small_products_after_a_large_one(cuda_lib, T, E):
    """Expert a's logit is 1024 and products of 2^-18 in later instructions of
    the same sum: 16 of them are half of the last bit of 1024, so that a long
    fp32 sum drops them all.  Expert b's is 1024 + 2^-10, which is less."""
    import rotalabs_accel_b200 as ra
    g = torch.Generator(device="cuda").manual_seed(E)
    H, I = 4096, 16
    for a, b in ((5, 9), (9, 5), (E - 1, 0)):
        x = torch.zeros(T, H, device="cuda")
        router = torch.zeros(E, H, device="cuda")
        x[:, 0], router[a, 0], router[b, 0] = 32.0, 32.0, 32.0
        x[:, 128:512] = 2.0 ** -9
        router[a, 128:512] = 2.0 ** -9
        x[:, 3000], router[b, 3000] = 2.0 ** -5, 2.0 ** -5
        x, router = x.half(), router.half()
        logits = x.double() @ router.double().t()
        assert bool((logits[:, a] == 1024 + 384 * 2.0 ** -18).all()) and bool((logits[:, b] == 1024 + 2.0 ** -10).all())
        w = _experts(E, H, I, g)
        y = ra.int8_moe(x, router, *w, top_k=1)
        assert torch.equal(y, ra.int8_moe(x, router[[a]], *_only(w, [a]), top_k=1)), (a, b)
        assert not torch.equal(y, ra.int8_moe(x, router[[b]], *_only(w, [b]), top_k=1))


@pytest.mark.parametrize("E", [128, 256])
def test_close_logits(cuda_lib, E):
    """Two experts a token whose logits differ by little more than their sums'
    error: 8 additions to each sum of 128 products, each off by 2^-23 of it at most
    (and the products of an instruction by as much of the largest of them)."""
    import rotalabs_accel_b200 as ra
    H, I, T = 4096, 16, 32
    g = torch.Generator(device="cuda").manual_seed(E + 1)
    x = torch.randn(T, H, generator=g, device="cuda").half()
    small = torch.arange(3, H, 7, device="cuda")[:64]        # fine adjustments: products of 2^-17, 2^-20 and 2^-23
    x[:, small[:32]], x[:, small[32:]] = 2.0 ** -5, 2.0 ** -8
    router = (torch.randn(E, H, generator=g, device="cuda") * 1.5 / H ** 0.5).half()
    pairs = torch.randperm(E, generator=g, device="cuda")[:2 * T].view(T, 2)
    want = []
    for t in range(T):
        i, j = pairs[t].tolist()
        for e in (i, j):                                     # the token's largest logits, about 8
            r = router[e].float()
            r += x[t].float() * ((8 - r @ x[t].float()) / x[t].float().pow(2).sum())
            router[e] = r.half()
        router[[i, j]] = router[[i, j]].index_fill(1, small, 0.0)
        # bounds of the sums' errors, from their own 64-bit partial sums
        limit = 0.0
        for e in (i, j):
            p = (x[t].double() * router[e].double()).view(H // 128, 8, 16)
            limit += ((p.sum(-1).cumsum(-1).abs() + p.abs().amax(-1)).sum() * 2.0 ** -23).item()
        gap = 1.25 * limit * (1 if t % 2 else -1)             # l_i - l_j
        d = lambda: gap - (x[t].double() @ (router[i].double() - router[j].double())).item()  # noqa: E731
        for cols, unit, step in ((small[:16], 2.0 ** -12, 2.0 ** -17), (small[16:32], 2.0 ** -15, 2.0 ** -20),
                                 (small[32:48], 2.0 ** -15, 2.0 ** -23)):
            n = int(round(d() / step))
            per = max(-2000, min(2000, n // len(cols)))
            router[i, cols] = per * unit
            router[i, cols[0]] = max(-2000, min(2000, per + n - per * len(cols))) * unit
        assert abs(d()) < 0.1 * limit, (d(), limit)
        want.append(i if gap > 0 else j)
    logits = x.double() @ router.double().t()
    assert logits.argmax(-1).tolist() == want
    w = _experts(E, H, I, g)
    y = ra.int8_moe(x, router, *w, top_k=1)
    other = 0
    for t in range(T):
        i, j = pairs[t].tolist()
        right = ra.int8_moe(x[t:t + 1], router[[want[t]]], *_only(w, [want[t]]), top_k=1)
        wrong = ra.int8_moe(x[t:t + 1], router[[i + j - want[t]]], *_only(w, [i + j - want[t]]), top_k=1)
        close = lambda v: (y[t].float() - v[0].float()).norm() < 1e-2 * v.float().norm()  # noqa: E731
        assert not torch.equal(right, wrong)
        other += not bool(close(right))
    assert other == 0, f"{other} of {T} tokens took the other expert"
