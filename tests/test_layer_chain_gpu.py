"""Layers of dependent launches in one graph: every kernel starts beside the end
of the one that writes its input, on buffers that the layers share.  Replayed
with new inputs, against the same calls with a wait after each."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1, 7, 20, 32])
def test_chain_of_layers(cuda_lib, T):
    import rotalabs_accel_b200 as ra
    from rotalabs_accel_b200 import _capi
    g = torch.Generator(device="cuda").manual_seed(T)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    H, I, E = 512, 256, 8
    moe = ra.Int8MoE(H, I, E, 2).cuda()
    moe.quantize_weights(rnd(E, H) * 0.1, rnd(E, I, H) * 0.05, rnd(E, I, H) * 0.05, rnd(E, H, I) * 0.05)
    mlp = ra.Int8SwiGLU(H, I).cuda()
    mlp.quantize_weights(rnd(I, H) * 0.05, rnd(I, H) * 0.05, rnd(H, I) * 0.05)
    lin = ra.Int8Linear(H, H).cuda()
    lin.quantize_weights(rnd(H, H) * 0.05)
    w = torch.rand(H, generator=g, device="cuda") + 0.5
    wait = lambda t: t  # noqa: E731

    def layers(x):
        h = x
        for _ in range(4):
            y = wait(lin(wait(ra.rmsnorm(h, w))))
            xn, h = ra.add_rmsnorm(y, h, w)
            y = wait(moe(wait(xn)))
            q, s, h = ra.add_rmsnorm_int8(y, h, w)
            wait(h)
            y = wait(mlp.forward_w8a8(q, s))
            xn, h = ra.add_rmsnorm(y, h, w)
            h = (wait(mlp(wait(xn))).float() + h.float()).half()
        return h

    xs = [rnd(T, H).half() for _ in range(12)]
    x = xs[0].clone()
    layers(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layers(x)

    def wait(t):
        torch.cuda.synchronize()
        return t

    want = [layers(v) for v in xs]
    for _ in range(5):
        for v, y in zip(xs, want):
            x.copy_(v)
            graph.replay()
            assert torch.equal(out, y)
    assert _capi.device_error() == 0
