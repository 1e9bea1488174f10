"""A mixture-of-experts layer with int8 experts, for decode batches.

Each expert is a SwiGLU block with W8A16 projections (``Int8SwiGLU``; the
reference's ``SwiGLU``, src/rotalabs_accel/kernels/activations.py:140-181, over
``Int8Linear``, kernels/gemm.py:241-336), the weights of all experts stacked.
rotalabs-accel has no mixture-of-experts layer.  On CUDA tensors the whole
layer -- router, choice, gate/up, SwiGLU, down, combination -- is two kernels
(``rla_moe``) for up to 32 tokens; longer batches run 32 tokens at a time and
read their experts each time (256 tokens take eight times as long as 32).
CPU tensors follow the same formulas in torch operations.  For inference: no
gradients flow through ``int8_moe``, on either.
"""

from __future__ import annotations

import torch

from . import _capi
from .gemm import _as_2d_fp16
from .quantization import quantize_weight_per_channel
from .w8a8 import _silu_mul


def int8_moe_torch(x: torch.Tensor, router_weight: torch.Tensor, w_gate: torch.Tensor, scale_gate: torch.Tensor,
                   w_up: torch.Tensor, scale_up: torch.Tensor, w_down: torch.Tensor, scale_down: torch.Tensor,
                   top_k: int, renormalize: bool = True) -> torch.Tensor:
    """The layer in torch operations, any device (``int8_moe`` uses it for CPU
    tensors): fp32, rounded to ``x.dtype`` at the end."""
    H = x.shape[-1]
    x2 = x.reshape(-1, H).float()
    # a choice between two experts is a border: its logits in 64 bits
    p = torch.softmax(x2.double() @ router_weight.double().t(), dim=-1)
    chosen, ids = torch.sort(p, dim=-1, descending=True, stable=True)
    chosen, ids = chosen[:, :top_k], ids[:, :top_k]
    if renormalize:
        chosen = chosen / chosen.sum(dim=-1, keepdim=True)
    y = torch.zeros_like(x2)
    for e in torch.unique(ids).tolist():
        token, place = torch.nonzero(ids == e, as_tuple=True)
        xe = x2[token]
        gate = xe @ w_gate[e].float().t() * scale_gate[e].float()
        up = xe @ w_up[e].float().t() * scale_up[e].float()
        a = _silu_mul(gate, up)
        y[token] += chosen[token, place].float().unsqueeze(1) * (a @ w_down[e].float().t() * scale_down[e].float())
    return y.to(x.dtype).view(x.shape)


def int8_moe(x: torch.Tensor, router_weight: torch.Tensor, w_gate: torch.Tensor, scale_gate: torch.Tensor,
             w_up: torch.Tensor, scale_up: torch.Tensor, w_down: torch.Tensor, scale_down: torch.Tensor,
             top_k: int, renormalize: bool = True) -> torch.Tensor:
    """``y = sum over the top_k experts of c * down(silu(gate(x)) * up(x))``.

    Args:
        x: ``(..., H)`` fp16 (fp32 and bf16 are cast, as by ``int8_gemm``).
        router_weight: fp16 ``(E, H)``; ``p = softmax(x @ router_weight.T)``
            over the experts, the ``top_k`` largest are chosen, ties to the
            lower index.
        w_gate, w_up: int8 ``(E, I, H)``; w_down: int8 ``(E, H, I)``;
            contiguous.
        scale_gate, scale_up ``(E, I)``, scale_down ``(E, H)``: one a channel,
            all fp32 or all fp16.
        renormalize: ``c = p / sum of the chosen p`` (else ``c = p``).

    Sums are fp32; ``silu(gate) * up`` keeps fp32's range and 16 bits (CUDA:
    two bf16 terms; CPU: fp32).

    Returns ``(..., H)``, fp16 for CUDA inputs, ``x.dtype`` for CPU inputs.
    On CUDA: E <= 256, top_k <= 32, H and I multiples of 16.
    """
    if x.is_cuda and x.dim() == 2 and x.dtype == torch.float16:
        # (the per-token case: the extension checks; see w8a8.py)
        try:
            return _capi.torch_ops().moe(x, router_weight, w_gate, scale_gate, w_up, scale_up, w_down, scale_down,
                                         top_k, renormalize)
        except RuntimeError:
            _moe_args(x, router_weight, w_gate, scale_gate, w_up, scale_up, w_down, scale_down, top_k)
            raise
    _moe_args(x, router_weight, w_gate, scale_gate, w_up, scale_up, w_down, scale_down, top_k)
    if x.is_cuda:
        y = _capi.torch_ops().moe(_as_2d_fp16(x, x.shape[-1]), router_weight, w_gate, scale_gate, w_up, scale_up,
                                  w_down, scale_down, top_k, renormalize)
        return y.view(x.shape)
    with torch.no_grad():
        return int8_moe_torch(x, router_weight, w_gate, scale_gate, w_up, scale_up, w_down, scale_down, top_k,
                              renormalize)


def _moe_args(x, router_weight, w_gate, scale_gate, w_up, scale_up, w_down, scale_down, top_k):
    assert w_gate.dtype == torch.int8 and w_up.dtype == torch.int8 and w_down.dtype == torch.int8, \
        "Weight must be INT8"
    E, H = router_weight.shape
    I = w_gate.shape[1]
    assert x.shape[-1] == H, f"Hidden dim mismatch: {x.shape[-1]} vs {H}"
    assert w_gate.shape == (E, I, H) and w_up.shape == (E, I, H) and w_down.shape == (E, H, I), \
        f"Weight shape mismatch: {tuple(w_gate.shape)} / {tuple(w_up.shape)} / {tuple(w_down.shape)}"
    assert scale_gate.shape == (E, I) and scale_up.shape == (E, I) and scale_down.shape == (E, H), \
        f"Scale shape mismatch: {tuple(scale_gate.shape)} / {tuple(scale_up.shape)} / {tuple(scale_down.shape)}"
    if not 1 <= top_k <= E:
        raise ValueError(f"top_k must be in [1, {E}], got {top_k}")


class Int8MoE(torch.nn.Module):
    """Mixture of ``num_experts`` ``Int8SwiGLU`` experts, ``top_k`` of them for
    each token.

    State dict: ``router_weight`` fp16 ``[E, hidden]``; ``w_gate``, ``w_up``
    int8 ``[E, intermediate, hidden]``, ``w_down`` int8 ``[E, hidden,
    intermediate]``; ``scale_gate``, ``scale_up``, ``scale_down`` fp32.
    ``_quantized`` is a plain attribute as in ``Int8Linear``: a module restored
    with ``load_state_dict`` must be re-marked (``mark_quantized()``)."""

    def __init__(self, hidden_size: int, intermediate_size: int, num_experts: int, top_k: int,
                 renormalize: bool = True):
        super().__init__()
        if not 1 <= top_k <= num_experts:
            raise ValueError(f"top_k must be in [1, {num_experts}], got {top_k}")
        self.hidden_size, self.intermediate_size = hidden_size, intermediate_size
        self.num_experts, self.top_k, self.renormalize = num_experts, top_k, renormalize
        E, H, I = num_experts, hidden_size, intermediate_size
        self.register_buffer("router_weight", torch.zeros(E, H, dtype=torch.float16))
        self.register_buffer("w_gate", torch.zeros(E, I, H, dtype=torch.int8))
        self.register_buffer("w_up", torch.zeros(E, I, H, dtype=torch.int8))
        self.register_buffer("w_down", torch.zeros(E, H, I, dtype=torch.int8))
        self.register_buffer("scale_gate", torch.ones(E, I))
        self.register_buffer("scale_up", torch.ones(E, I))
        self.register_buffer("scale_down", torch.ones(E, H))
        self._quantized = False

    def quantize_weights(self, router: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                         w_down: torch.Tensor) -> None:
        """Quantize float expert weights (``[E, out, in]`` each, one scale an
        output channel) and take over the router's (rounded to fp16)."""
        assert router.shape == self.router_weight.shape
        self.router_weight.copy_(router)
        for name, w in (("gate", w_gate), ("up", w_up), ("down", w_down)):
            to, scale = getattr(self, "w_" + name), getattr(self, "scale_" + name)
            assert w.shape == to.shape
            q, s = quantize_weight_per_channel(w.reshape(-1, w.shape[-1]))
            to.copy_(q.view(to.shape))
            scale.copy_(s.view(scale.shape))
        self._quantized = True

    def mark_quantized(self) -> None:
        """Declare the buffers (e.g. from ``load_state_dict``) quantized."""
        self._quantized = True

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self._quantized:
            raise RuntimeError("Weights not quantized. Call quantize_weights() first.")
        return int8_moe(x, self.router_weight, self.w_gate, self.scale_gate, self.w_up, self.scale_up, self.w_down,
                        self.scale_down, self.top_k, self.renormalize)

    def extra_repr(self) -> str:
        return (f"hidden_size={self.hidden_size}, intermediate_size={self.intermediate_size}, "
                f"num_experts={self.num_experts}, top_k={self.top_k}, renormalize={self.renormalize}")
