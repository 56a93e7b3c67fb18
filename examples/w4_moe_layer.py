"""A mixture-of-experts layer with 4-bit weights, from hidden states to hidden states.

  logits  = x . W_gate^T                                     (plain product: the gate is small and stays in bf16)
  picks   = route_experts(logits): 6 of 64 experts           (softmax scores, renormalised)
  routed  = experts_w4(x, picks): both products of the picked experts, SwiGLU between them, weighted sum
  shared  = linear_w4 up, SwiGLU, linear_w4 down             (one expert for every token)
  output  = routed + shared

and one training step of the gate through route_experts' gradient. Prints how far the layer is from a 32-bit
computation of the same weights and how long a decode step takes. Needs a GPU:

  python examples/w4_moe_layer.py [tokens]
"""
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
moe = importlib.import_module("15642_moe_b200")


def quantize(w: torch.Tensor, group: int = 128):
    """Symmetric 4-bit codes of w [..., N, K]: one scale per `group` columns, so that the largest is 7."""
    g = w.unflatten(-1, (-1, group))
    scale = (g.abs().amax(-1) / 7).clamp_min(1e-8).to(torch.bfloat16)
    q = (g / scale.float().unsqueeze(-1)).round().clamp(-8, 7).add(8).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), scale


def dequantize(codes: torch.Tensor, scale: torch.Tensor, group: int = 128) -> torch.Tensor:
    q = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8
    return q * scale.float().repeat_interleave(group, -1)


class W4MoELayer:
    def __init__(self, H=1024, I=512, E=64, top_k=6, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: 0.03 * torch.randn(s, generator=g, device="cuda")  # noqa: E731
        self.top_k = top_k
        self.gate = rand(E, H).to(torch.bfloat16)
        self.w13, self.s13 = quantize(rand(E, 2 * I, H))
        self.w2, self.s2 = quantize(rand(E, H, I))
        self.shared13, self.shared_s13 = quantize(rand(2 * I, H))
        self.shared2, self.shared_s2 = quantize(rand(H, I))

    def forward(self, x: torch.Tensor):
        idx, w = moe.route_experts(x @ self.gate.T, self.top_k)
        routed = moe.experts_w4(x, idx, w, self.w13, self.s13, self.w2, self.s2)
        u1, u2 = moe.linear_w4(x, self.shared13, self.shared_s13).chunk(2, -1)
        shared = moe.linear_w4(u1 * torch.nn.functional.silu(u2), self.shared2, self.shared_s2)
        return routed + shared, idx, w

    def plain(self, x: torch.Tensor, idx: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        """The same weights and picks in 32 bits."""
        def expert(rows, a, b):
            u1, u2 = (rows @ a.T).chunk(2, -1)
            return (u1 * torch.nn.functional.silu(u2)) @ b.T
        x = x.float()
        out = expert(x, dequantize(self.shared13, self.shared_s13), dequantize(self.shared2, self.shared_s2))
        for e in range(self.w13.shape[0]):
            t, j = torch.nonzero(idx == e, as_tuple=True)
            if t.numel():
                y = expert(x[t], dequantize(self.w13[e], self.s13[e]), dequantize(self.w2[e], self.s2[e]))
                out.index_add_(0, t, w[t, j, None] * y)
        return out


def gate_step(layer: W4MoELayer, x: torch.Tensor, lr: float = 0.5):
    """One gradient step of the gate that raises the weight of every token's best expert; (before, after)."""
    gate = layer.gate.float().requires_grad_()
    best = lambda g: moe.route_experts(x.float() @ g.T, layer.top_k)[1][:, 0].mean()  # noqa: E731
    before = best(gate)
    before.backward()
    with torch.no_grad():
        after = best(gate + lr * gate.grad)
    return float(before.detach()), float(after)


def main(tokens: int = 16) -> float:
    layer = W4MoELayer()
    x = torch.randn((tokens, 1024), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    out, idx, w = layer.forward(x)
    ref = layer.plain(x, idx, w)
    off = float((out.float() - ref).norm() / ref.norm())
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for _ in range(3):
        layer.forward(x)
    start.record()
    for _ in range(50):
        layer.forward(x)
    end.record()
    torch.cuda.synchronize()
    before, after = gate_step(layer, x)
    print(f"{tokens} tokens: relative difference from 32 bits {off:.1e}, {start.elapsed_time(end) * 20:.0f} us a layer; "
          f"mean weight of the best expert {before:.4f} -> {after:.4f} after one step of the gate")
    assert after > before
    return off


if __name__ == "__main__":
    main(int(sys.argv[1]) if len(sys.argv) > 1 else 16)
