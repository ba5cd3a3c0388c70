"""A decoder layer's feed-forward halves on microscaled weights, one after the
other: a dense one with 8-bit activations, then a mixture of experts.

    python examples/mxfp4_layer.py [--tokens T] [--hidden H] [--inter I] [--experts E] [--top-k K]

    h, a      residual addition, norm, mxfp8 rows           ops.rms_norm_quantize
    gate, up  a @ W^T, mxfp8 times mxfp4                    ops.mx_matmul
    act       silu(gate) * up, to mxfp8                     ops.quantize
    h         h + act @ W_down^T                            ops.mx_matmul
    experts   the same with each token's top-k experts      ops.mx_matmul / ops.gather_qmm, grouped

Prints the difference from the same layer in fp32 on the dequantised weights,
and the time of a pass.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from mlxturbo_b200 import nn, ops  # noqa: E402

MX = dict(group_size=32, bits=4, mode="mxfp4")


def bank(experts: int, n: int, k: int) -> nn.QuantizedSwitchLinear:
    layer = nn.QuantizedSwitchLinear(k, n, experts, device="cuda", **MX)
    w, s = ops.quantize(torch.randn(experts, n, k, device="cuda") * 0.02, 32, 4, mode="mxfp4")
    layer.weight.copy_(w)
    layer.scales.copy_(s)
    return layer


class Layer(torch.nn.Module):
    def __init__(self, hidden: int, inter: int, experts: int, expert_inter: int, top_k: int):
        super().__init__()
        linear = lambda n, k: nn.QuantizedLinear.from_float(  # noqa: E731
            torch.randn(n, k, device="cuda") * 0.02, **MX)
        self.norm1 = nn.RMSNormQuantized(hidden, device="cuda")
        self.norm2 = nn.RMSNormQuantized(hidden, device="cuda")
        self.gate, self.up, self.down = linear(inter, hidden), linear(inter, hidden), linear(hidden, inter)
        self.router = torch.randn(experts, hidden, device="cuda", dtype=torch.bfloat16) * 0.05
        self.gate_bank, self.up_bank = bank(experts, expert_inter, hidden), bank(experts, expert_inter, hidden)
        self.down_bank = bank(experts, hidden, expert_inter)
        self.top_k = top_k

    def forward(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """(output of the experts, residual stream) of tokens [T, hidden]."""
        aq, a_scales, h = self.norm1(x, residual)
        act = nn.swiglu(self.up.forward_mx(aq, a_scales), self.gate.forward_mx(aq, a_scales))
        y = self.down.forward_mx(*ops.quantize(act, 32, 8, mode="mxfp8"))
        aq, a_scales, h = self.norm2(y, h)
        a = ops.dequantize(aq, a_scales, None, 32, 8, mode="mxfp8")
        weights, ids = (a @ self.router.T).float().softmax(-1).topk(self.top_k)
        ids = ids.to(torch.int32).reshape(-1)
        tokens = torch.arange(x.shape[0], device="cuda", dtype=torch.int32).repeat_interleave(self.top_k)
        # gate and up from the 8-bit rows, down from 16-bit ones
        route = dict(lhs_indices=tokens, rhs_indices=ids)
        gate = ops.mx_matmul(aq, a_scales, self.gate_bank.weight, self.gate_bank.scales, **route)
        up = ops.mx_matmul(aq, a_scales, self.up_bank.weight, self.up_bank.scales, **route)
        out = self.down_bank(nn.swiglu(up, gate).unsqueeze(1), ids)
        return (out.reshape(*weights.shape, -1) * weights.unsqueeze(-1).to(out.dtype)).sum(1), h

    def reference(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The same in fp32, on the dequantised weights and with the activations' 8-bit rounding kept."""
        deq = lambda m: ops.dequantize(m.weight, m.scales, None, 32, 4, mode="mxfp4", dtype=torch.float32)  # noqa: E731

        def to8(v):
            return ops.dequantize(*ops.quantize(v, 32, 8, mode="mxfp8"), None, 32, 8, mode="mxfp8", dtype=torch.float32)

        def norm(v, m):
            return to8(v * torch.rsqrt(v.square().mean(-1, keepdim=True) + m.eps) * m.weight.float())

        h = x.float() + residual.float()
        a = norm(h, self.norm1)
        act = nn.swiglu((a @ deq(self.up).T).bfloat16(), (a @ deq(self.gate).T).bfloat16())
        h = h.bfloat16().float() + (to8(act) @ deq(self.down).T).bfloat16().float()
        a = norm(h, self.norm2)
        weights, ids = (a.bfloat16() @ self.router.T).float().softmax(-1).topk(self.top_k)
        out = torch.zeros_like(h)
        g, u, d = deq(self.gate_bank), deq(self.up_bank), deq(self.down_bank)
        for e in ids.unique().tolist():
            t, k = (ids == e).nonzero(as_tuple=True)
            act = nn.swiglu((a[t] @ u[e].T).bfloat16(), (a[t] @ g[e].T).bfloat16())
            out.index_add_(0, t, (act.float() @ d[e].T) * weights[t, k, None])
        return out, h


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--inter", type=int, default=5120)
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--expert-inter", type=int, default=512)
    ap.add_argument("--top-k", type=int, default=10)
    args = ap.parse_args()
    torch.manual_seed(0)
    torch.backends.cuda.matmul.allow_tf32 = False
    layer = Layer(args.hidden, args.inter, args.experts, args.expert_inter, args.top_k)
    x = torch.randn(args.tokens, args.hidden, device="cuda", dtype=torch.bfloat16)
    residual = torch.randn(args.tokens, args.hidden, device="cuda", dtype=torch.bfloat16)
    y, h = layer(x, residual)
    y_ref, h_ref = layer.reference(x, residual)
    for name, a, b in (("residual stream", h, h_ref), ("experts' output", y, y_ref)):
        print(f"{name}: relative difference {((a.float() - b).norm() / b.norm()).item():.2e}")
    for _ in range(3):
        layer(x, residual)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(20):
        layer(x, residual)
    end.record()
    torch.cuda.synchronize()
    print(f"{args.tokens} tokens: {start.elapsed_time(end) / 20 * 1e3:.0f} us a pass")
    return 0


if __name__ == "__main__":
    sys.exit(main())
