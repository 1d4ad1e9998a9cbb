"""A pre-norm MoE block, trained and then served from 4-bit experts, every
operator this library's:

    layer norm -> router logits -> threshold routing -> gate/up projection ->
    SwiGLU -> down projection -> combine, added to the block's input

Training runs the backward of each and steps all weights with AdamW (8-bit
states, f32 masters, clipped by the global gradient norm).  Serving takes the
same weights with the experts in 4 bits and decodes a few tokens at a time
with fixed-size buffers: no host synchronisation.

    python examples/moe_block.py [--tokens 2048 --width 512 --experts 8 --hidden 256 --steps 60]
"""
import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
et = importlib.import_module("peer-review-agents_amd")


class Block:
    """The weights of one block and its forward and backward pass."""

    def __init__(self, width, experts, hidden, k_target, device, seed):
        g = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape, scale):
            return torch.randn(*shape, generator=g, device=device).mul_(scale).bfloat16()

        self.gain = torch.ones(width, device=device)
        self.bias = torch.zeros(width, device=device)
        self.w_router = randn(experts, width, scale=width ** -0.5)
        self.w_gate_up = randn(experts, 2 * hidden, width, scale=width ** -0.5)
        self.w_down = randn(experts, width, hidden, scale=hidden ** -0.5)
        self.router = et.ExpertThresholdRouter(experts, k_target, device=device)

    @property
    def params(self):
        return [self.gain, self.bias, self.w_router, self.w_gate_up, self.w_down]

    def forward(self, x):
        """The block's output, and what the backward needs."""
        h, mean, rstd = et.layer_norm(x, self.gain, self.bias, stats=True)
        plan = self.router(et.router_logits(h, self.w_router))
        gu = et.expert_gemm(h, self.w_gate_up, plan)
        a = et.swiglu(gu, plan)
        yp = et.expert_gemm(a, self.w_down, plan, gather=False)
        return x + et.combine(yp, plan), (x, h, mean, rstd, plan, gu, a, yp)

    def backward(self, dy, kept):
        """Gradients of the input and of `params`."""
        x, h, mean, rstd, plan, gu, a, yp = kept
        dyp, dgate, dlogits = et.combine_backward(dy, yp, plan, need_dlogits=True)
        da = et.expert_gemm_input_grad(dy, self.w_down, plan, gather=True, row_scale=plan.slot_gate)
        dgu = et.swiglu_backward(gu, da, plan)
        dxp = et.expert_gemm_input_grad(dgu, self.w_gate_up, plan)
        dh = et.dispatch_backward(dxp, plan, router_weight=self.w_router, dgate=dgate)
        # (dy reaches x past the norm too)
        dx, dgain, dbias = et.layer_norm_backward(dh, x, self.gain, mean, rstd, dsum=dy)
        return dx, [dgain, dbias, et.router_weight_grad(dlogits, h),
                    et.expert_gemm_weight_grad(dgu, et.dispatch(h, plan), plan),
                    et.expert_gemm_weight_grad(dyp, a, plan)]


class Server:
    """The block with its experts in 4 bits, for a few tokens at a time."""

    def __init__(self, block, group=64):
        self.block, self.thr = block, block.router.thr
        self.w_gate_up = et.pack_w4(*et.quantize_w4(block.w_gate_up, group=group), group=group, parts=2)
        self.w_down = et.pack_w4(*et.quantize_w4(block.w_down, group=group), group=group)

    def __call__(self, x):
        b = self.block
        h = et.layer_norm(x, b.gain, b.bias)
        logits = et.router_logits(h, b.w_router)
        plan = et.route(logits, self.thr, slot_capacity=logits.numel())
        a = et.expert_gemm_w4(h, self.w_gate_up, plan, epilogue="swiglu")
        return x + et.combine(et.expert_gemm_w4(a, self.w_down, plan, gather=False), plan)


def train(block, teacher, tokens, steps, state="e4m3", seed=0):
    """Fits `block` to `teacher` on fresh random tokens; the losses."""
    device = block.gain.device
    g = torch.Generator(device=device).manual_seed(seed)
    opt = et.AdamW(block.params, lr=3e-3, betas=(0.9, 0.99), weight_decay=0.01, state=state, seed=seed)
    losses = []
    for _ in range(steps):
        x = torch.randn(tokens, block.gain.shape[0], generator=g, device=device).bfloat16()
        y, kept = block.forward(x)
        off = y.float() - teacher.forward(x)[0].float()
        losses.append(off.square().mean())
        _, grads = block.backward((off * (2.0 / off.shape[1])).bfloat16(), kept)
        _, scale = et.grad_norm(grads, max_norm=1.0)
        opt.step(grads, grad_scale=scale)
    return torch.stack(losses).tolist()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 2048), ("width", 512), ("experts", 8), ("hidden", 256), ("k", 2), ("steps", 60)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args(argv)
    make = lambda seed: Block(a.width, a.experts, a.hidden, a.k, "cuda", seed)  # noqa: E731
    teacher, block = make(1), make(2)
    teacher.router.eval()
    losses = train(block, teacher, a.tokens, a.steps)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {a.steps} steps")
    block.router.eval()
    server, errors = Server(block), []
    for tokens in (1, 3, 16):
        x = torch.randn(tokens, a.width, device="cuda").bfloat16()
        want, got = block.forward(x)[0].float(), server(x).float()
        errors.append(((got - want).norm() / (want - x.float()).norm()).item())
        print(f"{tokens} token(s) from 4-bit experts: {errors[-1]:.3f} of the block's own output off")
    return losses, errors


if __name__ == "__main__":
    main()
