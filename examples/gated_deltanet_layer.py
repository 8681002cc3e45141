"""A Gated DeltaNet decoder layer from this package's operators: a prompt, then
tokens one at a time, and a training step of its feed-forward half.

    python examples/gated_deltanet_layer.py

The layer is pre-norm: norm, input projection, the mixer (front-end, delta rule,
output norm), output projection; the residual's addition with the second norm;
the gated feed-forward block, which adds the residual in its last product. With
`eight_bit`, the first norm's output and the input projection's weight are held
in 8 bits.
"""

import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
dn = importlib.import_module("burn-deltanet_amd")


class Layer:
    """nheads heads of head_k_dim keys and head_v_dim values; bf16 weights."""

    def __init__(self, d_model, nheads, head_k_dim, head_v_dim, hidden, device="cuda",
                 eight_bit=False, seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, cols):
            return (torch.randn(rows, cols, generator=gen, device=device)
                    * rows ** -0.5).to(torch.bfloat16)

        conv_dim = nheads * (2 * head_k_dim + head_v_dim)
        conv = dn.ShortConv(torch.randn(conv_dim, 4, generator=gen, device=device) * 0.5)
        self.proj = dn.QkvProjection(nheads, head_k_dim, head_v_dim, conv=conv, has_gate=True,
                                     extra_channels=nheads)
        self.in_proj = matrix(d_model, self.proj.d_in_proj())
        self.in_proj_8bit = dn.quantize_rows(self.in_proj.t()) if eight_bit else None
        self.out_proj = matrix(nheads * head_v_dim, d_model)
        self.out_norm = dn.OutNorm(torch.ones(head_v_dim, device=device))
        self.norm1 = torch.ones(d_model, dtype=torch.bfloat16, device=device)
        self.norm2 = torch.ones(d_model, dtype=torch.bfloat16, device=device)
        self.w_gate, self.w_up = matrix(d_model, hidden), matrix(d_model, hidden)
        self.w_down = matrix(hidden, d_model)
        self.log_a = torch.zeros(nheads, device=device)
        self.nheads, self.head_k_dim, self.head_v_dim = nheads, head_k_dim, head_v_dim

    def cache(self, batch, device="cuda"):
        """The convolution's window and the delta rule's state before any token."""
        return (self.proj.zero_conv_window(batch, device, torch.bfloat16),
                torch.zeros(batch, self.nheads, self.head_k_dim, self.head_v_dim, device=device))

    def _project(self, x):
        if self.in_proj_8bit is None:
            h, _ = dn.add_rms_norm(x, None, self.norm1)
            return dn.linear(h, self.in_proj)
        rows8, _ = dn.add_rms_norm_8bit(x, None, self.norm1)
        return dn.linear_8bit(rows8, self.in_proj_8bit).reshape(*x.shape[:-1], -1)

    def _log_decay(self, extra):
        """The forget gate of the projection's last columns, one a head."""
        return (-torch.exp(self.log_a) * torch.nn.functional.softplus(extra.float())).unsqueeze(-1)

    def _rest(self, x, mixed):
        """Output projection, residual and second norm, feed-forward."""
        h, total = dn.add_rms_norm(dn.linear(mixed, self.out_proj), x, self.norm2)
        return dn.gated_ffn(h, self.w_gate, self.w_up, self.w_down, dn.Activation.SILU, total)

    def prompt(self, x, cache):
        """x [batch, sequence, d_model] and the cache before it: (y, the cache after)."""
        window, state = cache
        qkv, window = self.proj.forward_projected(self._project(x), window)
        y, state = dn.DeltaInput(qkv.q_bshk, qkv.k_bShk, qkv.v_bShv, qkv.erase_bShK,
                                 qkv.write_bShV, self._log_decay(qkv.extra_bsx), state).run()
        mixed = self.out_norm.forward(y, qkv.gate_bshv).flatten(2)
        return self._rest(x, mixed), (window, state)

    def token(self, x, cache):
        """x [batch, d_model], the cache updated where it is: y [batch, d_model]."""
        window, state = cache
        projected = self._project(x)
        extra = projected[:, -self.nheads:]
        out, window, state = dn.block_step(self.proj, self.out_norm, projected, window,
                                           self._log_decay(extra), state, in_place=True)
        return self._rest(x, out.flatten(1)), (window, state)

    def feed_forward_loss(self, x, target):
        """The squared error of the feed-forward half, for training its weights."""
        h, total = dn.add_rms_norm(x, None, self.norm2)
        y = dn.gated_ffn(h, self.w_gate, self.w_up, self.w_down, dn.Activation.SILU, total)
        return (y.float() - target.float()).square().mean()


def main(d_model=256, nheads=4, head_k_dim=64, head_v_dim=64, hidden=683, batch=2, sequence=96,
         tokens=8):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(batch, sequence + tokens, d_model, generator=gen, device="cuda").bfloat16()
    worst = {}
    for eight_bit in (False, True):
        layer = Layer(d_model, nheads, head_k_dim, head_v_dim, hidden, eight_bit=eight_bit)
        whole, _ = layer.prompt(x, layer.cache(batch))
        _, cache = layer.prompt(x[:, :sequence], layer.cache(batch))
        off = 0.0
        for t in range(sequence, sequence + tokens):
            y, cache = layer.token(x[:, t].contiguous(), cache)
            off = max(off, ((y - whole[:, t]).float().norm() / whole[:, t].float().norm()).item())
        worst["8-bit" if eight_bit else "bf16"] = off
        print(f"{'8-bit' if eight_bit else 'bf16'} input projection: tokens one at a time differ "
              f"from the prompt by {off:.2e}")
    layer = Layer(d_model, nheads, head_k_dim, head_v_dim, hidden)
    target = torch.randn(x.shape, generator=gen, device="cuda").bfloat16()
    weights = [layer.w_gate, layer.w_up, layer.w_down]
    for w in weights:
        w.requires_grad_(True)
    losses = []
    for _ in range(5):
        loss = layer.feed_forward_loss(x, target)
        grads = torch.autograd.grad(loss, weights)
        with torch.no_grad():
            for w, g in zip(weights, grads):
                w -= (4.0 * g.float()).to(w.dtype)
        losses.append(loss.item())
    print("feed-forward training: " + " ".join(f"{v:.4f}" for v in losses))
    return worst, losses


if __name__ == "__main__":
    main()
