"""A small decoder from this package's operators whose layers mix tokens in turn by
softmax attention and by the delta rule: whole prompts, tokens one at a time over
caches, and a training step.

    python examples/hybrid_decoder.py

Ids go through the embedding into the residual stream. Each layer is a mixer and a
gated feed-forward block; each of them ends in block_norm: norm of its output, a gate a
channel, the scaled residual and the norm before what follows. The last norm's output
goes through a linear projection to the logits.
"""

import importlib
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
dn = importlib.import_module("burn-deltanet_amd")


class Decoder:
    """`mixers` names each layer's mixer: "attention" or "delta"."""

    def __init__(self, vocab, d_model, nheads, kv_heads, head_dim, hidden,
                 mixers=("attention", "delta"), dtype=torch.bfloat16, device="cuda", seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def matrix(rows, cols, scale=None):
            return (torch.randn(rows, cols, generator=gen, device=device)
                    * (rows ** -0.5 if scale is None else scale)).to(dtype)

        def ones(value=1.0):
            return torch.full((d_model,), value, dtype=dtype, device=device)

        self.nheads, self.kv_heads, self.head_dim = nheads, kv_heads, head_dim
        self.scale, self.residual_scale = d_model ** 0.5, 0.9
        self.table = matrix(vocab, d_model, d_model ** -0.5)
        self.head, self.first_norm = matrix(d_model, vocab), ones()
        self.mixers, self.layers = mixers, []
        for kind in mixers:
            kv = kv_heads if kind == "attention" else nheads
            # The delta rule's write strength, one a head, beside q, k and v.
            extra = nheads if kind == "delta" else 0
            self.layers.append({
                "qkv": matrix(d_model, (nheads + 2 * kv) * head_dim + extra),
                "out": matrix(nheads * head_dim, d_model),
                "mix_post": ones(), "mix_gate": ones(0.5), "mix_pre": ones(),
                "w_gate": matrix(d_model, hidden), "w_up": matrix(d_model, hidden),
                "w_down": matrix(hidden, d_model),
                "ffn_post": ones(), "ffn_gate": ones(0.5), "ffn_pre": ones()})

    def weights(self):
        return [self.table, self.head, self.first_norm] + [w for l in self.layers
                                                           for w in l.values()]

    def _split(self, kind, projected):
        """q, k, v [..., heads, head_dim], and for the delta rule its write strength."""
        n, d = self.nheads, self.head_dim
        kv = self.kv_heads if kind == "attention" else n
        q, k, v, extra = projected.split(
            [n * d, kv * d, kv * d, projected.shape[-1] - (n + 2 * kv) * d], -1)
        q, k, v = q.unflatten(-1, (n, d)), k.unflatten(-1, (kv, d)), v.unflatten(-1, (kv, d))
        if kind == "attention":
            return q, k, v, None
        unit = lambda t: torch.nn.functional.normalize(t.float(), dim=-1).to(t.dtype)
        return (unit(q), unit(k), v.contiguous(),
                torch.sigmoid(extra.float()).unsqueeze(-1).contiguous())

    def _rest(self, layer, mixed, stream):
        y = dn.linear(mixed.flatten(-2), layer["out"])
        h, stream = dn.block_norm(y, stream, layer["mix_pre"], layer["mix_post"],
                                  layer["mix_gate"], self.residual_scale)
        y = dn.gated_ffn(h, layer["w_gate"], layer["w_up"], layer["w_down"])
        return dn.block_norm(y, stream, layer["ffn_pre"], layer["ffn_post"], layer["ffn_gate"],
                             self.residual_scale)

    def _state(self, batch):
        return torch.zeros(batch, self.nheads, self.head_dim, self.head_dim,
                           device=self.table.device)

    def prompt(self, tokens):
        """Logits [batch, sequence, vocab] of ids [batch, sequence]."""
        stream = dn.embedding(tokens, self.table, self.scale)
        h, stream = dn.add_rms_norm(stream, None, self.first_norm)
        for kind, layer in zip(self.mixers, self.layers):
            q, k, v, write = self._split(kind, dn.linear(h, layer["qkv"]))
            if kind == "attention":
                mixed = dn.attention(q, k, v)
            else:
                mixed, _ = dn.DeltaInput(q, k, v, write, write, None,
                                         self._state(tokens.shape[0])).run()
            h, stream = self._rest(layer, mixed, stream)
        return dn.linear(h, self.head)

    def caches(self, batch, most):
        """For `most` tokens of each sequence: keys and values, or the delta rule's state."""
        new = lambda: torch.empty(batch, most, self.kv_heads, self.head_dim,
                                  dtype=self.table.dtype, device=self.table.device)
        return [(new(), new()) if kind == "attention" else self._state(batch)
                for kind in self.mixers]

    def token(self, tokens, at, caches):
        """Logits [batch, vocab] of one id a sequence, at position `at`; the caches are
        updated where they are."""
        batch, dev = tokens.shape[0], tokens.device
        stream = dn.embedding(tokens, self.table, self.scale)
        h, stream = dn.add_rms_norm(stream, None, self.first_norm)
        for i, (kind, layer) in enumerate(zip(self.mixers, self.layers)):
            q, k, v, write = self._split(kind, dn.linear(h, layer["qkv"]))
            if kind == "attention":
                keys, values = caches[i]
                keys[:, at], values[:, at] = k, v
                most = keys.shape[1]
                starts = torch.arange(batch, dtype=torch.int32, device=dev) * most
                spans = dn.KeySpans(starts, torch.full_like(starts, at + 1))
                mixed = dn.attention(q.unsqueeze(1), keys, values, None, spans).squeeze(1)
            else:
                mixed, _ = dn.delta_step(q, k, v, write, write, None, caches[i],
                                         self.head_dim ** -0.5, in_place=True)
                mixed = mixed.to(h.dtype)
            h, stream = self._rest(layer, mixed, stream)
        return dn.linear(h, self.head)


def loss_of(decoder, tokens):
    """The mean cross-entropy of each next id."""
    logits = decoder.prompt(tokens[:, :-1]).float()
    return torch.nn.functional.cross_entropy(logits.flatten(0, 1), tokens[:, 1:].flatten())


def main(vocab=300, d_model=128, nheads=4, kv_heads=2, head_dim=64, hidden=341, batch=2,
         sequence=70):
    gen = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, vocab, (batch, sequence), generator=gen, device="cuda")
    decoder = Decoder(vocab, d_model, nheads, kv_heads, head_dim, hidden)
    whole = decoder.prompt(tokens)
    caches, off = decoder.caches(batch, sequence), 0.0
    for t in range(sequence):
        logits = decoder.token(tokens[:, t].contiguous(), t, caches)
        off = max(off, ((logits - whole[:, t]).float().norm() / whole[:, t].float().norm()).item())
    print(f"tokens one at a time differ from the prompt by {off:.2e}")
    weights = decoder.weights()
    for w in weights:
        w.requires_grad_(True)
    losses = []
    for _ in range(3):
        loss = loss_of(decoder, tokens)
        grads = torch.autograd.grad(loss, weights)
        with torch.no_grad():
            for w, g in zip(weights, grads):
                w -= 0.2 * g
        losses.append(loss.item())
    print("training: " + " ".join(f"{v:.4f}" for v in losses))
    return off, losses


if __name__ == "__main__":
    main()
