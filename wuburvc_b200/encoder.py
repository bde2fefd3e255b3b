"""A self-attention encoder in front of the generator, trained with the operators of
``wuburvc_b200.transformer``.

Two forms of layer, over a padded batch x [B, T, width] with lengths:

* ``post`` (LayerNorm after each block, as in the prior encoder, whose relative position terms it leaves out):
      x <- LN(x + attention(x)),  x <- LN(x + feed_forward(x));
* ``gated`` (norms before and after each block, a gate per item from the speaker embedding g):
      r <- r + gate_a(g) * rms(attention(h)),  h = rms(r),  and the same for the feed-forward.

Attention, the fused norms and the 8-bit activation checkpoint are the library's kernels; the matrix
products between them are torch's.  ``python -m wuburvc_b200.encoder`` trains one on synthetic features and
prints the loss (``--help`` for its sizes; the defaults are the prior encoder's width of 192, 2 heads,
feed-forward of 768, 6 layers).
"""
from __future__ import annotations

import argparse

import torch

from . import transformer as tf


class Encoder(torch.nn.Module):
    def __init__(self, width=192, heads=2, hidden=768, layers=6, style="post", speaker=256, kv_heads=None,
                 causal=False, dtype=torch.bfloat16, seed=0):
        super().__init__()
        if style not in ("post", "gated") or width % heads or width // heads % 8:
            raise ValueError("Encoder: style is 'post' or 'gated'; heads divide the width into multiples of 8")
        self.width, self.heads, self.style, self.causal, self.dtype = width, heads, style, causal, dtype
        self.kv_heads = kv_heads or heads
        self.head = width // heads
        self.layers = layers
        g = torch.Generator().manual_seed(seed)

        def matrix(rows, cols):
            return torch.nn.Parameter(torch.randn(rows, cols, generator=g) * cols ** -0.5)

        p = {}
        for i in range(layers):
            p[f"{i}.qkv"] = matrix((heads + 2 * self.kv_heads) * self.head, width)
            p[f"{i}.out"] = matrix(width, width)
            p[f"{i}.w1"], p[f"{i}.w2"] = matrix(hidden, width), matrix(width, hidden)
            p[f"{i}.b1"] = torch.nn.Parameter(torch.zeros(hidden))
            p[f"{i}.b2"] = torch.nn.Parameter(torch.zeros(width))
            for n in ("a", "f"):  # the norms of the attention and of the feed-forward
                p[f"{i}.{n}_norm"] = torch.nn.Parameter(torch.ones(width))
                if style == "post":
                    p[f"{i}.{n}_bias"] = torch.nn.Parameter(torch.zeros(width))
                else:
                    p[f"{i}.{n}_post"] = torch.nn.Parameter(torch.ones(width))
                    p[f"{i}.{n}_gate"] = matrix(width, speaker)
        self.p = torch.nn.ParameterDict({k.replace(".", "_"): v for k, v in p.items()})

    def weight(self, i, name, cast=True):
        w = self.p[f"{i}_{name}"]
        return w.to(self.dtype) if cast else w

    def block(self, i, n, x, f, g):
        """(sum, input of the next block) of block n ("a" or "f") with result f."""
        w = self.weight(i, n + "_norm", cast=False)
        if self.style == "post":
            h = tf.resnorm(x, f, norm="layer", weight=w, bias=self.weight(i, n + "_bias", cast=False), keep_sum=False)[1]
            return h, h
        gate = g.float() @ self.weight(i, n + "_gate", cast=False).T
        return tf.resnorm(x, f, norm="rms", weight=w, post="rms", post_weight=self.weight(i, n + "_post", cast=False),
                          gate=gate)

    def forward(self, x, lens=None, g=None):
        """x [B, T, width], lens int32 [B] or None, g [B, speaker] (gated): [B, T, width]."""
        B, T, _ = x.shape
        H, K, D = self.heads, self.kv_heads, self.head
        x = x.to(self.dtype)
        h = x if self.style == "post" else tf.resnorm(x, torch.zeros_like(x), norm="rms", keep_sum=False)[1]
        for i in range(self.layers):
            qkv = torch.nn.functional.linear(h, self.weight(i, "qkv")).view(B, T, H + 2 * K, D)
            a = tf.attention(qkv[:, :, :H], qkv[:, :, H:H + K], qkv[:, :, H + K:], causal=self.causal, q_lens=lens,
                             k_lens=lens)
            a = torch.nn.functional.linear(a.view(B, T, H * D), self.weight(i, "out"))
            x, h = self.block(i, "a", x, a, g)
            f = tf.feed_forward(h, self.weight(i, "w1"), self.weight(i, "b1"), self.weight(i, "w2"), self.weight(i, "b2"),
                                act="gelu")
            x, h = self.block(i, "f", x, f, g)
        return h


def train(steps=20, batch=16, frames=400, lr=3e-4, style="post", seed=0, report=print, **sizes):
    """Trains an encoder to predict fixed synthetic features; the losses, one a step."""
    model = Encoder(style=style, seed=seed, **sizes).cuda()
    rnd = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(batch, frames, model.width, generator=rnd, device="cuda")
    want = torch.randn(batch, frames, model.width, generator=rnd, device="cuda")
    g = torch.randn(batch, 256, generator=rnd, device="cuda") if style == "gated" else None
    lens = torch.tensor([max(1, frames - (3 * b * frames) // (4 * batch)) for b in range(batch)], dtype=torch.int32,
                        device="cuda")
    live = (torch.arange(frames, device="cuda")[None] < lens[:, None])[..., None]
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for step in range(steps):
        opt.zero_grad(set_to_none=True)
        out = model(x, lens, g)
        loss = ((out.float() - want) * live).square().sum() / (live.sum() * model.width)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        report(f"step {step}: loss {losses[-1]:.5f}")
    tf.ops_sync()
    return losses


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--frames", type=int, default=400)
    ap.add_argument("--width", type=int, default=192)
    ap.add_argument("--heads", type=int, default=2)
    ap.add_argument("--hidden", type=int, default=768)
    ap.add_argument("--layers", type=int, default=6)
    ap.add_argument("--style", choices=("post", "gated"), default="post")
    ap.add_argument("--lr", type=float, default=3e-4)
    a = ap.parse_args()
    train(a.steps, a.batch, a.frames, a.lr, a.style, width=a.width, heads=a.heads, hidden=a.hidden, layers=a.layers)


if __name__ == "__main__":
    main()
