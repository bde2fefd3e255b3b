"""The encoder that runs attention, the fused norms and the 8-bit feed-forward together
(wuburvc_b200/encoder.py), against the same network in float64 with torch's autograd.

Tolerances, relative L2: a bf16 rounding is 2^-9 / sqrt(3) = 1.1e-3 of a value, and a layer makes about ten
of them in a chain (7 x 1.1e-3 with errors adding in quadrature over two layers and back: below 2e-2); the
8-bit form of a hidden value is off by max / 254 / sqrt(3), about 0.7 % of its standard deviation, which
enters the feed-forward's gradients alone.  3e-2 for the result and 5e-2 for each gradient hold both, and a
wrong or missing term in any of the operators is of order 1."""
import pytest
import torch

from wuburvc_b200 import encoder
from wuburvc_b200 import transformer as tf

pytestmark = pytest.mark.gpu


def norm(v, kind):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-5)


def reference(model, p, x, lens, g):
    B, T, _ = x.shape
    H, K, D = model.heads, model.kv_heads, model.head
    post = model.style == "post"
    see = torch.arange(T, device=x.device)[None, None, None] < lens.view(-1, 1, 1, 1)
    if model.causal:
        see = see & torch.ones(T, T, dtype=torch.bool, device=x.device).tril()

    def block(i, n, x, f):
        w = p[f"{i}_{n}_norm"]
        if post:
            h = norm(x + f, "layer") * w + p[f"{i}_{n}_bias"]
            return h, h
        gate = (g @ p[f"{i}_{n}_gate"].T)[:, None]
        r = x + gate * norm(f, "rms") * p[f"{i}_{n}_post"]
        return r, norm(r, "rms") * w

    h = x if post else norm(x, "rms")
    for i in range(model.layers):
        q, k, v = (h @ p[f"{i}_qkv"].T).view(B, T, H + 2 * K, D).transpose(1, 2).split((H, K, K), 1)
        k, v = (t.repeat_interleave(H // K, 1) for t in (k, v))
        s = (q @ k.transpose(2, 3)) * D ** -0.5
        a = torch.softmax(s.masked_fill(~see, -1e30), -1) @ v
        a = a * (torch.arange(T, device=x.device)[None, None, :, None] < lens.view(-1, 1, 1, 1))
        x, h = block(i, "a", x, a.transpose(1, 2).reshape(B, T, H * D) @ p[f"{i}_out"].T)
        u = h @ p[f"{i}_w1"].T + p[f"{i}_b1"]
        x, h = block(i, "f", x, torch.nn.functional.gelu(u) @ p[f"{i}_w2"].T + p[f"{i}_b2"])
    return h


@pytest.mark.parametrize("style,kv_heads,causal", [("post", 2, False), ("gated", 2, True), ("gated", 1, False)])
def test_result_and_gradients(style, kv_heads, causal):
    model = encoder.Encoder(width=96, heads=2, hidden=200, layers=2, style=style, kv_heads=kv_heads, causal=causal,
                            seed=1).cuda()
    rnd = torch.Generator(device="cuda").manual_seed(3)
    B, T = 3, 150
    x = torch.randn(B, T, 96, generator=rnd, device="cuda").bfloat16()
    w = torch.randn(B, T, 96, generator=rnd, device="cuda")
    g = torch.randn(B, 256, generator=rnd, device="cuda")
    lens = torch.tensor([150, 129, 7], dtype=torch.int32, device="cuda")
    live = (torch.arange(T, device="cuda")[None] < lens[:, None])[..., None]
    with torch.no_grad():  # the float64 network starts from the weights that the products see
        for n, v in model.p.items():
            if v.dim() == 2 and "gate" not in n:
                v.copy_(v.bfloat16())
    out = model(x, lens, g)
    (out.float() * w * live).sum().backward()
    p = {n: v.detach().double().requires_grad_(True) for n, v in model.p.items()}
    want = reference(model, p, x.double(), lens, g.double())
    (want * w * live).sum().backward()
    off = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert off(out.detach() * live, want.detach() * live) < 3e-2
    for n, v in model.p.items():
        assert off(v.grad, p[n].grad) < 5e-2, n


def test_training_lowers_the_loss():
    for style in ("post", "gated"):
        losses = encoder.train(steps=12, batch=4, frames=60, lr=1e-3, style=style, width=64, heads=2, hidden=128, layers=2,
                               report=lambda line: None)
        assert losses[-1] < 0.97 * losses[0] and all(x == x for x in losses)


def test_second_derivatives_raise():
    """Of the example's operators together: a gradient penalty is refused, not left out."""
    model = encoder.Encoder(width=64, heads=2, hidden=128, layers=1, style="gated").cuda()
    x = torch.randn(1, 20, 64, device="cuda").bfloat16().requires_grad_(True)
    out = model(x, torch.tensor([20], dtype=torch.int32, device="cuda"), torch.randn(1, 256, device="cuda"))
    g, = torch.autograd.grad(out.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        (g.float().square().sum() + x.float().square().sum()).backward()


def test_autocast():
    """float32 leaves under autocast: the bits that the same calls give on leaves cast by hand, and gradients that are
    those rounded to no more than the leaves' type."""
    rnd = torch.Generator(device="cuda").manual_seed(5)
    leaf = lambda *s: torch.randn(*s, generator=rnd, device="cuda").requires_grad_(True)  # noqa: E731
    qkv = [leaf(2, 33, 4, 64) for _ in range(3)]
    ffn = [leaf(2, 33, 64), leaf(128, 64), leaf(128), leaf(64, 128), leaf(64)]
    for leaves, f in ((qkv, tf.attention), (ffn, tf.feed_forward)):
        hand = [t.detach().bfloat16().requires_grad_(True) for t in leaves]
        with torch.autocast("cuda", dtype=torch.bfloat16):
            out = f(*leaves)
        out.float().square().sum().backward()
        want = f(*hand)
        want.float().square().sum().backward()
        assert torch.equal(out, want)
        for t, h in zip(leaves, hand):
            assert t.grad.dtype == torch.float32 and torch.equal(t.grad, h.grad.float())
    x, f = leaf(2, 33, 64), leaf(2, 33, 64).detach().bfloat16().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):  # a float32 sum and a block's 16-bit result
        r, h = tf.resnorm(x, f)
    (r.square().sum() + (h * x.detach()).sum()).backward()
    wide = [t.detach().float().requires_grad_(True) for t in (x, f)]
    r2, h2 = tf.resnorm(*wide)
    (r2.square().sum() + (h2 * x.detach()).sum()).backward()
    assert torch.equal(r, r2) and torch.equal(h, h2)
    assert torch.equal(x.grad, wide[0].grad) and torch.equal(f.grad, wide[1].grad.bfloat16())
    with pytest.raises(ValueError):
        tf.resnorm(x, f)  # outside a region types are the caller's


@pytest.mark.parametrize("act,slope", [("lrelu", 0.0), ("lrelu", 0.1), ("lrelu_sign", 0.0), ("gelu", 0.0), ("silu", 0.0)])
def test_feed_forward_gradients(act, slope):
    """Against float64's of the function itself, relative L2, float32 operands (products in float32: 1e-6 and a cube root
    of it for the kink's flips).  The 8-bit form is off by max / 254 / sqrt(3) of a block, 0.7 % of its spread: it
    enters w2's gradient whole (1.2 % for a ReLU, half of whose values are 0 and whose norm is less) and through
    act' those of x, w1 and b1, where the leaky ReLU has none.  Differentiated at the rounded value, its own would be off
    by 7 %."""
    g = torch.Generator(device="cuda").manual_seed(7)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    leaves = [rnd(300, 64), rnd(512, 64) / 8, 0.1 * rnd(512), rnd(64, 512) / 22, 0.1 * rnd(64)]
    dout = rnd(300, 64)
    low = [t.clone().requires_grad_(True) for t in leaves]
    tf.feed_forward(*low, act=act, slope=slope).backward(dout)
    x, w1, b1, w2, b2 = high = [t.double().requires_grad_(True) for t in leaves]
    f = {"gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}.get(
        act, lambda u: torch.nn.functional.leaky_relu(u, slope))
    (f(x @ w1.T + b1) @ w2.T + b2).backward(dout.double())
    off = [float((a.grad.double() - b.grad).norm() / b.grad.norm()) for a, b in zip(low, high)]
    exact = 1e-3 if act.startswith("lrelu") else 1e-2
    assert max(off[:3]) < exact and off[3] < 2e-2 and off[4] < 1e-5, off
