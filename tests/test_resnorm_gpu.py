"""The fused norms, gate and residual scale (wubu_b200_resnorm_*) against float64 autograd.

r, h, dx and df are float32 results rounded once: an element may be off by the unit roundoff u of its type
times its size, plus 2e-5 of the tensor's largest value (float32 rounding of sums over up to 8192 columns,
about sqrt(8192) x 2^-24 = 5e-6, through up to two norms).  The vectors' gradients are float32 sums over
rows: relative L2 1e-5."""
import pytest
import torch

from wuburvc_b200 import transformer as tf

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
NAMES = ("weight", "bias", "post_weight", "post_bias", "gate")


def norm64(v, kind, w, b, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)
    v = v if w is None else v * w
    return v if b is None else v + b


def forward64(t, norm, post, res_scale, eps):
    u = norm64(t["f"], post, t["post_weight"], t["post_bias"], eps)
    if t["gate"] is not None:
        g = t["gate"]
        u = u * (g if g.dim() == 1 else g.view(g.shape[0], *([1] * (u.dim() - 2)), -1))
    r = res_scale * t["x"] + u
    return r, norm64(r, norm, t["weight"], t["bias"], eps)


def make(shape, dtype, norm, post, gate, seed=0, affine=True):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    rnd = lambda *s, m=0.0, d=1.0: (m + d * torch.randn(*s, generator=g)).cuda()  # noqa: E731
    t = {"x": rnd(*shape).to(dtype), "f": rnd(*shape, m=0.3).to(dtype)}
    t["weight"] = rnd(C, m=1.0, d=0.2) if norm and affine else None
    t["bias"] = rnd(C, d=0.2) if norm == "layer" and affine else None
    t["post_weight"] = rnd(C, m=1.0, d=0.2) if post and affine else None
    t["post_bias"] = rnd(C, d=0.2) if post == "layer" and affine else None
    t["gate"] = {None: None, "column": rnd(C), "item": rnd(shape[0], C)}[gate]
    dr, dh = rnd(*shape).to(dtype), rnd(*shape).to(dtype)
    return t, dr, dh


def near(a, b, dtype):
    b = b.detach()
    return bool((a.double() - b).abs().le(U[dtype] * b.abs() + 2e-5 * b.abs().max()).all())


def check(shape, dtype, norm, post, gate, res_scale=1.0, use_dr=True, use_dh=True, affine=True, eps=1e-5):
    t, dr, dh = make(shape, dtype, norm, post, gate, seed=sum(shape), affine=affine)
    kw = dict(norm=norm, post=post, res_scale=res_scale, eps=eps, **{n: t[n] for n in NAMES})
    r, h = tf.resnorm_forward(t["x"], t["f"], **kw)
    t64 = {n: None if v is None else v.double().requires_grad_(True) for n, v in t.items()}
    r64, h64 = forward64(t64, norm, post, res_scale, eps)
    assert near(r, r64, dtype)
    assert (h is None) == (norm is None)
    if norm:
        assert near(h, h64, dtype)
        none, h2 = tf.resnorm_forward(t["x"], t["f"], keep_sum=False, **kw)
        assert none is None and torch.equal(h, h2)
    dr, dh = dr if use_dr or not norm else None, dh if use_dh and norm else None
    got = tf.resnorm_backward(dr, dh, t["x"], t["f"], **kw)
    loss = sum((a * g.double()).sum() for a, g in ((r64, dr), (h64, dh)) if g is not None)
    loss.backward()
    assert near(got["dx"], t64["x"].grad, dtype) and near(got["df"], t64["f"].grad, dtype)
    for n in NAMES:
        if t[n] is None:
            assert got["d" + n] is None
            continue
        want = t64[n].grad if t64[n].grad is not None else torch.zeros_like(t64[n])
        off = (got["d" + n].double() - want).norm()
        assert off <= 1e-5 * want.norm(), (n, float(off / want.norm()))


SHAPES = [(1, 1, 1), (1, 1, 8), (2, 3, 31), (1, 33, 192), (3, 17, 768), (2, 5, 100), (2, 700, 64), (5, 1, 333),
          (1, 40, 2048), (2, 9, 2056), (1, 3, 8192), (1, 3, 8191), (2, 3, 4, 48)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_shapes_and_types(shape, dtype):
    for norm, post, gate in (("layer", None, None), ("rms", "rms", "item"), ("layer", "layer", "column")):
        if shape[-1] == 1:  # a norm over one column: its gradient is eps / v^2 of the terms that cancel in it
            t, _, _ = make(shape, dtype, norm, post, gate)
            r, h = tf.resnorm_forward(t["x"], t["f"], norm=norm, post=post, **{n: t[n] for n in NAMES})
            r64, h64 = forward64({n: None if v is None else v.double() for n, v in t.items()}, norm, post, 1.0, 1e-5)
            assert near(r, r64, dtype) and near(h, h64, dtype)
            continue
        check(shape, dtype, norm, post, gate)


@pytest.mark.parametrize("norm", [None, "layer", "rms"])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("gate", [None, "column", "item"])
def test_every_form(norm, post, gate):
    for C in (96, 97):
        check((3, 21, C), torch.float32, norm, post, gate, res_scale=0.5)
        check((3, 21, C), torch.bfloat16, norm, post, gate, affine=False)
    check((2, 21, 96), torch.float32, norm, post, gate, use_dr=False)
    if norm:
        check((2, 21, 96), torch.float32, norm, post, gate, use_dh=False)


def test_rows_without_items():
    """[rows, cols]: every row is an item, which takes no more workspace than the same rows in one item."""
    for gate in (None, "column", "item"):
        check((70, 96), torch.float32, "layer", "rms", gate)
    x = torch.randn(40000, 64, device="cuda").to(torch.bfloat16)
    w = torch.rand(64, device="cuda")
    flat = tf.resnorm_backward(x, x, x, x, weight=w)
    whole = tf.resnorm_backward(*(x[None],) * 4, weight=w)
    assert torch.equal(flat["dx"], whole["dx"][0]) and torch.equal(flat["dweight"], whole["dweight"])


def test_strided_rows():
    big = torch.randn(4, 10, 3 * 64, device="cuda").to(torch.bfloat16)
    x, f = big[..., :64], big[..., 64:128]
    w = torch.rand(64, device="cuda")
    r, h = tf.resnorm_forward(x, f, weight=w)
    r2, h2 = tf.resnorm_forward(x.contiguous(), f.contiguous(), weight=w)
    assert torch.equal(r, r2) and torch.equal(h, h2)
    a = tf.resnorm_backward(x, f, x, f, weight=w)
    b = tf.resnorm_backward(x.contiguous(), f.contiguous(), x.contiguous(), f.contiguous(), weight=w)
    assert torch.equal(a["dx"], b["dx"]) and torch.equal(a["df"], b["df"]) and torch.equal(a["dweight"], b["dweight"])
    odd = torch.randn(4, 10, 65, device="cuda")[..., 1:]  # rows that no 16-byte piece starts
    assert torch.allclose(tf.resnorm_forward(odd, odd)[1], tf.resnorm_forward(odd.contiguous(), odd.contiguous())[1],
                          rtol=0, atol=1e-5)


def test_large_mean_keeps_its_variance():
    """Values near 1000 with a spread of 1: E[v^2] - E[v]^2 in float32 would be off by 5 %."""
    x = 1000 + torch.randn(4, 5, 768, device="cuda")
    _, h = tf.resnorm_forward(x, torch.zeros_like(x))
    want = norm64(x.double(), "layer", None, None, 1e-5)
    assert (h.double() - want).abs().max() < 1e-3  # 1000 x 2^-24 per element, 17 standard errors


def test_zero_rows_and_nan_stay_in_their_row():
    x = torch.randn(1, 6, 64, device="cuda")
    f = torch.zeros_like(x)
    x[0, 1] = 0
    x[0, 3, 7] = float("nan")
    _, h = tf.resnorm_forward(x, f, norm="rms")
    assert (h[0, 1] == 0).all() and h[0, 3].isnan().all() and h[0, [0, 2, 4, 5]].isfinite().all()
    e = tf.resnorm_backward(None, torch.empty(2, 0, 64, device="cuda"), *(torch.empty(2, 0, 64, device="cuda"),) * 2,
                            weight=torch.ones(64, device="cuda"), gate=torch.ones(2, 64, device="cuda"))
    assert (e["dweight"] == 0).all() and (e["dgate"] == 0).all() and e["dgate"].shape == (2, 64)


@pytest.mark.parametrize("shape,norm,post,gate", [((2, 1500, 4096), "layer", None, None), ((3, 700, 3200), "rms", "rms", "item"),
                                                  ((1, 2000, 5001), "layer", "layer", "column")], ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_wide_rows_by_the_thousand(shape, dtype, norm, post, gate):
    """Rows that take a block each, many to a block."""
    check(shape, dtype, norm, post, gate)


@pytest.mark.parametrize("C", [96, 97, 4000])
def test_each_gradient_alone(C):
    """`need` leaves outputs out; what is left has the same bits."""
    t, dr, dh = make((3, 50, C), torch.bfloat16, "layer", "layer", "item")
    kw = dict(norm="layer", post="layer", **{n: t[n] for n in NAMES})
    want = tf.resnorm_backward(dr, dh, t["x"], t["f"], **kw)
    assert all(v is not None for v in want.values())
    for n, v in want.items():
        got = tf.resnorm_backward(dr, dh, t["x"], t["f"], need=[n], **kw)
        assert torch.equal(got.pop(n), v) and all(u is None for u in got.values())


def test_deterministic():
    t, dr, dh = make((4, 500, 768), torch.bfloat16, "rms", "rms", "item")
    kw = dict(norm="rms", post="rms", **{n: t[n] for n in NAMES})
    a, b = (tf.resnorm_backward(dr, dh, t["x"], t["f"], **kw) for _ in range(2))
    assert all(v is None or torch.equal(v, b[n]) for n, v in a.items())


def test_gradient_against_differences():
    """The directional derivative of sum(dr r + dh h) in float32 against central differences of the
    forward: a step of 1e-2 of unit-variance inputs is off by order 1e-4, rounding by 1e-7 sqrt(n) / 1e-2."""
    t, dr, dh = make((2, 8, 64), torch.float32, "layer", "rms", "item", seed=3)
    kw = dict(norm="layer", post="rms", **{n: t[n] for n in NAMES})
    got = tf.resnorm_backward(dr, dh, t["x"], t["f"], **kw)

    def value(x, f):
        r, h = tf.resnorm_forward(x, f, **kw)
        return (r.double() * dr + h.double() * dh).sum()

    g = torch.Generator(device="cuda").manual_seed(1)
    for n in ("x", "f"):
        d = torch.randn(t[n].shape, generator=g, device="cuda")
        e = 1e-2
        up, down = (value(*(t[m] + (s * e * d if m == n else 0) for m in ("x", "f"))) for s in (1, -1))
        want = (got["d" + n].double() * d).sum()
        assert abs((up - down) / (2 * e) - want) <= 2e-3 * got["d" + n].double().norm() * d.double().norm() / 8


def test_refusals():
    x = torch.randn(2, 4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    for bad in (lambda: tf.resnorm_forward(x, x[:1]), lambda: tf.resnorm_forward(x, x.half()),
                lambda: tf.resnorm_forward(x, x, norm="batch"), lambda: tf.resnorm_forward(x, x, weight=w[:3]),
                lambda: tf.resnorm_forward(x, x, norm="rms", bias=w), lambda: tf.resnorm_forward(x, x, gate=x),
                lambda: tf.resnorm_forward(x.cpu(), x.cpu()), lambda: tf.resnorm_forward(x, x, weight=w.cpu()),
                lambda: tf.resnorm_backward(None, None, x, x), lambda: tf.resnorm_backward(x, x, x, x, norm=None),
                lambda: tf.resnorm_forward(x.double(), x.double()), lambda: tf.resnorm_forward(x, x, norm=None, weight=w)):
        with pytest.raises(ValueError):
            bad()
    wide = torch.randn(1, 1, 8200, device="cuda")
    with pytest.raises(RuntimeError):
        tf.resnorm_forward(wide, wide)
