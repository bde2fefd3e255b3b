"""The 8-bit activation checkpoint (wubu_b200_act8_*) against its definition.

The kept form is whole numbers and scales, each one IEEE operation on float32 values, so it is compared bit
for bit with the same operations on the CPU.  y, dx and the recomputed y are compared with float64
functions of x and of the restored x': an element may be off by the unit roundoff u of its type (2^-8
bf16, 2^-11 fp16, 2^-24 fp32), plus 2e-6 of the value range for the float32 erf / exp and the
cancellation in 1 + erf (a few ulps of 1 times |x| <= 8)."""
import math

import pytest
import torch

from wuburvc_b200 import transformer as tf

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def kept_reference(x):
    """(q, scale) of the definition, float32 on the CPU."""
    x = x.float().cpu()
    C = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -C % 128)).unflatten(-1, (-1, 128))
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    none = top < 2.0 ** -100
    top1 = torch.where(none | bad, torch.ones_like(top), top)
    scale = torch.where(none, torch.zeros_like(top), top1 / 127)
    inv = torch.where(none, torch.zeros_like(top), torch.full_like(top, 127.0) / top1)
    q = torch.round(b * inv.unsqueeze(-1))
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q).to(torch.int8)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    return q.flatten(-2)[..., :C], scale


def act64(x, act, slope):
    """(act(x), act'(x)) in float64."""
    x = x.double()
    if act == "lrelu":
        return torch.where(x > 0, x, slope * x), torch.where(x > 0, 1.0, slope)
    if act == "silu":
        t = torch.sigmoid(x)
        return x * t, t + x * t * (1 - t)
    if act == "gelu":
        phi = torch.special.ndtr(x)
        return x * phi, phi + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    return x, torch.ones_like(x)


def near(a, b, dtype, scale=1.0):
    return bool((a.double().cpu() - b.cpu()).abs().le(U[dtype] * b.cpu().abs() + 2e-6 * scale).all())


SHAPES = [(1, 1), (3, 7), (1, 128), (5, 129), (2, 33, 768), (7, 200), (4, 2048), (1, 1000), (3, 121), (2, 3, 5, 64)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("act,slope", [("gelu", 0.0), ("silu", 0.0), ("lrelu", 0.0), ("lrelu", 0.1), ("identity", 0.0)])
def test_forward_and_backward(shape, dtype, act, slope):
    g = torch.Generator().manual_seed(sum(shape) + len(act))
    x = (1.5 * torch.randn(shape, generator=g)).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    y, kept = tf.act8_forward(x.cuda(), act, slope=slope)
    dx, again = tf.act8_backward(dy.cuda(), kept, recompute=True)
    q, scale = kept_reference(x)
    assert torch.equal(kept.q.cpu(), q) and torch.equal(kept.scale.cpu(), scale)
    assert near(y, act64(x, act, slope)[0], dtype)
    held = (q.float() * scale.repeat_interleave(128, -1)[..., : shape[-1]])
    y2, d2 = act64(held, act, slope)
    assert near(again, y2, dtype) and near(dx, dy.double() * d2, dtype, scale=4.0)
    assert near(tf.act8_restore(kept), held.double(), dtype, scale=0.0)
    # alone: the recomputed output, the gradient, and a checkpoint without the output
    assert torch.equal(tf.act8_backward(None, kept)[1], again)
    only, none = tf.act8_backward(dy.cuda(), kept)
    assert none is None and torch.equal(only, dx)
    none, kept2 = tf.act8_forward(x.cuda(), act, slope=slope, with_output=False)
    assert none is None and torch.equal(kept2.q, kept.q) and torch.equal(kept2.scale, kept.scale)


@pytest.mark.parametrize("C", [256, 250])
def test_strided_rows_and_unaligned_addresses(C):
    big = torch.randn(6, 9, 2 * C + 8, device="cuda").to(torch.bfloat16)
    dyb = torch.randn(6, 9, 3 * C, device="cuda").to(torch.bfloat16)
    for off in (0, 1, 8):
        x, dy = big[:, :, off:off + C], dyb[:, :, off:off + C]
        y, kept = tf.act8_forward(x)
        yc, keptc = tf.act8_forward(x.contiguous())
        assert torch.equal(y, yc) and torch.equal(kept.q, keptc.q) and torch.equal(kept.scale, keptc.scale)
        assert torch.equal(tf.act8_backward(dy, kept)[0], tf.act8_backward(dy.contiguous(), kept)[0])
    xt = big[:, :, :C].transpose(0, 1)  # no single row stride: copied
    assert torch.equal(tf.act8_forward(xt)[0], tf.act8_forward(xt.contiguous())[0])


@pytest.mark.parametrize("C", [384, 381])
def test_zeros_tiny_values_infinities_and_nan(C):
    x = torch.randn(4, C)
    x[0, :128] = 0
    x[1, 128:256] *= 2.0 ** -110
    x[2, 5] = math.inf
    x[3, 300] = math.nan
    _, kept = tf.act8_forward(x.cuda(), "identity")
    q, scale = kept_reference(x)
    assert torch.equal(kept.q.cpu(), q) and torch.equal(kept.scale.cpu().nan_to_num(-1), scale.nan_to_num(-1))
    back = tf.act8_restore(kept).cpu()
    assert (back[0, :128] == 0).all() and (back[1, 128:256] == 0).all()
    assert back[2, :128].isnan().all() and back[3, 256:384].isnan().all()
    assert back[2, 128:].isfinite().all() and back[3, :256].isfinite().all()


@pytest.mark.parametrize("C", [384, 381])
@pytest.mark.parametrize("dtype", list(U), ids=str)
@pytest.mark.parametrize("act,slope", [("gelu", 0.0), ("silu", 0.0), ("lrelu", 0.0), ("lrelu", 0.1), ("lrelu_sign", 0.0)])
def test_a_block_that_is_not_finite_has_no_finite_gradient(act, slope, dtype, C):
    """An overflow shows in the gradient under every activation, and in its own block alone."""
    x, dy = torch.randn(4, C).to(dtype), torch.randn(4, C).to(dtype)
    x[2, 5] = math.inf
    x[3, 300] = math.nan
    _, kept = tf.act8_forward(x.cuda(), act, slope=slope)
    for t in tf.act8_backward(dy.cuda(), kept, recompute=True):
        assert t[2, :128].isnan().all() and t[3, 256:].isnan().all()
        assert t[:2].isfinite().all() and t[2, 128:].isfinite().all() and t[3, :256].isfinite().all()


def test_gradient_against_differences():
    """dx dy-weighted against central differences of the forward at the restored point (float32): the
    third derivative of gelu is below 2, so a step of 1e-2 is off by 4e-5, rounding by 1e-7 / 1e-2."""
    x = torch.randn(64, 256, device="cuda")
    _, kept = tf.act8_forward(x, "gelu")
    held = tf.act8_restore(kept)
    dx, _ = tf.act8_backward(torch.ones_like(x), kept)
    h = 1e-2
    up, down = (tf.act8_forward(held + s * h, "gelu")[0] for s in (1, -1))
    assert ((up - down).double() / (2 * h) - dx).abs().max() < 2e-4


@pytest.mark.parametrize("C", [256, 250])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_lrelu_sign_keeps_every_derivative(C, dtype):
    """Positive values are kept as at least one step: the derivative is that of x itself, exactly, and x' is off
    by less than a step."""
    g = torch.Generator().manual_seed(C)
    x = torch.randn(60, C, generator=g).to(dtype).cuda()
    dy = torch.randn(60, C, generator=g).to(dtype).cuda()
    y, kept = tf.act8_forward(x, "lrelu_sign", slope=0.25)
    dx, again = tf.act8_backward(dy, kept, recompute=True)
    assert torch.equal(y, tf.act8_forward(x, "lrelu", slope=0.25)[0])
    assert torch.equal(dx, torch.where(x > 0, dy, (dy.float() * 0.25).to(dtype)))
    step = kept.scale.repeat_interleave(128, -1)[:, :C]
    assert ((again.float() - y.float()).abs() <= 1.01 * step + U[dtype] * y.float().abs()).all()


@pytest.mark.parametrize("C", [256, 250])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_lrelu_sign_of_tiny_blocks(C, dtype):
    """Blocks below 2^-100, with zeros among them, keep their derivatives too; x' is off by 2^-100 at most, and a block
    of zeros is restored as zeros."""
    x = (torch.randn(6, C) * 2.0 ** -110).to(dtype).cuda()
    x[:, ::5] = 0
    x[1, :128] = 0
    x[2, 128:] *= 2.0 ** -12  # float32: subnormal
    dy = torch.randn(6, C).to(dtype).cuda()
    _, kept = tf.act8_forward(x, "lrelu_sign", slope=0.25)
    dx, again = tf.act8_backward(dy, kept, recompute=True)
    assert torch.equal(dx, torch.where(x > 0, dy, (dy.float() * 0.25).to(dtype)))
    assert (again.double() - x.double()).abs().max() <= 2.0 ** -100 and (again[1, :128] == 0).all()


def test_parts_of_a_kept_form():
    """Rows, or whole blocks of columns, of a kept form are a kept form: the same bits as that part of the whole."""
    x, dy = (torch.randn(3, 40, 512, device="cuda").bfloat16() for _ in range(2))
    _, kept = tf.act8_forward(x)
    dx, y = tf.act8_backward(dy, kept, recompute=True)
    for rows, cols, blocks in ((slice(1, 2), slice(None), slice(None)), (slice(None), slice(128, 384), slice(1, 3))):
        part = kept._replace(q=kept.q[:, 5:, cols][rows], scale=kept.scale[:, 5:, blocks][rows])
        dx2, y2 = tf.act8_backward(dy[:, 5:, cols][rows], part, recompute=True)
        assert torch.equal(dx2, dx[:, 5:, cols][rows]) and torch.equal(y2, y[:, 5:, cols][rows])
    t = kept._replace(q=kept.q.transpose(0, 1), scale=kept.scale.transpose(0, 1))
    assert torch.equal(tf.act8_backward(dy.transpose(0, 1), t)[0], dx.transpose(0, 1))


def test_empty():
    for shape in ((0, 64), (3, 0)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        y, kept = tf.act8_forward(x)
        assert y.shape == x.shape and tf.act8_backward(x, kept)[0].shape == x.shape


def test_another_stream():
    x = torch.randn(2000, 2048, device="cuda").to(torch.bfloat16)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y, kept = tf.act8_forward(x)
        dx, _ = tf.act8_backward(y, kept)
    side.synchronize()
    y2, kept2 = tf.act8_forward(x)
    assert torch.equal(y, y2) and torch.equal(dx, tf.act8_backward(y2, kept2)[0])
    tf.ops_sync()


def test_refusals():
    x = torch.randn(4, 64, device="cuda")
    _, kept = tf.act8_forward(x)
    for bad in (lambda: tf.act8_forward(x.double()), lambda: tf.act8_forward(x, "tanh"),
                lambda: tf.act8_forward(x.cpu()), lambda: tf.act8_backward(x[:3], kept),
                lambda: tf.act8_backward(x.half(), kept)):
        with pytest.raises(ValueError):
            bad()
