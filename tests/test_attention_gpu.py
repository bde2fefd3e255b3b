"""Softmax attention and its gradient (wubu_b200_attn_*) against float64 and its autograd.

Tolerances follow from the roundings of the operator, element by element.  With u the unit roundoff of the
inputs' type (2^-8 bf16, 2^-11 fp16) and everything else in float32 (relative 1e-5 of the sums' absolute
terms covers sums over a few thousand keys):
  out  one rounding of P, one of the result:            u |O| + u P|V|
  dV   the same:                                        u |dV| + u P^T|dO|
  dS   one rounding, and rowsum(dO O) from the out that the forward returned:
                                                        eS = u |dS| + P (|dO| . eO)
  dQ, dK                                                u |dQ| + scale eS |K|,   u |dK| + scale eS^T |Q|
fp16 results below 2^-14 have a step of 2^-24, so 2^-25 is added."""
import math

import pytest
import torch

from wuburvc_b200 import transformer as tf

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 1e-5


def visible(Tq, Tk, causal, window, ql, kl):
    i = torch.arange(Tq, device="cuda")[:, None]
    j = torch.arange(Tk, device="cuda")[None, :]
    p = i + kl - ql
    see = (i < ql) & (j < kl)
    if causal:
        see = see & (j <= p)
    if window:
        see = see & ((p - j).abs() < window)
    return see


def check(q, k, v, dout, causal=False, window=0, scale=None, q_lens=None, k_lens=None, backward=True):
    opts = dict(causal=causal, window=window, scale=scale, q_lens=q_lens, k_lens=k_lens)
    out, lse = tf.attention_forward(q, k, v, **opts)
    grads = tf.attention_backward(dout, q, k, v, out, lse, **opts) if backward else None
    B, Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[1:3]
    G, u, a = Hq // Hkv, U[q.dtype], scale or D ** -0.5
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == (B, Hq, Tq)

    def near(x, want, tol, what):
        if not x.numel():
            return
        off = (x.double() - want).abs() - tol - tiny
        assert x.isfinite().all() and off.max() <= 0, (what, float(off.max()), float(tol.max()))

    def clean(t, n):  # what lies beyond an item's length takes no part
        t = t.double().clone()
        t[n:] = 0
        return t

    for b in range(B):
        ql = Tq if q_lens is None else int(q_lens[b])
        kl = Tk if k_lens is None else int(k_lens[b])
        see = visible(Tq, Tk, causal, window, ql, kl)
        for hk in range(Hkv):
            K, V = clean(k[b, :, hk], kl), clean(v[b, :, hk], kl)
            dK, dV, eK, eV = (torch.zeros_like(K) for _ in range(4))
            for h in range(hk * G, hk * G + G):
                Q, dO = clean(q[b, :, h], ql), clean(dout[b, :, h], ql)
                S = (Q @ K.T) * a
                S = S.masked_fill(~see, -math.inf)
                m = S.amax(-1, keepdim=True) if Tk else torch.zeros(Tq, 1, device="cuda", dtype=torch.float64)
                m = m.masked_fill(m == -math.inf, 0)
                e = torch.exp(S - m)
                total = e.sum(-1, keepdim=True)
                P = e / total.clamp_min(1e-300)
                O = P @ V
                eO = (u + F32) * (O.abs() + P @ V.abs())
                near(out[b, :, h], O, eO, "out")
                L = (m + total.log()).squeeze(-1)
                some = see.any(-1)
                assert (lse[b, h][~some] == -math.inf).all() and (out[b, :, h][~some] == 0).all()
                assert ((lse[b, h].double() - L)[some].abs() <= 2e-6 * (8 + L[some].abs())).all()
                if not backward:
                    continue
                dP = dO @ V.T
                dS = P * (dP - (P * dP).sum(-1, keepdim=True))
                eS = (u + F32) * dS.abs() + P * (dO.abs() * eO).sum(-1, keepdim=True)
                eS = eS + F32 * P * (dO.abs() @ V.abs().T)
                dQ = a * (dS @ K)
                near(grads[0][b, :, h], dQ, u * dQ.abs() + a * (eS + F32 * dS.abs()) @ K.abs(), "dq")
                assert (grads[0][b, :, h][~some] == 0).all()
                dK += a * (dS.T @ Q)
                eK += a * (eS + F32 * dS.abs()).T @ Q.abs()
                dV += P.T @ dO
                eV += (u + F32) * P.T @ dO.abs()
            if backward:
                near(grads[1][b, :, hk], dK, u * dK.abs() + eK, "dk")
                near(grads[2][b, :, hk], dV, u * dV.abs() + eV, "dv")
                assert (grads[1][b, kl:, hk] == 0).all() and (grads[2][b, kl:, hk] == 0).all()


def make(B, Hq, Hkv, Tq, Tk, D, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return ((spread * r(B, Tq, Hq, D)).to(dtype), r(B, Tk, Hkv, D).to(dtype), r(B, Tk, Hkv, D).to(dtype),
            r(B, Tq, Hq, D).to(dtype))


SHAPES = [  # B, Hq, Hkv, Tq, Tk, D
    (1, 1, 1, 1, 1, 8), (2, 3, 3, 1, 77, 64), (1, 2, 2, 33, 33, 96), (2, 4, 2, 128, 128, 64), (1, 4, 1, 129, 257, 128),
    (2, 2, 2, 300, 200, 40), (1, 2, 1, 513, 513, 64), (3, 12, 12, 50, 50, 64), (1, 2, 2, 1, 1500, 64),
    (1, 8, 2, 2, 700, 128), (1, 1, 1, 260, 1, 16), (2, 2, 1, 127, 130, 104), (1, 3, 3, 256, 640, 96), (1, 6, 2, 384, 384, 80)]
MASKS = {"none": {}, "causal": dict(causal=True), "window": dict(window=40), "self": dict(window=1),
         "causal window": dict(causal=True, window=100)}


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_shapes_and_masks(shape, mask, dtype):
    check(*make(*shape, dtype, seed=sum(shape)), **MASKS[mask])


@pytest.mark.parametrize("shape", [(8, 12, 12, 300, 300, 64), (8, 8, 4, 260, 389, 128), (16, 6, 6, 400, 400, 96)], ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_many_heads(shape, dtype):
    """More items than SMs, several tiles each: every CTA takes several, and no item is split."""
    check(*make(*shape, dtype, seed=7), causal=True)


@pytest.mark.parametrize("shape", [(24, 8, 8, 300, 300, 128), (20, 8, 2, 260, 390, 96), (2, 16, 1, 1500, 1500, 128),
                                   (24, 8, 8, 300, 300, 64)], ids=str)
@pytest.mark.parametrize("mask", ["none", "causal"])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_many_padded_items(shape, mask, dtype):
    """Several times more items than SMs, whole and in parts, many of them empty: a CTA meets an item without steps
    between a keys' and a queries' item, whose second score tile at 128 values lies where dV is read from.  The same
    bits every time."""
    B, Hq, Hkv, Tq, Tk, D = shape
    q, k, v, dout = make(*shape, dtype, seed=sum(shape))
    lens = lambda T: torch.tensor([(T, T // 4, 3 * T // 5, 0, T // 2, 1)[b % 6] for b in range(B)], dtype=torch.int32, device="cuda")  # noqa: E731
    opts = dict(q_lens=lens(Tq), k_lens=lens(Tk), **MASKS[mask])
    check(q, k, v, dout, **opts)
    out, lse = tf.attention_forward(q, k, v, **opts)
    first = tf.attention_backward(dout, q, k, v, out, lse, **opts)
    for _ in range(8):
        again = tf.attention_backward(dout, q, k, v, out, lse, **opts)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    tf.ops_sync()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_many_calls_in_a_row(D, causal):
    """A padded batch, back to back and on changing inputs: no wait in the kernels may depend on how late a warp comes to
    it (steps whose halves are done before the issuing warp looks).  One that did would end after its limit of
    two seconds and show in ops_sync."""
    lens = torch.tensor([max(1, 499 - 23 * b) for b in range(16)], dtype=torch.int32, device="cuda")
    opts = dict(q_lens=lens, k_lens=lens, causal=causal)
    states = [make(16, 12, 12, 499, 499, D, torch.bfloat16, seed=n) for n in range(3)]
    kept = [tf.attention_forward(q, k, v, **opts) for q, k, v, _ in states]
    first = [tf.attention_backward(dout, q, k, v, *o, **opts) for (q, k, v, dout), o in zip(states, kept)]
    tf.ops_sync()
    for n in range(600):
        (q, k, v, dout), o = states[n % 3], kept[n % 3]
        tf.attention_forward(q, k, v, **opts)
        grads = tf.attention_backward(dout, q, k, v, *o, **opts)
        if n % 50 < 3:
            assert all(torch.equal(a, b) for a, b in zip(grads, first[n % 3]))
    tf.ops_sync()


@pytest.mark.parametrize("D", [64, 128])
def test_long_sequences(D):
    """Many tiles an item: the rings go round, the running maximum and the sums span 20 tiles."""
    check(*make(1, 4, 1, 2500, 2500, D, torch.bfloat16, seed=D), causal=True)
    check(*make(1, 2, 2, 3, 5000, D, torch.float16, seed=D))


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("shape", [(1, 2, 1, 1700, 1600, 64), (1, 2, 2, 1540, 1830, 128), (2, 6, 1, 300, 1570, 96),
                                   (3, 2, 2, 1, 900, 64)], ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_items_in_parts(shape, mask, dtype):
    """Few items of many steps, which are split and joined: of one role or both, whole, and with lengths that leave
    parts without a step."""
    q, k, v, dout = make(*shape, dtype, seed=sum(shape))
    check(q, k, v, dout, **MASKS[mask])
    B, Tq, Tk = shape[0], shape[3], shape[4]
    lens = lambda T, first: torch.tensor([first, T // 2 + 1, 0][:B], dtype=torch.int32, device="cuda")  # noqa: E731
    check(q, k, v, dout, q_lens=lens(Tq, min(Tq, 131)), k_lens=lens(Tk, 140), **MASKS[mask])


@pytest.mark.parametrize("mask", list(MASKS))
@pytest.mark.parametrize("T,D", [(300, 64), (130, 96), (70, 128)])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_lengths_and_what_lies_beyond_them(mask, T, D, dtype):
    """Lengths of 0, 1, inside and at a tile's end and whole; NaN and infinities beyond them."""
    lens = torch.tensor([0, 1, T // 2 + 3, min(T, 128), T], dtype=torch.int32, device="cuda")
    q, k, v, dout = make(5, 4, 2, T, T, D, dtype, seed=T)
    for b, n in enumerate(lens.tolist()):
        for t in (q, k, v, dout):
            t[b, n:] = math.nan
            t[b, n::2] = math.inf if b % 2 else -math.inf
    check(q, k, v, dout, q_lens=lens, k_lens=lens, **MASKS[mask])
    # keys alone; queries alone (more queries than keys, or fewer, shift the causal order)
    q, k, v, dout = make(5, 4, 2, 90, T, D, dtype, seed=T + 1)
    check(q, k, v, dout, k_lens=lens, **MASKS[mask])
    ql = torch.tensor([0, 1, 44, 64, 90], dtype=torch.int32, device="cuda")
    check(q, k, v, dout, q_lens=ql, k_lens=lens.flip(0), **MASKS[mask])


@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_peaked_scores(dtype):
    """Scores of about +-60: most probabilities underflow, the running maximum moves by many powers of 2.
    (bf16 and fp16 products are exact in float32; the sums' error of 1e-7 x 60 is inside the tolerance.)"""
    q, k, v, dout = make(1, 2, 2, 400, 400, 64, dtype, seed=5, spread=8.0)
    check(q, k, v, dout)
    k = k.sort(dim=1).values.contiguous()  # rising: every tile moves the maximum
    check(q, k, v, dout, causal=True)


@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("shape", [(1, 32, 32, 70, 200, 64), (1, 32, 32, 70, 200, 128), (1, 32, 32, 70, 200, 24),
                                   (1, 32, 32, 2, 1500, 64), (1, 32, 32, 2, 1500, 128)], ids=str)
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_live_keys_that_are_not_finite(shape, dtype, what):
    """Head h has one key, at a place j = h (mod 32), whose score is NaN or +infinity for every query: whatever its
    place in a tile, the rows that see it are NaN with a NaN lse, and the others have the bits that they have without it."""
    _, H, _, Tq, Tk, D = shape
    q, k, v, _ = make(*shape, dtype, seed=3)
    q[..., 0] = 1
    at = [Tk - 1 - (Tk - 1 - h) % 32 for h in range(H)]  # within the last 32 keys
    for causal in (False, True):
        clean = tf.attention_forward(q, k, v, causal=causal)
        bad = k.clone()
        for h, j in enumerate(at):
            bad[0, j, h, 0] = math.nan if what == "nan" else math.inf
        out, lse = tf.attention_forward(q, bad, v, causal=causal)
        for h, j in enumerate(at):
            sees = visible(Tq, Tk, causal, 0, Tq, Tk)[:, j]
            assert out[0, sees, h].isnan().all() and lse[0, h, sees].isnan().all(), (h, j, causal)
            assert torch.equal(out[0, ~sees, h], clean[0][0, ~sees, h]) and torch.equal(lse[0, h, ~sees], clean[1][0, h, ~sees])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_live_keys_of_no_weight(dtype, D):
    """Scores of -infinity: such keys have no weight, and a row that sees no others has out 0 and lse -inf."""
    q, k, v, _ = make(1, 2, 2, 40, 150, D, dtype, seed=4)
    q[..., 0] = 1
    some, none = k.clone(), k.clone()
    some[:, 100:, :, 0] = -math.inf
    none[..., 0] = -math.inf
    out, lse = tf.attention_forward(q, some, v)
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    out2, lse2 = tf.attention_forward(q, k, v, k_lens=lens)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    out, lse = tf.attention_forward(q, none, v)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("T", [1, 2, 3, 4, 8, 12, 16, 17, 40])
@pytest.mark.parametrize("mask", [{}, dict(causal=True), dict(window=3), dict(causal=True, window=9)], ids=str)
@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_gradients_of_rows_of_few_keys(dtype, D, mask, T):
    """Error against float64 in units of rounding the exact gradient once.  dQ and dK: that rounding and the one of dS,
    whose relative size is the same and which their sums average as they average dS itself: sqrt(2) where both
    spread alike; 1.6 leaves a tenth for the spread over the few elements of short cases (dV: P's, the same).  With D
    from the 16-bit out two keys are at 2.3 and four to sixteen at 1.7-2."""
    B = 4096 // T // (D // 32)
    q, k, v, dout = make(B, 4, 2, T, T, D, dtype, seed=T + D)
    out, lse = tf.attention_forward(q, k, v, **mask)
    got = tf.attention_backward(dout, q, k, v, out, lse, **mask)
    a, b, c = (t.double().transpose(1, 2).requires_grad_(True) for t in (q, k, v))
    s = (a @ b.repeat_interleave(2, 1).transpose(2, 3)) * D ** -0.5
    s = s.masked_fill(~visible(T, T, mask.get("causal", False), mask.get("window", 0), T, T), -math.inf)
    o = torch.softmax(s, -1) @ c.repeat_interleave(2, 1)
    for x, w in zip(got, torch.autograd.grad(o, (a, b, c), dout.double().transpose(1, 2))):
        w = w.transpose(1, 2)
        once = (w.to(dtype).double() - w).norm()
        assert (x.double() - w).norm() <= (1.6 if T > 1 else 1.0) * once + 1e-6 * w.norm() + 1e-6 * dout.double().norm()


@pytest.mark.parametrize("mask", [{}, dict(causal=True), dict(window=20), dict(causal=True, window=5)], ids=str)
@pytest.mark.parametrize("Tq,Tk", [(70, 40), (33, 50), (90, 12)])
def test_gradients_of_rows_of_few_keys_with_lengths(Tq, Tk, mask):
    """The same for items of any length, more and fewer queries than keys, rows that see few keys alone (the others have
    no gradient to give: their dO is 0)."""
    B, D = 64, 64
    q, k, v, dout = make(B, 2, 2, Tq, Tk, D, torch.bfloat16, seed=Tq)
    g = torch.Generator().manual_seed(Tk)
    ql, kl = (torch.randint(1, T + 1, (B,), generator=g).int() for T in (Tq, Tk))
    ql[:8], kl[8:16] = Tq, torch.arange(1, 9)
    see = torch.stack([visible(Tq, Tk, mask.get("causal", False), mask.get("window", 0), int(m), int(n)) for m, n in zip(ql, kl)])
    keys = see.sum(-1)
    few = (keys > 0) & (keys <= 16)
    dout = dout * few[:, :, None, None]
    opts = dict(q_lens=ql.cuda(), k_lens=kl.cuda(), **mask)
    out, lse = tf.attention_forward(q, k, v, **opts)
    got = tf.attention_backward(dout, q, k, v, out, lse, **opts)
    a, b, c = (t.double().transpose(1, 2).requires_grad_(True) for t in (q, k, v))
    s = ((a @ b.transpose(2, 3)) * D ** -0.5).masked_fill(~see[:, None], -1e300)
    o = torch.softmax(s, -1) @ c
    for x, w in zip(got, torch.autograd.grad(o, (a, b, c), dout.double().transpose(1, 2))):
        w = w.transpose(1, 2)
        once = (w.bfloat16().double() - w).norm()
        assert (x.double() - w).norm() <= 1.6 * once + 1e-6 * w.norm() + 1e-6 * dout.double().norm()


@pytest.mark.parametrize("size", [1e-3, 1.0, 300.0])
@pytest.mark.parametrize("dtype", list(U), ids=str)
def test_gradients_of_any_size(size, dtype):
    """dS of a few millionths (1000 keys) or of hundreds: fp16 would lose the first and overflow near the second."""
    q, k, v, dout = make(1, 2, 1, 1000, 1000, 64, dtype, seed=9)
    check(q, k, v, (dout.float() * size).to(dtype))


def test_scale_and_no_keys():
    q, k, v, dout = make(1, 2, 2, 40, 60, 64, torch.bfloat16)
    check(q, k, v, dout, scale=0.5)
    e = torch.empty(1, 0, 2, 64, device="cuda", dtype=torch.bfloat16)
    check(q, e, e, dout)
    dq, dk, dv = tf.attention_backward(e, e, k, v, e, torch.empty(1, 2, 0, device="cuda"))
    assert dq.shape == e.shape and (dk == 0).all() and (dv == 0).all()
    out, lse = tf.attention_forward(q[:0], k[:0], v[:0])
    assert out.shape[0] == 0


def test_strides_and_orders():
    """Views of one projection, heads before tokens, a slice that starts inside a row, an address that is
    not a multiple of 16 bytes and a broadcast head: the same results as from copies."""
    B, T, H, D = 2, 150, 3, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(B, T, 3, H, D, generator=g, device="cuda").to(torch.bfloat16)
    bh = torch.randn(3, B, H, T, D, generator=g, device="cuda").to(torch.bfloat16).transpose(2, 3)
    odd = torch.randn(3, B, T, H, D + 1, generator=g, device="cuda").to(torch.bfloat16)[..., 1:]
    wide = torch.randn(3, B, T + 9, H + 1, D + 8, generator=g, device="cuda").to(torch.bfloat16)[:, :, 5:T + 5, 1:, 8:]
    for q, k, v in (qkv.unbind(2), bh.unbind(0), odd.unbind(0), wide.unbind(0)):
        dout = wide[0]
        out, lse = tf.attention_forward(q, k, v, causal=True)
        c = [t.contiguous() for t in (q, k, v)]
        out2, lse2 = tf.attention_forward(*c, causal=True)
        assert torch.equal(out, out2) and torch.equal(lse, lse2)
        a = tf.attention_backward(dout, q, k, v, out, lse, causal=True)
        b = tf.attention_backward(dout.contiguous(), *c, out, lse, causal=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    one = bh[0][:, :, :1].expand(B, T, H, D)
    assert torch.equal(tf.attention_forward(one, one, one)[0], tf.attention_forward(*(one.contiguous(),) * 3)[0])


def test_deterministic_and_on_another_stream():
    q, k, v, dout = make(2, 8, 2, 700, 700, 64, torch.bfloat16)
    out, lse = tf.attention_forward(q, k, v, causal=True)
    grads = tf.attention_backward(dout, q, k, v, out, lse, causal=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out2, lse2 = tf.attention_forward(q, k, v, causal=True)
        grads2 = tf.attention_backward(dout, q, k, v, out2, lse2, causal=True)
    side.synchronize()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    assert all(torch.equal(x, y) for x, y in zip(grads, grads2))
    tf.ops_sync()


def test_autograd():
    q, k, v, dout = make(1, 4, 2, 65, 65, 64, torch.bfloat16)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = tf.attention(*leaves, causal=True)
    out.backward(dout)
    o, lse = tf.attention_forward(q, k, v, causal=True)
    for t, g in zip(leaves, tf.attention_backward(dout, q, k, v, o, lse, causal=True)):
        assert torch.equal(t.grad, g)


def test_gradient_against_differences():
    """d sum(out dO) along s = sign(gradient), whose slope is sum |gradient|, by central differences of the
    forward with steps of 2^-5 that leave the inputs exact in fp16.  The step's third-order term is near
    1e-3 of it, the fp16 rounding of out 2^-12 sqrt(n) / 2^-5 against sum |gradient|: 3 % holds both."""
    q, k, v, dout = (((t * 64).round() / 64).half() for t in make(1, 2, 1, 150, 150, 32, torch.float32, seed=4))
    out, lse = tf.attention_forward(q, k, v, causal=True)
    grads = tf.attention_backward(dout, q, k, v, out, lse, causal=True)
    for n in range(3):
        s = torch.sign(grads[n])
        e = 2.0 ** -5

        def value(sign):
            x = [t + sign * e * s if m == n else t for m, t in enumerate((q, k, v))]
            return (tf.attention_forward(*x, causal=True)[0].double() * dout.double()).sum()

        want = grads[n].double().abs().sum()
        assert abs((value(1) - value(-1)) / (2 * e) - want) <= 0.03 * want


def test_refusals():
    q, k, v, dout = make(1, 4, 2, 20, 20, 64, torch.bfloat16)
    out, lse = tf.attention_forward(q, k, v)
    for bad in (lambda: tf.attention_forward(q.float(), k.float(), v.float()), lambda: tf.attention_forward(q, k.half(), v.half()),
                lambda: tf.attention_forward(q[..., :36], k[..., :36], v[..., :36]),
                lambda: tf.attention_forward(q[:, :, :3], k, v), lambda: tf.attention_forward(q, k, v[:, :5]),
                lambda: tf.attention_forward(q, k, v, window=-1), lambda: tf.attention_forward(q, k, v, scale=0.0),
                lambda: tf.attention_forward(q, k, v, k_lens=torch.ones(2, dtype=torch.int32, device="cuda")),
                lambda: tf.attention_forward(q, k, v, k_lens=torch.ones(1, dtype=torch.int32)),
                lambda: tf.attention_forward(q.cpu(), k.cpu(), v.cpu()),
                lambda: tf.attention_backward(dout[:, :3], q, k, v, out, lse),
                lambda: tf.attention_backward(dout, q, k, v, out, lse[:, :2])):
        with pytest.raises(ValueError):
            bad()
