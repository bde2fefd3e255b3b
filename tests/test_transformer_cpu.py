"""The transformer operators' checks that come before anything is launched: no GPU is needed.  The addresses
are never followed."""
import ctypes
import struct

import pytest
import torch

from wuburvc_b200 import transformer as tf

OK, ARG, SHAPE, NOMEM = 0, -1, -3, -6
A = 1 << 20  # an aligned address


def act8(fn="forward", dtype=1, act=2, x=A, stride=64, y=A, q=A, scale=A, dx=A, rows=4, cols=64):
    h = tf.L()
    if fn == "forward":
        return h.wubu_b200_act8_forward(dtype, act, 0.0, x, stride, y, q, scale, rows, cols, None)
    return h.wubu_b200_act8_backward(dtype, act, 0.0, x, stride, q, scale, dx, y, rows, cols, None)


def test_act8_refusals():
    assert act8(rows=0) == OK and act8(cols=0) == OK and act8("backward", rows=0) == OK
    for bad in (dict(dtype=3), dict(dtype=-1), dict(act=5), dict(act=-1), dict(rows=-1), dict(cols=-1), dict(q=None),
                dict(scale=None), dict(x=None), dict(stride=63)):
        assert act8(**bad) == ARG, bad
    for bad in (dict(q=None), dict(scale=None), dict(x=None), dict(dx=None), dict(stride=10), dict(x=None, dx=None, y=None)):
        assert act8("backward", **bad) == ARG, bad
    assert act8(rows=1 << 40) == SHAPE


RESNORM = ("dtype norm post gate items rows cols res_scale eps reserved x xs f fs weight bias post_weight post_bias gate_values "
           "r h dr drs dh dhs dx df dgate dpost_weight dpost_bias dweight dbias ws n").split()


def resnorm(fn, **kw):
    v = dict.fromkeys(RESNORM, 0)
    v.update(dtype=1, norm=1, items=2, rows=3, cols=64, res_scale=1.0, eps=1e-5, x=A, xs=64, f=A, fs=64, r=A, h=A, dh=A,
             dhs=64, dx=A, df=A)
    v.update(kw)
    b = tf._RESNORM.pack(*(v[n] for n in RESNORM))
    h = tf.L()
    return h.wubu_b200_resnorm_workspace(b) if fn == "workspace" else getattr(h, "wubu_b200_resnorm_" + fn)(b, None)


def test_resnorm_refusals():
    assert resnorm("forward", items=0) == OK and resnorm("forward", rows=0) == OK
    assert resnorm("workspace") > 0 and resnorm("workspace", items=0) == 0
    for bad in (dict(dtype=5), dict(norm=3), dict(post=-1), dict(gate=3), dict(items=-1), dict(x=0), dict(f=0), dict(xs=63),
                dict(gate=1), dict(eps=-1.0), dict(eps=float("nan"))):
        assert resnorm("forward", **bad) == ARG, bad
        assert resnorm("backward", **bad) == ARG, bad
    for bad in (dict(cols=0), dict(cols=8193), dict(items=1 << 20, rows=1 << 20)):
        assert resnorm("forward", **bad) == SHAPE and resnorm("workspace", **bad) == SHAPE
    assert resnorm("forward", h=0) == ARG and resnorm("forward", norm=0) == ARG and resnorm("forward", norm=0, h=0, r=0) == ARG
    for bad in (dict(norm=0), dict(dgate=A), dict(dpost_weight=A), dict(dweight=A), dict(dhs=8), dict(norm=0, dh=0, dweight=A)):
        assert resnorm("backward", **bad) == ARG, bad
    assert resnorm("backward", dweight=A, ws=A, n=16) == NOMEM


ATTN = "dtype B Hq Hkv Tq Tk D causal window scale q_lens k_lens".split()


def attn(fn, views=None, lse=A, ws=0, n=0, **kw):
    v = dict(dtype=1, B=2, Hq=4, Hkv=2, Tq=10, Tk=12, D=64, causal=0, window=0, scale=0.0, q_lens=0, k_lens=0)
    v.update(kw)
    names = "q k v out dout dq dk dv".split()
    w = {m: (A, v["D"] * 4 * 16, v["D"] * 4, v["D"]) for m in names}
    w.update(views or {})
    flat = [w[m] for m in names]
    b = tf._ATTN.pack(*(v[m] for m in ATTN), *sum(flat[:4], ()), lse, *sum(flat[4:], ()), ws, n)
    h = tf.L()
    return h.wubu_b200_attn_workspace(b, 1) if fn == "workspace" else getattr(h, "wubu_b200_attn_" + fn)(b, None)


def test_attention_refusals():
    assert attn("forward", B=0) == OK and attn("backward", B=0) == OK and attn("forward", Tq=0, Tk=0) == OK
    assert attn("workspace") > 0
    for bad in (dict(dtype=0), dict(dtype=7), dict(B=-1), dict(Tq=-5), dict(window=-1), dict(scale=-1.0),
                dict(scale=float("nan")), dict(scale=float("inf"))):
        assert attn("forward", **bad) == ARG and attn("backward", **bad) == ARG, bad
    for bad in (dict(D=0), dict(D=60), dict(D=136), dict(Hkv=3), dict(Hkv=0), dict(Hq=0), dict(B=70000), dict(Tk=1 << 29)):
        assert attn("forward", **bad) == SHAPE and attn("workspace", **bad) == SHAPE, bad
    for m in ("q", "k", "v", "out"):
        for view in ((0, 4096, 256, 64), (A + 2, 4096, 256, 64), (A, 4096, 256, 60), (A, 4096, 0, 64), (A, -8, 256, 64),
                     (A, 4096, 252, 64)):
            assert attn("forward", views={m: view}) == ARG, (m, view)
    for m in ("dout", "dq", "dk", "dv"):
        assert attn("backward", views={m: (A + 8, 4096, 256, 64)}) == ARG
    assert attn("forward", lse=0) == ARG
    assert attn("backward", ws=A, n=8) == NOMEM and attn("backward") == ARG


def test_structures_match_the_header(tmp_path):
    src = tmp_path / "size.c"
    src.write_text('#include "wuburvc_b200.h"\nint resnorm(void){return sizeof(WubuB200ResNorm);}\n'
                   "int attn(void){return sizeof(WubuB200Attn);}\n")
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    so = str(tmp_path / "size.so")
    subprocess.check_call(["gcc", "-shared", "-fPIC", "-I" + os.path.join(root, "include"), str(src), "-o", so])
    lib = ctypes.CDLL(so)
    assert lib.resnorm() == tf._RESNORM.size and lib.attn() == tf._ATTN.size
    assert struct.calcsize("@P") == 8


def test_binding_refuses_cpu_tensors():
    x = torch.zeros(2, 3, 64)
    for call in (lambda: tf.act8_forward(x), lambda: tf.resnorm_forward(x, x),
                 lambda: tf.attention_forward(*(torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16),) * 3)):
        with pytest.raises(ValueError):
            call()


@pytest.fixture
def stand_ins(monkeypatch):
    """torch on the CPU in place of the native calls, as their outputs are to autograd: without a history.  Returns
    the list of the calls: (name, arguments, keyword arguments)."""
    calls = []

    def called(name, f):
        def g(*args, **kw):
            calls.append((name, args, kw))
            with torch.no_grad():
                return f(*args, **kw)
        monkeypatch.setattr(tf, name, g)

    def scores(q, k):
        return torch.einsum("bihd,bjhd->bhij", q, k) * q.shape[-1] ** -0.5

    def attention_forward(q, k, v, **opts):
        s = scores(q, k)
        return torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v), torch.logsumexp(s, -1)

    def attention_backward(dout, q, k, v, out, lse, **opts):
        p = torch.exp(scores(q, k) - lse[..., None])
        dp = torch.einsum("bihd,bjhd->bhij", dout, v)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * q.shape[-1] ** -0.5
        return (torch.einsum("bhij,bjhd->bihd", ds, k), torch.einsum("bhij,bihd->bjhd", ds, q),
                torch.einsum("bhij,bihd->bjhd", p, dout))

    def resnorm_forward(x, f, keep_sum=True, **kw):  # rms, without parameters
        r = x + f
        return r if keep_sum else None, r / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-5)

    def resnorm_backward(dr, dh, x, f, **kw):
        r = x + f
        inv = 1 / torch.sqrt(r.square().mean(-1, keepdim=True) + 1e-5)
        d = 0 if dr is None else dr
        if dh is not None:
            d = d + (dh - r * inv * (dh * r * inv).mean(-1, keepdim=True)) * inv
        return dict(dx=d, df=d, **dict.fromkeys(("dweight", "dbias", "dpost_weight", "dpost_bias", "dgate")))

    def act8_forward(x, act="gelu", slope=0.0, with_output=True):
        return torch.nn.functional.gelu(x), tf.Kept8(x.clone(), x.new_ones(1), act, slope, x.dtype)

    def act8_backward(dy, kept, recompute=False):
        with torch.enable_grad():
            x = kept.q.detach().requires_grad_(True)
            y = torch.nn.functional.gelu(x)
            dx = None if dy is None else torch.autograd.grad(y, x, dy)[0]
        return dx, y.detach()

    for f in (attention_forward, attention_backward, resnorm_forward, resnorm_backward, act8_forward, act8_backward):
        called(f.__name__, f)
    return calls


def autograd_forms():
    """name -> (leaves, function of them) of each form, in float64"""
    g = torch.Generator().manual_seed(0)
    leaf = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_(True)  # noqa: E731
    return {
        "attention": ([leaf(1, 5, 2, 8) for _ in range(3)], lambda q, k, v: tf.attention(q, k, v)),
        "resnorm": ([leaf(2, 3, 8) for _ in range(2)], lambda x, f: sum(tf.resnorm(x, f, norm="rms"))),
        "feed_forward": ([leaf(2, 3, 8), leaf(16, 8), leaf(16), leaf(8, 16), leaf(8)], tf.feed_forward),
    }


@pytest.mark.parametrize("form", ["attention", "resnorm", "feed_forward"])
def test_first_derivatives_are_right_and_second_ones_raise(form, stand_ins):
    leaves, f = autograd_forms()[form]
    assert torch.autograd.gradcheck(f, leaves)
    grads = torch.autograd.grad(f(*leaves).square().sum(), leaves, create_graph=True)
    for g in grads:  # beside a term that can be differentiated
        with pytest.raises(RuntimeError):
            (g.square().sum() + leaves[0].square().sum()).backward(retain_graph=True)


@pytest.mark.parametrize("which", ["q_lens", "k_lens"])
def test_lengths_changed_before_the_backward_are_noticed(which, stand_ins):
    q, k, v = autograd_forms()["attention"][0]
    lens = {n: torch.tensor([5], dtype=torch.int32) for n in ("q_lens", "k_lens")}
    tf.attention(q, k, v, **lens).sum().backward()
    assert all(kw["q_lens"] is not None and kw["k_lens"] is not None for _, _, kw in stand_ins)
    out = tf.attention(q, k, v, **lens)
    lens[which].fill_(3)  # the next batch's lengths in the same buffer
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("form", ["attention", "resnorm", "feed_forward"])
def test_autocast(form, inside, stand_ins):
    """float32 leaves under autocast: what the native calls see is in one type, the gradients come back in the leaves'
    type and near the float64 ones (bf16 roundings of a few terms: 2^-9 each, 2 % holds ten in a row), whether
    the backward runs inside the region or outside."""
    leaves, f = autograd_forms()[form]
    want = torch.autograd.grad(f(*leaves).square().sum(), leaves)
    low = [t.detach().float().requires_grad_(True) for t in leaves]
    if form == "resnorm":  # a float32 sum and a block's 16-bit result
        low[1] = low[1].detach().bfloat16().requires_grad_(True)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        out = f(*low)
        assert out.dtype == (torch.float32 if form == "resnorm" else torch.bfloat16)
        if inside:
            out.float().square().sum().backward()
    if not inside:
        out.float().square().sum().backward()
    for t, w in zip(low, want):
        assert t.grad.dtype == t.dtype and (t.grad.double() - w).norm() <= 0.02 * w.norm()


@pytest.mark.parametrize("which", range(5))
def test_frozen_operands_of_feed_forward(which, stand_ins):
    """One operand trained: its gradient is that of training all, and the native call is asked for no more than
    it takes."""
    leaves, f = autograd_forms()["feed_forward"]
    want = torch.autograd.grad(f(*leaves).square().sum(), leaves)[which]
    f(*(t if n == which else t.detach() for n, t in enumerate(leaves))).square().sum().backward()
    assert torch.allclose(leaves[which].grad, want, rtol=1e-12, atol=0)
    assert all(t.grad is None for n, t in enumerate(leaves) if n != which)
    asked = [(a[0] is not None, kw["recompute"]) for name, a, kw in stand_ins if name == "act8_backward"][1:]
    assert asked == {0: [(True, False)], 1: [(True, False)], 2: [(True, False)], 3: [(False, True)], 4: []}[which]


@pytest.mark.parametrize("which", range(7))
def test_frozen_operands_of_resnorm(which, monkeypatch):
    asked = []

    def backward(dr, dh, x, f, need=None, **kw):
        asked.append(need)
        return {n: torch.zeros(8) if n in need else None for n in
                ("dx", "df", "dweight", "dbias", "dpost_weight", "dpost_bias", "dgate")}

    monkeypatch.setattr(tf, "resnorm_forward", lambda x, f, **kw: (x + f, x - f))
    monkeypatch.setattr(tf, "resnorm_backward", backward)
    names = ("x", "f", "weight", "bias", "post_weight", "post_bias", "gate")
    t = {n: torch.ones(8).requires_grad_(m == which) for m, n in enumerate(names)}
    tf.resnorm(t.pop("x"), t.pop("f"), norm="layer", post="layer", **t)[1].sum().backward()
    assert asked == [["d" + names[which]]]


def test_workspaces_are_asked_for_on_the_tensors_device(monkeypatch):
    """Two devices whose workspaces differ: each is asked for with its own device current, whichever was first."""
    import contextlib
    current = [0]

    @contextlib.contextmanager
    def device(dev):
        before, current[0] = current[0], dev
        yield
        current[0] = before

    class Library:
        def wubu_b200_attn_workspace(self, args, backward):
            return 1000 * (1 + current[0]) + backward

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(tf, "L", Library)
    tf._workspace.cache_clear()
    head = (1, 2, 4, 2, 10, 12, 64, 0, 0, 0.0)
    assert [tf._workspace(dev, head, b) for b in (0, 1) for dev in (1, 0, 1)] == [2000, 1000, 2000, 2001, 1001, 2001]
    tf._workspace.cache_clear()


@pytest.mark.parametrize("items,rows", [(1, 0x7FFFFFFF), (0x7FFFFFFF, 1), (1, 0x7FFFFFFF - 12)])
def test_resnorm_refuses_rows_whose_numbers_would_pass_32_bits(items, rows):
    """A block adds as many rows as it takes at a time to a row's number."""
    assert resnorm("workspace", items=items, rows=rows, cols=1, xs=1, fs=1) == SHAPE
    assert resnorm("workspace", items=1, rows=0x7FFFFF00, cols=1, xs=1, fs=1) > 0


def test_act8_backward_refuses_what_is_no_kept_form():
    """Scales that do not go with the values would be read past their end."""
    q, scale = torch.zeros(4, 300, dtype=torch.int8), torch.zeros(4, 3)
    kept = tf.Kept8(q, scale, "gelu", 0.0, torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        tf.act8_backward(None, kept)  # a kept form, on the wrong device
    for bad in (dict(scale=scale[:3]), dict(scale=scale[:, :2]), dict(scale=scale.double()), dict(q=q.float()), dict(q=q[0]),
                dict(q=q[:, :128]), dict(dtype=torch.float64), dict(q=q[0, 0])):
        with pytest.raises(ValueError, match="not a kept form"):
            tf.act8_backward(None, kept._replace(**bad))
    with pytest.raises(ValueError, match="act is one of"):
        tf.act8_backward(None, kept._replace(act="tanh"))


def test_sizes_beyond_32_bits_are_refused(monkeypatch):
    """2^32 + 64 columns are not 64; what the library is called with is recorded, not called."""
    calls = []
    monkeypatch.setattr(tf, "_cuda", lambda what, *ts: 0)
    monkeypatch.setattr(tf, "_call", lambda *args: calls.append(args))
    big = 2 ** 32 + 64
    empty = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="meta")  # noqa: E731
    kept = tf.Kept8(empty(1, big, dtype=torch.int8), empty(1, -(-big // 128), dtype=torch.float32), "gelu", 0.0, torch.bfloat16)
    for call in (lambda: tf.act8_forward(empty(1, big)), lambda: tf.act8_backward(None, kept),
                 lambda: tf.resnorm_forward(empty(1, 1, big), empty(1, 1, big)),
                 lambda: tf.attention_forward(*(empty(1, big, 1, 64),) * 3)):
        with pytest.raises(ValueError, match="beyond 32 bits"):
            call()
    assert not calls
    for cols in (0x7FFFFFFF, 0x7FFFFFFF - 130):  # to the end of a block they would pass 32 bits
        assert act8(cols=cols, rows=1) == SHAPE and act8("backward", cols=cols, rows=1) == SHAPE


@pytest.mark.parametrize("device,want", [(None, 3), ("cuda", 3), (torch.device("cuda"), 3), ("cuda:0", 0), ("cuda:1", 1), (2, 2)])
def test_ops_sync_waits_on_the_device_it_is_given(device, want, monkeypatch):
    calls = []
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    monkeypatch.setattr(tf, "_call", lambda what, fn, dev: calls.append(dev))
    tf.ops_sync(device)
    assert calls == [want]
