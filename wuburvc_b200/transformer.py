"""Transformer training operators on the native library (section 4 of include/wuburvc_b200.h), for
torch CUDA tensors: what the layers of a self-attention encoder in front of the generator are made of,
besides their matrix products.

* ``act8_forward`` / ``act8_backward``: an activation whose input is kept in 8 bits for the backward;
* ``resnorm_forward`` / ``resnorm_backward``: the norms around a block, its gate and the residual scale;
* ``attention_forward`` / ``attention_backward``: softmax attention, its gradient with the probabilities
  recomputed from the log-sum-exp;
* ``attention``, ``resnorm``, ``feed_forward``: the same for torch's autograd, differentiable once (a second
  derivative raises).

Calls enqueue on the current torch stream of the tensors' device and do not synchronise; outputs are new
tensors.  A call that cannot be made raises (``ValueError`` for its arguments, ``RuntimeError`` for a
code of the library); there is no fallback to torch.  Last dimensions are contiguous (others are copied
first); ``ops_sync`` reports what an asynchronous call could not.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from ._lib import lib

_vp, _ip, _fp, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_longlong
_SIGS = {
    "wubu_b200_ops_sync": (_ip, [_vp]),
    "wubu_b200_act8_forward": (_ip, [_ip, _ip, _fp, _vp, _ll, _vp, _vp, _vp, _ll, _ip, _vp]),
    "wubu_b200_act8_backward": (_ip, [_ip, _ip, _fp, _vp, _ll, _vp, _vp, _vp, _vp, _ll, _ip, _vp]),
    "wubu_b200_resnorm_forward": (_ip, [ctypes.c_char_p, _vp]),
    "wubu_b200_resnorm_workspace": (_ll, [ctypes.c_char_p]),
    "wubu_b200_resnorm_backward": (_ip, [ctypes.c_char_p, _vp]),
    "wubu_b200_attn_workspace": (_ll, [ctypes.c_char_p, _ip]),
    "wubu_b200_attn_forward": (_ip, [ctypes.c_char_p, _vp]),
    "wubu_b200_attn_backward": (_ip, [ctypes.c_char_p, _vp]),
}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"identity": 0, "lrelu": 1, "gelu": 2, "silu": 3, "lrelu_sign": 4}
_NORMS = {None: 0, "layer": 1, "rms": 2}
ACT8_BLOCK = 128
_bound = None


def L():
    global _bound
    if _bound is None:
        h = lib()
        for name, (res, args) in _SIGS.items():
            f = getattr(h, name)
            f.restype = res
            f.argtypes = args
        _bound = h
    return _bound


def _check(rc, what):
    if rc < 0:
        raise RuntimeError(f"wuburvc_b200 {what} failed with code {rc}")
    return rc


def _dtype(t, what):
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise ValueError(f"{what}: float32, bfloat16 or float16 tensors, got {t.dtype}")
    return d


def _cuda(what, *ts):
    """The index of the device that all of ``ts`` (None left out) are on."""
    dev = ts[0].get_device()
    if dev < 0:
        raise ValueError(f"{what}: CUDA tensors only")
    for t in ts[1:]:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"{what}: tensors on cuda:{dev} and {t.device}")
    return dev


# the current stream's handle without a torch.cuda.Stream object around it, where torch has that
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda dev: torch.cuda.current_stream(dev).cuda_stream)


def _int32(what, n):
    """n, a size that the library takes in 32 bits (ctypes would cut it, struct raises an error of its own)."""
    if n > 2 ** 31 - 1:
        raise ValueError(f"{what}: a size of {n} is beyond 32 bits")
    return n


def _on(dev, fn, *args):
    """fn(*args) with dev current (the library asks and launches on the current device)."""
    if dev == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _call(what, fn, dev, *args):
    """fn(*args, current stream of dev) with dev current."""
    if dev == torch.cuda.current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        _check(rc, what)


def _empty(like, dtype=None):
    """A contiguous tensor of like's shape."""
    if like.is_contiguous():
        return torch.empty_like(like, dtype=dtype)
    return like.new_empty(like.shape, dtype=dtype)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _rows(t):
    """(t, row stride) of a tensor seen as rows of its last dimension: a view where one row stride
    describes it, else a copy."""
    C = t.shape[-1]
    if t.is_contiguous():
        return t, C
    if t.dim() and t.stride(-1) == 1 or C == 1:
        step = None
        want = None
        for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if n == 1:
                continue
            if step is None:
                step, want = s, s * n
            elif s != want:
                step = None
                break
            else:
                want = s * n
        if step is not None and step >= C and (C == 1 or t.stride(-1) == 1):
            return t, step
    t = t.contiguous()
    return t, C


def ops_sync(device=None):
    """Waits for the current stream and raises if a kernel of these operators gave up on a wait."""
    dev = None if device is None else torch.device(device).index
    dev = torch.cuda.current_device() if dev is None else dev
    _call("ops_sync", L().wubu_b200_ops_sync, dev)


# ---- activation with an 8-bit checkpoint of its input --------------------------------------------


class Kept8(NamedTuple):
    """What ``act8_forward`` keeps of its input: int8 values and a scale per 128 values of a row."""

    q: torch.Tensor
    scale: torch.Tensor
    act: str
    slope: float
    dtype: torch.dtype


def act8_forward(x, act="gelu", slope=0.0, with_output=True):
    """``(act(x), kept)``; ``kept`` is what ``act8_backward`` reads in place of x.  ``act``: "gelu", "silu",
    "identity", or a leaky ReLU with ``slope`` (0: the ReLU) in one of two forms.  "lrelu_sign" keeps positive values
    positive: its derivatives are those of x.  "lrelu" rounds like the others and differentiates at the rounded
    value: what lies within half a step above 0 has the slope's derivative (0.5 % of normally distributed
    values, a tenth of the gradient's norm).  ``with_output=False`` only keeps x."""
    d = _dtype(x, "act8_forward")
    if act not in _ACTS:
        raise ValueError(f"act8_forward: act is one of {sorted(_ACTS)}, got {act!r}")
    if x.dim() < 1:
        raise ValueError("act8_forward: x has a last dimension")
    dev = _cuda("act8_forward", x)
    x, step = _rows(x)
    C = _int32("act8_forward", x.shape[-1])
    rows = x.numel() // C if C else 0
    y = _empty(x) if with_output else None
    q = _empty(x, torch.int8)
    scale = x.new_empty((*x.shape[:-1], -(-C // ACT8_BLOCK)), dtype=torch.float32)
    _call("act8_forward", L().wubu_b200_act8_forward, dev, d, _ACTS[act], slope, x.data_ptr(), step, _ptr(y),
          q.data_ptr(), scale.data_ptr(), rows, C)
    return y, Kept8(q, scale, act, float(slope), x.dtype)


def act8_backward(dy, kept, recompute=False):
    """``(dx, y)`` from the kept form x' of x: dx = dy act'(x'); y = act(x') if ``recompute``, else
    None.  ``dy=None`` gives ``(None, act(x'))`` alone."""
    q, scale = kept.q, kept.scale
    shape, blocks, d, act = q.shape, scale.shape, _DTYPES.get(kept.dtype), _ACTS.get(kept.act)
    if (not shape or q.dtype != torch.int8 or scale.dtype != torch.float32 or d is None or blocks[:-1] != shape[:-1]
            or len(blocks) != len(shape) or blocks[-1] != -(-shape[-1] // ACT8_BLOCK)):
        raise ValueError(f"act8_backward: not a kept form: q {tuple(shape)} {q.dtype}, scale {tuple(blocks)} "
                         f"{scale.dtype}, of {kept.dtype}")
    if act is None:
        raise ValueError(f"act8_backward: act is one of {sorted(_ACTS)}, got {kept.act!r}")
    if not (q.is_contiguous() and scale.is_contiguous()):  # parts of a kept form may be strided
        q, scale = q.contiguous(), scale.contiguous()
    if dy is not None and (dy.shape != shape or dy.dtype != kept.dtype):
        raise ValueError(f"act8_backward: dy is {tuple(shape)} {kept.dtype}, got {tuple(dy.shape)} {dy.dtype}")
    dev = _cuda("act8_backward", q, scale, dy)
    C = _int32("act8_backward", shape[-1])
    rows = q.numel() // C if C else 0
    step, dx, y = 0, None, None
    if dy is not None:
        dy, step = _rows(dy)
        dx = torch.empty_like(q, dtype=kept.dtype)
    if recompute or dy is None:
        y = torch.empty_like(q, dtype=kept.dtype)
    _call("act8_backward", L().wubu_b200_act8_backward, dev, d, act, kept.slope, _ptr(dy),
          step, q.data_ptr(), scale.data_ptr(), _ptr(dx), _ptr(y), rows, C)
    return dx, y


def act8_restore(kept):
    """The kept form of x itself, in x's type."""
    return act8_backward(None, kept._replace(act="identity"), recompute=True)[1]


# ---- norms around a block, gate and residual scale ------------------------------------------------

_RESNORM_GRADS = frozenset(("dx", "df", "dgate", "dweight", "dbias", "dpost_weight", "dpost_bias"))
_RESNORM = struct.Struct("@4i2qi2fi" + "4q" + "4P" + "P" + "2P" + "4q" + "2P" + "5P" + "Pq")


def _vector(v, shape, dev, what):
    if v is None:
        return None
    if v.shape != shape:
        raise ValueError(f"{what}: shape {shape}, got {tuple(v.shape)}")
    if v.get_device() != dev:
        raise ValueError(f"{what}: tensors on cuda:{dev} and {v.device}")
    if v.dtype != torch.float32 or not v.is_contiguous():
        v = v.to(torch.float32).contiguous()
    return v


def _resnorm_operands(what, x, f, norm, weight, bias, post, post_weight, post_bias, gate):
    if x.dim() < 2 or f.shape != x.shape or f.dtype != x.dtype:
        raise ValueError(f"{what}: x and f are [items, ..., cols] of one shape and type")
    if norm not in _NORMS or post not in _NORMS:
        raise ValueError(f"{what}: norm and post are None, 'layer' or 'rms'")
    if (bias is not None and norm != "layer") or (post_bias is not None and post != "layer"):
        raise ValueError(f"{what}: only a layer norm has a bias")
    if (weight is not None and norm is None) or (post_weight is not None and post is None):
        raise ValueError(f"{what}: a weight without its norm")
    dev = _cuda(what, x, f)
    items, C = x.shape[0], _int32(what, x.shape[-1])
    rows = x.numel() // (items * C) if items and C else 0
    vec = [v if v is None else _vector(v, (C,), dev, what) for v in (weight, bias, post_weight, post_bias)]
    kind = 0
    if gate is not None:
        kind = 1 if gate.dim() == 1 else 2
        gate = _vector(gate, (C,) if kind == 1 else (items, C), dev, what)
    return dev, items, rows, C, vec, kind, gate


def resnorm_forward(x, f, *, norm="layer", weight=None, bias=None, post=None, post_weight=None, post_bias=None,
                    gate=None, res_scale=1.0, eps=1e-5, keep_sum=True):
    """``(r, h)`` with r = res_scale * x + gate * post(f) and h = norm(r), for x, f ``[items, ..., cols]``.

    ``norm`` / ``post``: "layer", "rms" or None, with ``weight`` / ``bias`` and ``post_weight`` /
    ``post_bias`` of ``[cols]`` (None: ones / zeros; RMS norms have no bias).  ``gate``: None,
    ``[cols]`` or ``[items, cols]``.  ``keep_sum=False`` returns None for r; ``norm=None`` None for h."""
    d = _dtype(x, "resnorm_forward")
    dev, items, rows, C, vec, kind, gate = _resnorm_operands("resnorm_forward", x, f, norm, weight, bias, post,
                                                             post_weight, post_bias, gate)
    x, xs = _rows(x)
    f, fs = _rows(f)
    r = _empty(x) if keep_sum else None
    h = _empty(x) if norm else None
    args = _RESNORM.pack(d, _NORMS[norm], _NORMS[post], kind, items, rows, C, res_scale, eps, 0, x.data_ptr(), xs,
                         f.data_ptr(), fs, *map(_ptr, vec), _ptr(gate), _ptr(r), _ptr(h), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                         0, 0, 0)
    _call("resnorm_forward", L().wubu_b200_resnorm_forward, dev, args)
    return r, h


def resnorm_backward(dr, dh, x, f, *, norm="layer", weight=None, bias=None, post=None, post_weight=None,
                     post_bias=None, gate=None, res_scale=1.0, eps=1e-5, need=None):
    """Gradients of ``resnorm_forward`` for the gradients ``dr`` of r and ``dh`` of h (either may be
    None): a dict of dx, df, dgate, dweight, dbias, dpost_weight, dpost_bias, None for what the
    operator was not given, or what ``need`` (names of the dict; None: all) leaves out.  The vectors' gradients are
    float32 sums over the rows."""
    what = "resnorm_backward"
    d = _dtype(x, what)
    dev, items, rows, C, vec, kind, gate = _resnorm_operands(what, x, f, norm, weight, bias, post, post_weight,
                                                             post_bias, gate)
    strides = [0, 0]
    grads = [dr, dh]
    for i, t in enumerate(grads):
        if t is None:
            continue
        if t.shape != x.shape or t.dtype != x.dtype or t.get_device() != dev:
            raise ValueError(f"{what}: dr and dh have x's shape, type and device")
        grads[i], strides[i] = _rows(t)
    if dr is None and dh is None:
        raise ValueError(f"{what}: dr or dh is needed")
    if dh is not None and norm is None:
        raise ValueError(f"{what}: dh without a norm")
    dr, dh = grads
    x, xs = _rows(x)
    f, fs = _rows(f)
    skip = () if need is None else _RESNORM_GRADS.difference(need)
    dx = None if "dx" in skip else _empty(x)
    df = None if "df" in skip else _empty(x)
    dweight, dbias, dpost_weight, dpost_bias = (None if v is None or n in skip else torch.empty_like(v) for n, v in
                                                zip(("dweight", "dbias", "dpost_weight", "dpost_bias"), vec))
    dgate = None if gate is None or "dgate" in skip else torch.empty_like(gate)

    def pack(ws, n):
        return _RESNORM.pack(d, _NORMS[norm], _NORMS[post], kind, items, rows, C, res_scale, eps, 0, x.data_ptr(), xs,
                             f.data_ptr(), fs, *map(_ptr, vec), _ptr(gate), 0, 0, _ptr(dr), strides[0], _ptr(dh),
                             strides[1], _ptr(dx), _ptr(df), _ptr(dgate), _ptr(dpost_weight), _ptr(dpost_bias),
                             _ptr(dweight), _ptr(dbias), ws, n)

    h = L()
    n = _check(_on(dev, h.wubu_b200_resnorm_workspace, pack(0, 0)), what)
    ws = x.new_empty(n, dtype=torch.uint8)
    _call(what, h.wubu_b200_resnorm_backward, dev, pack(ws.data_ptr(), n))
    return {"dx": dx, "df": df, "dgate": dgate, "dweight": dweight, "dbias": dbias, "dpost_weight": dpost_weight,
            "dpost_bias": dpost_bias}


# ---- attention --------------------------------------------------------------------------------------

_ATTN = struct.Struct("@9if2P" + "P3q" * 4 + "P" + "P3q" * 4 + "Pq")
_NO_VIEW = (0, 0, 0, 0)


def _view(t):
    """(t, (address, batch, token, head strides)): t itself where the library can address it (contiguous
    last dimension, 16-byte aligned rows), else a copy."""
    sb, st, sh, sd = t.stride()
    B, T, H, D = t.shape
    if (sd != 1 or t.data_ptr() & 15 or (B > 1 and (sb % 8 or sb < D)) or (T > 1 and (st % 8 or st < D))
            or (H > 1 and (sh % 8 or sh < D))):
        t = t.contiguous()
        if t.data_ptr() & 15:
            t = t.clone()
        sb, st, sh, _ = t.stride()
    return t, (t.data_ptr(), sb, st, sh)


def _lens(n, B, dev, what):
    if n is None:
        return None
    if n.shape != (B,) or n.get_device() != dev:
        raise ValueError(f"{what}: lengths are [{B}] on cuda:{dev}, got {tuple(n.shape)} on {n.device}")
    if n.dtype != torch.int32 or not n.is_contiguous():
        n = n.to(torch.int32).contiguous()
    return n


def _attn_operands(what, q, k, v, causal, window, scale, q_lens, k_lens):
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"{what}: q is [B, Tq, Hq, D], k and v are [B, Tk, Hkv, D]")
    B, Tq, Hq, D = q.shape
    Bk, Tk, Hkv, Dk = k.shape
    if B != Bk or D != Dk or (Hq % Hkv if Hkv else Hq):
        raise ValueError(f"{what}: q {tuple(q.shape)} does not go with k {tuple(k.shape)}")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"{what}: D is a multiple of 8 from 8 to 128, got {D}")
    d = _DTYPES.get(q.dtype)
    if d is None or d == 0 or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{what}: bfloat16 or float16 tensors of one type")
    if window < 0 or (scale is not None and not 0.0 < scale < float("inf")):
        raise ValueError(f"{what}: window is not negative, scale is positive")
    dev = _cuda(what, q, k, v)
    ql, kl = _lens(q_lens, B, dev, what), _lens(k_lens, B, dev, what)
    _int32(what, max(B, Hq, Tq, Tk))
    head = (d, B, Hq, Hkv, Tq, Tk, D, int(bool(causal)), min(int(window), 2 ** 30), scale or 0.0)
    return dev, head, (_ptr(ql), _ptr(kl)), (ql, kl)


@functools.lru_cache(maxsize=1024)
def _workspace(dev, head, backward):
    """Workspace bytes of a call's sizes on a device (the library's answer depends on those and on its SMs)."""
    args = _ATTN.pack(*head, 0, 0, *_NO_VIEW * 4, 0, *_NO_VIEW * 4, 0, 0)
    return _check(_on(dev, L().wubu_b200_attn_workspace, args, backward), "attn_workspace")


def attention_forward(q, k, v, *, causal=False, window=0, scale=None, q_lens=None, k_lens=None):
    """``(out, lse)``: softmax(scale q k^T) v over the visible keys, and the float32 log-sum-exp [B, Hq, Tq].

    q ``[B, Tq, Hq, D]``, k and v ``[B, Tk, Hkv, D]`` (Hq a multiple of Hkv: query head h reads key head
    h * Hkv // Hq); ``scale`` defaults to 1 / sqrt(D).  ``q_lens`` / ``k_lens``: int32 ``[B]`` on the device,
    the lengths of padded items (what lies beyond may hold anything).  Query i sits at place
    p = i + k_len - q_len among the keys and sees key j if j < k_len, j <= p (``causal``) and
    |p - j| < window (``window`` > 0).  A query that sees nothing, or lies beyond q_len, has out 0 and lse -inf; one
    with a visible score that is NaN or +infinity has both NaN."""
    what = "attention_forward"
    dev, head, lens, hold = _attn_operands(what, q, k, v, causal, window, scale, q_lens, k_lens)
    q, vq = _view(q)
    k, vk = _view(k)
    v, vv = _view(v)
    B, Tq, Hq, D = q.shape
    out = _empty(q)
    lse = q.new_empty((B, Hq, Tq), dtype=torch.float32)
    body = (*head, *lens, *vq, *vk, *vv, out.data_ptr(), Tq * Hq * D, Hq * D, D, lse.data_ptr(), *_NO_VIEW * 4)
    h = L()
    n = _workspace(dev, head, 0)
    ws = q.new_empty(n, dtype=torch.uint8) if n else None
    _call(what, h.wubu_b200_attn_forward, dev, _ATTN.pack(*body, _ptr(ws), n))
    return out, lse


def attention_backward(dout, q, k, v, out, lse, *, causal=False, window=0, scale=None, q_lens=None, k_lens=None):
    """``(dq, dk, dv)`` for the gradient ``dout`` of ``attention_forward``'s out; ``out`` and ``lse`` are what it
    returned for the same arguments.  The gradients of shared heads are sums over the heads that share them."""
    what = "attention_backward"
    dev, head, lens, hold = _attn_operands(what, q, k, v, causal, window, scale, q_lens, k_lens)
    B, Tq, Hq, D = q.shape
    for t in (dout, out):
        if t.shape != q.shape or t.dtype != q.dtype or t.get_device() != dev:
            raise ValueError(f"{what}: dout and out have q's shape, type and device")
    if lse.shape != (B, Hq, Tq) or lse.dtype != torch.float32 or lse.get_device() != dev:
        raise ValueError(f"{what}: lse is float32 [B, Hq, Tq]")
    lse = lse.contiguous()
    (q, vq), (k, vk), (v, vv), (out, vo), (dout, vg) = map(_view, (q, k, v, out, dout))
    Tk, Hkv = k.shape[1:3]
    dq, dk, dv = _empty(q), _empty(k), _empty(v)
    sq, skv = (Tq * Hq * D, Hq * D, D), (Tk * Hkv * D, Hkv * D, D)
    body = (*head, *lens, *vq, *vk, *vv, *vo, lse.data_ptr(), *vg, dq.data_ptr(), *sq, dk.data_ptr(), *skv,
            dv.data_ptr(), *skv)
    n = _workspace(dev, head, 1)
    ws = q.new_empty(n, dtype=torch.uint8)
    _call(what, L().wubu_b200_attn_backward, dev, _ATTN.pack(*body, ws.data_ptr(), n))
    return dq, dk, dv


def _autocast(*ts, to=None):
    """Under torch.autocast, ``ts`` (None left out) in the type ``to``, by default autocast's, cast where autograd sees
    it; else as they are.  float64 is left alone, as torch leaves it."""
    kind = ts[0].device.type
    if not torch.is_autocast_enabled(kind):
        return ts
    to = to or torch.get_autocast_dtype(kind)
    return tuple(t if t is None or t.dtype not in _DTYPES else t.to(to) for t in ts)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lens, k_lens, opts):
        out, lse = attention_forward(q, k, v, q_lens=q_lens, k_lens=k_lens, **opts)
        # (the lengths among the saved tensors: changed in place before the backward, they raise there)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, k_lens)
        ctx.opts = opts
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        *saved, q_lens, k_lens = ctx.saved_tensors
        return (*attention_backward(dout, *saved, q_lens=q_lens, k_lens=k_lens, **ctx.opts), None, None, None)


def attention(q, k, v, *, q_lens=None, k_lens=None, **opts):
    """``attention_forward``'s out, differentiable by torch's autograd.  Under autocast in its type."""
    return _Attention.apply(*_autocast(q, k, v), q_lens, k_lens, opts)


class _ResNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, weight, bias, post_weight, post_bias, gate, opts, keep_sum):
        vec = dict(weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias, gate=gate)
        ctx.save_for_backward(x, f, *vec.values())
        ctx.opts = opts
        ctx.set_materialize_grads(False)
        return resnorm_forward(x, f, keep_sum=keep_sum, **vec, **opts)

    @staticmethod
    @once_differentiable
    def backward(ctx, dr, dh):
        x, f, *vec = ctx.saved_tensors
        if dr is None and dh is None:
            return (None,) * 9
        names = ("weight", "bias", "post_weight", "post_bias", "gate")
        need = [n for n, wanted in zip(("dx", "df", *("d" + n for n in names)), ctx.needs_input_grad) if wanted]
        g = resnorm_backward(dr, dh, x, f, **dict(zip(names, vec)), **ctx.opts, need=need)
        cast = [g["d" + n] if g["d" + n] is None else g["d" + n].to(v.dtype) for n, v in zip(names, vec)]
        return (g["dx"], g["df"], *cast, None, None)


def resnorm(x, f, *, weight=None, bias=None, post_weight=None, post_bias=None, gate=None, keep_sum=True, **opts):
    """``resnorm_forward``'s (r, h), differentiable by torch's autograd.  Only x and f are kept for the backward.  Under
    autocast x and f may differ in type: the wider one counts."""
    x, f = _autocast(x, f, to=torch.promote_types(x.dtype, f.dtype))
    return _ResNorm.apply(x, f, weight, bias, post_weight, post_bias, gate, opts, keep_sum)


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, act, slope):
        y, kept = act8_forward(torch.nn.functional.linear(x, w1, b1), act, slope=slope)
        ctx.save_for_backward(x, w1, w2, kept.q, kept.scale)
        ctx.kept = (kept.act, kept.slope, kept.dtype)
        return torch.nn.functional.linear(y, w2, b2)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, w1, w2, q, scale = ctx.saved_tensors
        act, slope, dtype = ctx.kept
        need_x, need_w1, need_b1, need_w2, need_b2 = ctx.needs_input_grad[:5]
        rows = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
        dx = dw1 = db1 = dw2 = db2 = None
        with torch.autocast(x.device.type, enabled=False):  # the saved tensors are in the forward's type
            inner = need_x or need_w1 or need_b1
            if inner or need_w2:
                du, y = act8_backward(dout @ w2 if inner else None, Kept8(q, scale, act, slope, dtype), recompute=need_w2)
            if need_x:
                dx = du @ w1
            if need_w1:
                dw1 = rows(du).T @ rows(x)
            if need_b1:
                db1 = rows(du).sum(0)
            if need_w2:
                dw2 = rows(dout).T @ rows(y)
            if need_b2:
                db2 = rows(dout).sum(0)
        return dx, dw1, db1, dw2, db2, None, None


def feed_forward(x, w1, b1, w2, b2, act="gelu", slope=0.0):
    """act(x w1^T + b1) w2^T + b2, differentiable.  Of its hidden layer the backward keeps the 8-bit form alone: the
    activation's derivative and the input of w2's gradient are both formed from it ("lrelu" in the form that keeps
    signs, so that the derivative is the function's own).  Under autocast in its type."""
    act = "lrelu_sign" if act == "lrelu" else act
    return _FeedForward.apply(*_autocast(x, w1, b1, w2, b2), act, slope)
