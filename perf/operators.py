"""Cases, plain forms and exact values of the transformer training operators.

Three operators that the training of a voice-conversion encoder (a self-attention content or prior
encoder in front of the generator) is made of:

* ``attn_fwd`` / ``attn_bwd``: softmax attention over ``[B, T, H, D]`` views with shared key / value
  heads, causal order, a sliding window and per-item lengths, and its gradient with the
  probabilities recomputed from the log-sum-exp;
* ``resnorm_fwd`` / ``resnorm_bwd``: ``r = a x + gate * post_norm(f)``, ``h = norm(r)``, and the
  gradients of everything that goes in;
* ``act8``: an activation whose input is kept in 8 bits for the backward pass (blocks of 128 values
  share a scale), the forward followed by the backward that reads it.

``own`` false: elementary torch operations in 32 bits, rounded once at the end.  ``own`` true: the
library's calls.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
BLOCK = 128  # values that share a scale in the 8-bit form
TINY = 2.0 ** -100  # a block whose largest magnitude is below this is held as zeros


# ---- cases --------------------------------------------------------------------------------------

def attn(op, B, Hq, Hkv, Tq, Tk, D, dtype, causal=False, window=0, ragged=False, **more):
    return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, Tq=Tq, Tk=Tk, D=D, dtype=dtype, causal=causal, window=window,
                ragged=ragged, **more)


def resnorm(op, B, T, C, dtype, post, gate, norm, res_scale=1.0, keep_sum=True, **more):
    return dict(op=op, B=B, T=T, C=C, dtype=dtype, post=post, gate=gate, norm=norm, res_scale=res_scale,
                keep_sum=keep_sum, **more)


def act8(B, T, C, dtype, act, slope=0.0, recompute=True, **more):
    return dict(op="act8", B=B, T=T, C=C, dtype=dtype, act=act, slope=slope, recompute=recompute, **more)


def listed():
    return [
        # one new frame of a streaming conversion against 30 s of context at 50 frames a second
        attn("attn_fwd", 1, 12, 12, 1, 1500, 64, "bf16", name="frame, 30 s of context"),
        # a training batch of the content encoder: 12 heads of 64, clips of up to 10 s, padded
        attn("attn_fwd", 16, 12, 12, 499, 499, 64, "bf16", ragged=True, name="content encoder batch"),
        # the 6000-frame clip in causal order, four query heads to a key head
        attn("attn_fwd", 1, 16, 4, 6000, 6000, 128, "bf16", causal=True, name="long causal clip"),
        # the prior encoder's attention (192 channels, 2 heads of 96) on one training segment
        attn("attn_bwd", 1, 2, 2, 32, 32, 96, "fp16", name="prior encoder segment, gradient"),
        # the content encoder's batch, backward
        attn("attn_bwd", 16, 12, 12, 499, 499, 64, "bf16", ragged=True, name="content encoder, gradient"),
        # a long causal training sequence of odd length, four query heads to a key head
        attn("attn_bwd", 1, 16, 4, 4001, 4001, 128, "bf16", causal=True, name="long causal, gradient"),
        # the prior encoder's LayerNorm(x + f) on one segment: latency
        resnorm("resnorm_fwd", 1, 32, 192, "bf16", None, None, "layer", keep_sum=False, name="segment norm"),
        # a gated block of a 768-wide encoder: norm, gate per item, residual, next block's norm
        resnorm("resnorm_fwd", 16, 499, 768, "bf16", "rms", "item", "rms", name="gated block"),
        # the long clip at 768 channels, LayerNorm of the sum, backward
        resnorm("resnorm_bwd", 1, 6000, 768, "fp16", None, None, "layer", keep_sum=False, name="long norm, gradient"),
        # the gated block's backward
        resnorm("resnorm_bwd", 16, 499, 768, "bf16", "rms", "item", "rms", name="gated block, gradient"),
        # the prior encoder's feed-forward (768 wide, ReLU) on one segment
        act8(1, 32, 768, "bf16", "lrelu", name="segment feed-forward"),
        # feed-forward of a wide encoder over a training batch of 10 s clips
        act8(16, 499, 2048, "bf16", "gelu", name="wide feed-forward"),
    ]


def log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn_fwd", "attn_bwd", "resnorm_fwd", "resnorm_bwd", "act8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op.startswith("attn"):
        D = rng.choice([64, 64, 96, 128, 32, 80])
        group = rng.choice([1, 1, 1, 2, 4])
        Hkv = rng.choice([1, 2, 3, 4, 8, 12])
        B = log_int(rng, 1, 16)
        Tk = log_int(rng, 1, 5000)
        single = op == "attn_fwd" and rng.random() < 0.25
        Tq = rng.randint(1, 3) if single else Tk
        while B * Hkv * group * Tq * Tk > 2.0e8:
            if B > 1:
                B = B // 2
            elif Hkv > 1:
                Hkv = Hkv // 2
            else:
                group = group // 2
        causal = rng.random() < 0.5
        window = log_int(rng, 16, 512) if rng.random() < 0.2 else 0
        return attn(op, B, Hkv * group, Hkv, Tq, Tk, D, dtype, causal=causal, window=window,
                    ragged=rng.random() < 0.5)
    if op == "act8":
        act = rng.choice(["gelu", "silu", "lrelu"])
        return act8(log_int(rng, 1, 16), log_int(rng, 1, 499), log_int(rng, 64, 2048), dtype, act,
                    slope=rng.choice([0.0, 0.1]) if act == "lrelu" else 0.0, recompute=rng.random() < 0.7)
    dtype = rng.choice([dtype, dtype, "fp32"])
    return resnorm(op, log_int(rng, 1, 16), log_int(rng, 1, 499), log_int(rng, 64, 768), dtype,
                   rng.choice([None, "layer", "rms"]), rng.choice([None, "channel", "item"]),
                   rng.choice(["layer", "rms"]), res_scale=rng.choice([1.0, 0.5]), keep_sum=rng.random() < 0.7)


def lengths(case, T):
    """The lengths of a padded batch: the first item is whole, the last about a quarter of it."""
    B = case["B"]
    return [max(1, T - (3 * b * T) // (4 * B)) for b in range(B)]


# ---- what a user has in hand --------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt, std=1.0, mean=0.0):
        x = torch.randn(*shape, generator=g, device="cuda")
        return (x * std + mean).to(dtype)

    s = dict(case)
    if case["op"].startswith("attn"):
        B, Hq, Hkv, Tq, Tk, D = (case[n] for n in ("B", "Hq", "Hkv", "Tq", "Tk", "D"))
        s["q"] = normal(B, Tq, Hq, D)
        kv = normal(B, Tk, 2, Hkv, D)  # one projection makes both: strided views of it
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["q_lens"] = s["k_lens"] = None
        if case["ragged"]:
            s["k_lens"] = torch.tensor(lengths(case, Tk), dtype=torch.int32, device="cuda")
            if Tq == Tk:
                s["q_lens"] = s["k_lens"]
        if case["op"] == "attn_bwd":
            s["dout"] = normal(B, Tq, Hq, D, std=0.1)
            s["out"], s["lse"] = plain_attention(s)
        return s
    B, T, C = case["B"], case["T"], case["C"]
    if case["op"] == "act8":
        s["x"] = normal(B, T, C, std=1.5)
        s["dy"] = normal(B, T, C, std=0.1)
        return s
    f32 = torch.float32
    s["x"], s["f"] = normal(B, T, C), normal(B, T, C, std=0.7)
    s["post_weight"] = normal(C, dtype=f32, std=0.1, mean=1.0) if case["post"] else None
    s["post_bias"] = normal(C, dtype=f32, std=0.1) if case["post"] == "layer" else None
    s["gate_values"] = {None: lambda: None, "channel": lambda: normal(C, dtype=f32, std=0.5),
                        "item": lambda: normal(B, C, dtype=f32, std=0.5)}[case["gate"]]()
    s["weight"] = normal(C, dtype=f32, std=0.1, mean=1.0)
    s["bias"] = normal(C, dtype=f32, std=0.1) if case["norm"] == "layer" else None
    if case["op"] == "resnorm_bwd":
        s["dh"] = normal(B, T, C, std=0.1)
        s["dr"] = normal(B, T, C, std=0.1) if case["keep_sum"] else None
    return s


# ---- plain forms ---------------------------------------------------------------------------------

def visible(s):
    """[B or 1, 1, Tq, Tk] truth values: which keys a query sees; None where all do."""
    Tq, Tk = s["Tq"], s["Tk"]
    if not (s["causal"] or s["window"] or s["ragged"]):
        return None
    i = torch.arange(Tq, device="cuda").view(1, 1, Tq, 1)
    j = torch.arange(Tk, device="cuda").view(1, 1, 1, Tk)
    ql = Tq if s["q_lens"] is None else s["q_lens"].view(-1, 1, 1, 1)
    kl = Tk if s["k_lens"] is None else s["k_lens"].view(-1, 1, 1, 1)
    at = i + (kl - ql)  # a query's place among the keys: the last query sits at the last key
    see = (i < ql) & (j < kl)
    if s["causal"]:
        see = see & (j <= at)
    if s["window"]:
        see = see & (at - j < s["window"]) & (j - at < s["window"])
    return see


def scores(s):
    q = s["q"].float().transpose(1, 2)
    k = s["k"].float().transpose(1, 2)
    group = s["Hq"] // s["Hkv"]
    k = k.repeat_interleave(group, 1) if group > 1 else k
    x = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(s["D"]))
    see = visible(s)
    return (x if see is None else x.masked_fill(~see, -math.inf)), q, k


def plain_attention(s):
    x, _, _ = scores(s)
    v = s["v"].float().transpose(1, 2)
    group = s["Hq"] // s["Hkv"]
    v = v.repeat_interleave(group, 1) if group > 1 else v
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    p = torch.exp(x - m)
    total = p.sum(-1, keepdim=True)
    lse = torch.where(total > 0, m + torch.log(total), torch.full_like(total, -math.inf)).squeeze(-1)
    out = (p @ v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.transpose(1, 2).to(s["q"].dtype).contiguous(), lse


def plain_attention_backward(s):
    x, q, k = scores(s)
    v = s["v"].float().transpose(1, 2)
    group = s["Hq"] // s["Hkv"]
    v = v.repeat_interleave(group, 1) if group > 1 else v
    do = s["dout"].float().transpose(1, 2)
    lse = s["lse"].unsqueeze(-1)
    p = torch.exp(x - torch.where(lse == -math.inf, torch.zeros_like(lse), lse))
    dv = p.transpose(2, 3) @ do
    dp = do @ v.transpose(2, 3)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * (1.0 / math.sqrt(s["D"]))
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    if group > 1:
        dk, dv = (t.unflatten(1, (s["Hkv"], group)).sum(2) for t in (dk, dv))
    return tuple(t.transpose(1, 2).to(s["q"].dtype).contiguous() for t in (dq, dk, dv))


def normalised(x, kind):
    """(x normalised over its last axis, 1 / its standard deviation or root mean square)"""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    inv = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return x * inv, inv


def normalised_backward(g, n, inv, kind):
    """The gradient of `normalised` for the gradient g of its value n."""
    d = g - n * (g * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * inv


def affine(n, w, b):
    return n * w if b is None else n * w + b


def gate_of(s):
    gv = s["gate_values"]
    return gv if gv is None or gv.dim() == 1 else gv.unsqueeze(1)


def plain_resnorm(s):
    x, u, gate = s["x"].float(), s["f"].float(), gate_of(s)
    if s["post"]:
        u = affine(normalised(u, s["post"])[0], s["post_weight"], s["post_bias"])
    r = s["res_scale"] * x + (u if gate is None else gate * u)
    h = affine(normalised(r, s["norm"])[0], s["weight"], s["bias"]).to(s["x"].dtype)
    return {"r": r.to(s["x"].dtype) if s["keep_sum"] else None, "h": h}


def plain_resnorm_backward(s):
    x, f, gate, dh = s["x"].float(), s["f"].float(), gate_of(s), s["dh"].float()
    n, inv = normalised(f, s["post"]) if s["post"] else (f, None)
    u = affine(n, s["post_weight"], s["post_bias"]) if s["post"] else f
    r = s["res_scale"] * x + (u if gate is None else gate * u)
    rn, rinv = normalised(r, s["norm"])
    rows = (0, 1)
    out = {"dweight": (dh * rn).sum(rows), "dbias": dh.sum(rows) if s["bias"] is not None else None}
    dr = normalised_backward(dh * s["weight"], rn, rinv, s["norm"])
    if s["dr"] is not None:
        dr = dr + s["dr"].float()
    out["dx"] = (s["res_scale"] * dr).to(s["x"].dtype)
    out["dgate"] = None if gate is None else (dr * u).sum(rows if s["gate"] == "channel" else 1)
    du = dr if gate is None else dr * gate
    out["dpost_weight"] = (du * n).sum(rows) if s["post"] else None
    out["dpost_bias"] = du.sum(rows) if s["post_bias"] is not None else None
    df = normalised_backward(du * s["post_weight"], n, inv, s["post"]) if s["post"] else du
    out["df"] = df.to(s["f"].dtype)
    return out


def activation(x, act, slope):
    if act == "lrelu":
        return torch.where(x > 0, x, slope * x)
    if act == "silu":
        return x / (1.0 + torch.exp(-x))
    return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))


def activation_slope(x, act, slope):
    if act == "lrelu":
        return torch.where(x > 0, torch.ones_like(x), torch.full_like(x, slope))
    if act == "silu":
        t = 1.0 / (1.0 + torch.exp(-x))
        return t * (1.0 + x * (1.0 - t))
    return 0.5 * (1.0 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) * (1.0 / math.sqrt(2 * math.pi))


def held_in_8_bits(x):
    """What the 8-bit form of x stands for: whole multiples of a scale per block of a row."""
    C = x.shape[-1]
    b = torch.nn.functional.pad(x, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    none = top < TINY
    # tensor by tensor: a number divided by a tensor would be its reciprocal times the number, rounded twice
    inv = torch.where(none, torch.zeros_like(top), torch.full_like(top, 127.0) / torch.where(none, torch.ones_like(top), top))
    scale = torch.where(none, torch.zeros_like(top), top / 127.0)
    return (torch.round(b * inv) * scale).flatten(-2)[..., :C]


def plain_act8(s):
    x, dt = s["x"].float(), s["x"].dtype
    y = activation(x, s["act"], s["slope"]).to(dt)
    kept = held_in_8_bits(x)
    out = {"y": y, "dx": (s["dy"].float() * activation_slope(kept, s["act"], s["slope"])).to(dt)}
    if s["recompute"]:
        out["y_again"] = activation(kept, s["act"], s["slope"]).to(dt)
    return out


# ---- one pass ------------------------------------------------------------------------------------

def run(s):
    op = s["op"]
    if not own:
        return {"attn_fwd": plain_attention, "attn_bwd": plain_attention_backward, "resnorm_fwd": plain_resnorm,
                "resnorm_bwd": plain_resnorm_backward, "act8": plain_act8}[op](s)
    from wuburvc_b200 import transformer as tf

    if op == "attn_fwd":
        return tf.attention_forward(s["q"], s["k"], s["v"], causal=s["causal"], window=s["window"],
                                    q_lens=s["q_lens"], k_lens=s["k_lens"])
    if op == "attn_bwd":
        return tf.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], causal=s["causal"],
                                     window=s["window"], q_lens=s["q_lens"], k_lens=s["k_lens"])
    if op == "resnorm_fwd":
        r, h = tf.resnorm_forward(s["x"], s["f"], norm=s["norm"], weight=s["weight"], bias=s["bias"], post=s["post"],
                                  post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate_values"],
                                  res_scale=s["res_scale"], eps=EPS, keep_sum=s["keep_sum"])
        return {"r": r, "h": h}
    if op == "resnorm_bwd":
        return tf.resnorm_backward(s["dr"], s["dh"], s["x"], s["f"], norm=s["norm"], weight=s["weight"],
                                   bias=s["bias"], post=s["post"], post_weight=s["post_weight"],
                                   post_bias=s["post_bias"], gate=s["gate_values"], res_scale=s["res_scale"],
                                   eps=EPS)
    y, kept = tf.act8_forward(s["x"], s["act"], slope=s["slope"])
    dx, again = tf.act8_backward(s["dy"], kept, recompute=s["recompute"])
    out = {"y": y, "dx": dx}
    if s["recompute"]:
        out["y_again"] = again
    return out


# ---- work ----------------------------------------------------------------------------------------

def pairs(case):
    """Visible (query, key) pairs of one head, over the batch."""
    Tq, Tk, w = case["Tq"], case["Tk"], case["window"]
    total = 0
    kls = lengths(case, Tk) if case["ragged"] else [Tk] * case["B"]
    for kl in kls:
        ql = kl if case["ragged"] and Tq == Tk else Tq
        if not case["causal"] and not w:
            total += ql * kl
            continue
        for i in range(ql):
            at = i + kl - ql
            lo = max(0, at - w + 1) if w else 0
            hi = min(kl, at + 1) if case["causal"] else (min(kl, at + w) if w else kl)
            total += max(0, hi - lo)
    return total


def work(case):
    b = BYTES[case["dtype"]]
    if case["op"].startswith("attn"):
        Tk, D = case["Tk"], case["D"]
        keys = sum(lengths(case, Tk)) if case["ragged"] else case["B"] * Tk
        rows = keys if case["ragged"] and case["Tq"] == Tk else case["B"] * case["Tq"]
        q, kv = rows * case["Hq"] * D * b, keys * case["Hkv"] * D * b
        flops = 2.0 * pairs(case) * case["Hq"] * D
        lse = 4 * rows * case["Hq"]
        if case["op"] == "attn_fwd":
            return {"bytes": 2 * q + 2 * kv + lse, "flops": 2 * flops}
        return {"bytes": 4 * q + 4 * kv + lse, "flops": 5 * flops}
    B, C = case["B"], case["C"]
    n = B * case["T"] * C
    if case["op"] == "act8":
        held = n + 4 * B * case["T"] * (-(-C // BLOCK))
        return {"bytes": n * b * (4 + (1 if case["recompute"] else 0)) + 2 * held, "flops": 20.0 * n}
    vectors = 4 * C * (1 + (case["norm"] == "layer") + bool(case["post"]) + (case["post"] == "layer"))
    vectors += 4 * C * {None: 0, "channel": 1, "item": B}[case["gate"]]
    if case["op"] == "resnorm_fwd":
        return {"bytes": n * b * (3 + (1 if case["keep_sum"] else 0)) + vectors, "flops": 15.0 * n}
    return {"bytes": n * b * (5 + (1 if case["keep_sum"] else 0)) + 2 * vectors, "flops": 30.0 * n}


# ---- exact values --------------------------------------------------------------------------------

def exact_attention(s):
    """Softmax attention of each item and head by itself, in 64 bits; autograd for the gradients."""
    B, Hq, Tq, D, group = s["B"], s["Hq"], s["Tq"], s["D"], s["Hq"] // s["Hkv"]
    back = s["op"] == "attn_bwd"
    see = visible(s)
    z = lambda like: torch.zeros_like(like, dtype=torch.float64)  # noqa: E731
    out, lse, dq, dk, dv = z(s["q"]), torch.empty(B, Hq, Tq, dtype=torch.float64, device="cuda"), z(s["q"]), z(s["k"]), z(s["v"])
    for b in range(B):
        bias = None
        if see is not None:
            ok = see[min(b, see.shape[0] - 1), 0]
            bias = torch.zeros(ok.shape, dtype=torch.float64, device="cuda").masked_fill(~ok, -1e300)
            empty = ~ok.any(-1)
        for h in range(Hq):
            q, k, v = (t.double().contiguous().requires_grad_(back)
                       for t in (s["q"][b, :, h], s["k"][b, :, h // group], s["v"][b, :, h // group]))
            x = torch.einsum("id,jd->ij", q, k) / D ** 0.5
            if bias is not None:
                x = torch.where(bias < 0, bias, x)
            o = torch.softmax(x, -1) @ v
            if bias is not None:
                o = torch.where(empty[:, None], torch.zeros_like(o), o)
            if back:
                gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["dout"][b, :, h].double())
                dq[b, :, h] = gq
                dk[b, :, h // group] += gk
                dv[b, :, h // group] += gv
                continue
            out[b, :, h] = o
            total = torch.logsumexp(x, -1)
            lse[b, h] = total if bias is None else total.masked_fill(empty, -math.inf)
    return (dq, dk, dv) if back else (out, lse)


def exact_resnorm(s):
    F = torch.nn.functional
    back = s["op"] == "resnorm_bwd"
    names = ["x", "f", "post_weight", "post_bias", "gate_values", "weight", "bias"]
    t = {n: None if s[n] is None else s[n].double().requires_grad_(back) for n in names}
    C = s["C"]

    def norm(v, kind, w, b):
        if kind == "layer":
            return F.layer_norm(v, (C,), w, b, EPS)
        return v * w / torch.sqrt(v.pow(2).mean(-1, keepdim=True) + EPS)

    u = norm(t["f"], s["post"], t["post_weight"], t["post_bias"]) if s["post"] else t["f"]
    if s["gate"]:
        u = u * t["gate_values"].view(-1, 1, C)
    r = s["res_scale"] * t["x"] + u
    h = norm(r, s["norm"], t["weight"], t["bias"])
    if not back:
        return {"r": r if s["keep_sum"] else None, "h": h}
    loss = (h * s["dh"].double()).sum()
    if s["dr"] is not None:
        loss = loss + (r * s["dr"].double()).sum()
    have = [n for n in names if t[n] is not None]
    grads = dict(zip(have, torch.autograd.grad(loss, [t[n] for n in have])))
    called = {"x": "dx", "f": "df", "post_weight": "dpost_weight", "post_bias": "dpost_bias", "gate_values": "dgate",
              "weight": "dweight", "bias": "dbias"}
    return {called[n]: grads.get(n) for n in names}


def exact_act8(s):
    F = torch.nn.functional
    C, rows = s["C"], s["B"] * s["T"]
    f = {"gelu": F.gelu, "silu": F.silu, "lrelu": lambda v: F.leaky_relu(v, s["slope"])}[s["act"]]
    x = s["x"].double().view(rows, C)
    kept = torch.empty_like(x)
    for c in range(0, C, BLOCK):
        part = x[:, c:c + BLOCK]
        step = part.abs().max(1, keepdim=True).values / 127
        kept[:, c:c + BLOCK] = torch.where(step > 0, torch.round(part / step.clamp_min(1e-300)) * step, 0.0)
    kept = kept.view(s["x"].shape).requires_grad_(True)
    again = f(kept)
    dx, = torch.autograd.grad(again, kept, s["dy"].double())
    out = {"y": f(s["x"].double()), "dx": dx}
    if s["recompute"]:
        out["y_again"] = again.detach()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("attn"):
        return exact_attention(s)
    return exact_act8(s) if case["op"] == "act8" else exact_resnorm(s)
