"""Measured cases of the training operators: attention with its gradient, LayerNorm + modulation with its gradient, and
RMSNorm + rotary embedding with its gradient, the three steps of a Wan DiT block that are not matrix products.

``run`` is one training step of an operator: the forward pass and the backward pass for a given output gradient (the
forward pass alone where a case says so).  With ``own`` it makes the calls of ``dax_b200.ops``; without it the plain
forms below, in elementary torch operations on fp32.

Shapes: ``q, out, dout [B, H, Sq, 128]`` and ``k, v [B, H, Sk, 128]`` are views of token-major ``[B, S, H, 128]`` memory, as
the projections write them; ``x [B, S, D]``.  ``q_lens`` / ``k_lens`` (int32 ``[B]``) give the valid tokens of a padded batch.
"""
import math

import torch

own = False

HEAD = 128
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _attention(name, B, H, Sq, Sk, dtype="bf16", q_min=-1, k_min=-1, backward=True):
    c = {"op": "attention", "B": B, "H": H, "Sq": Sq, "Sk": Sk, "dtype": dtype, "q_min": q_min, "k_min": k_min, "backward": backward}
    return {"name": name, **c} if name else c


def _layernorm(name, B, S, D, dtype, affine, modulate):
    c = {"op": "layernorm", "B": B, "S": S, "D": D, "dtype": dtype, "affine": affine, "modulate": modulate}
    return {"name": name, **c} if name else c


def _rmsnorm(name, B, S, H, dtype, rotate):
    c = {"op": "rmsnorm_rope", "B": B, "S": S, "D": H * HEAD, "dtype": dtype, "rotate": rotate}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a token grid of 2 x 8 x 16 with four heads: the smallest model that the smoke run uses; latency counts
        _attention("attention_256", 1, 4, 256, 256),
        # three latent frames at 480p attending over two text contexts, one of them padded to 512
        _attention("attention_text", 2, 12, 4680, 512, k_min=77),
        # the odd length that a rank has of a 480p clip on eight GPUs, in fp16
        _attention("attention_4095_f16", 1, 12, 4095, 4095, dtype="f16"),
        # a padded batch of clips of different lengths, one of them empty
        _attention("attention_padded", 4, 10, 1560, 1560, q_min=0, k_min=0),
        # 480p, 81 frames, the five heads that one of eight GPUs has after the exchange
        _attention("attention_32760", 1, 5, 32760, 32760),
        # the forward pass that keeps what the backward pass needs, all 40 heads, a quarter of that clip
        _attention("attention_forward_8190", 1, 40, 8190, 8190, backward=False),
        # the smoke run's width and token count
        _layernorm("layernorm_256x512", 1, 256, 512, "bf16", False, True),
        # the affine norm in front of cross-attention at the width of the 1.3B model, two clips, in fp16
        _layernorm("layernorm_affine_4095x1536_f16", 2, 4095, 1536, "f16", True, False),
        # a residual stream kept in fp32, affine and modulated
        _layernorm("layernorm_1560x5120_f32", 4, 1560, 5120, "f32", True, True),
        # the adaLN step of the 14B model at 480p, 81 frames
        _layernorm("layernorm_32760x5120", 1, 32760, 5120, "bf16", False, True),
        # queries or keys of the smallest model, normalised and rotated
        _rmsnorm("rmsnorm_rope_256x512", 1, 256, 4, "bf16", True),
        # those of the 14B model at 480p, 81 frames
        _rmsnorm("rmsnorm_rope_32760x5120", 1, 32760, 40, "bf16", True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "layernorm", "rmsnorm_rope"])
    if op == "attention":
        Sq = _log(rng, 1, 32760)
        Sk = Sq if rng.random() < 0.5 else _log(rng, 1, 32760)
        B, H = rng.randint(1, 4), _log(rng, 1, 40)
        most = 5 * 32760 * 32760
        while B * H * Sq * Sk > most and B > 1:
            B -= 1
        H = max(1, min(H, most // (B * Sq * Sk)))
        q_min = rng.randint(0, Sq) if rng.random() < 0.3 else -1
        k_min = rng.randint(0, Sk) if rng.random() < 0.4 else -1
        return _attention("", B, H, Sq, Sk, rng.choice(["bf16", "bf16", "f16"]), q_min, k_min, rng.random() < 0.8)
    B, S = rng.randint(1, 4), _log(rng, 1, 32760)
    if op == "layernorm":
        D = 8 * _log(rng, 1, 1024)
        S = max(1, min(S, 32760 * 5120 // (B * D)))
        dtype, (affine, modulate) = rng.choice(["bf16", "f16", "f32"]), rng.choice([(False, False), (True, False), (False, True), (True, True)])
        if dtype == "f32":
            S = max(1, min(S, 32760 * 2560 // (B * D)))
        return _layernorm("", B, S, D, dtype, affine, modulate)
    H = _log(rng, 1, 64)
    dtype = rng.choice(["bf16", "f16", "f32"])
    S = max(1, min(S, 32760 * (2560 if dtype == "f32" else 5120) // (B * H * HEAD)))
    return _rmsnorm("", B, S, H, dtype, rng.random() < 0.75)


def _lens(B, S, low):
    """Valid tokens of each sequence of a padded batch: spread evenly from `low` to all of them; None without padding."""
    return None if low < 0 else [low + (S - low) * b // max(B - 1, 1) for b in range(B)]


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    if case["op"] == "attention":
        B, H, Sq, Sk = case["B"], case["H"], case["Sq"], case["Sk"]
        # normalised queries and keys; keys with an offset for each channel, as trained models have
        q = normal(B, Sq, H, HEAD, dtype=t).transpose(1, 2)
        k = (normal(B, Sk, H, HEAD) + normal(1, 1, H, HEAD, std=2.0)).to(t).transpose(1, 2)
        v = normal(B, Sk, H, HEAD, dtype=t).transpose(1, 2)
        dout = normal(B, Sq, H, HEAD, std=0.1, dtype=t).transpose(1, 2)
        q_lens, k_lens = _lens(B, Sq, case["q_min"]), _lens(B, Sk, case["k_min"])
        q_lens = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device="cuda")
        k_lens = None if k_lens is None else torch.tensor(k_lens, dtype=torch.int32, device="cuda")
        return {"op": "attention", "backward": case["backward"], "q": q, "k": k, "v": v, "dout": dout, "q_lens": q_lens, "k_lens": k_lens}
    B, S, D = case["B"], case["S"], case["D"]
    x = (normal(B, S, D) + normal(1, 1, D, std=0.5)).to(t)
    dy = normal(B, S, D, std=0.1, dtype=t)
    if case["op"] == "layernorm":
        s = {"op": "layernorm", "x": x, "dy": dy, "weight": None, "bias": None, "shift": None, "scale": None}
        if case["affine"]:
            s["weight"], s["bias"] = 1 + normal(D, std=0.1), normal(D, std=0.1)
        if case["modulate"]:
            s["shift"], s["scale"] = normal(B, D, std=0.3), normal(B, D, std=0.3)
        return s
    s = {"op": "rmsnorm_rope", "x": x, "dy": dy, "weight": 1 + normal(D, std=0.1), "cos": None, "sin": None}
    if case["rotate"]:  # rows of a rotary table, one angle for each pair of a head's channels
        ang = torch.arange(S, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, device="cuda", dtype=torch.float64) / 64)
        s["cos"], s["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
    return s


# ---------------------------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------------------------
def _valid(lens, S):
    """[B, 1, S]: which tokens are inside their sequence."""
    return torch.arange(S, device=lens.device) < lens[:, None, None]


def _plain_attention(s):
    q, k, v, dout = s["q"].float(), s["k"].float(), s["v"].float(), s["dout"].float()
    t, scale = s["q"].dtype, 1 / math.sqrt(HEAD)
    p = (q @ k.transpose(2, 3)).mul_(scale)
    if s["k_lens"] is not None:
        p.masked_fill_(~_valid(s["k_lens"], k.shape[2])[:, :, None, :], -math.inf)
    if s["q_lens"] is not None:
        p.masked_fill_(~_valid(s["q_lens"], q.shape[2])[:, :, :, None], -math.inf)
    top = p.amax(3, keepdim=True).clamp_min_(-3e38)  # a row that sees no key: every exponential is zero
    p.sub_(top).exp_()
    total = p.sum(3, keepdim=True)
    lse = (top + total.log()).squeeze(3)
    p.div_(total.clamp_min(1e-38))
    out = p @ v
    if not s["backward"]:
        return out.to(t), lse
    dv = p.transpose(2, 3) @ dout
    ds = dout @ v.transpose(2, 3)
    ds.sub_((ds * p).sum(3, keepdim=True)).mul_(p).mul_(scale)
    return out.to(t), lse, (ds @ k).to(t), (ds.transpose(2, 3) @ q).to(t), dv.to(t)


def _plain_layernorm(s):
    x, dy, t = s["x"].float(), s["dy"].float(), s["x"].dtype
    x = x - x.mean(2, keepdim=True)
    rstd = (x.square().mean(2, keepdim=True) + 1e-6).rsqrt()
    n = x.mul_(rstd)
    y, g, r = n, dy, {}
    if s["weight"] is not None:
        y = y * s["weight"] + s["bias"]
    if s["scale"] is not None:
        r["dshift"], r["dscale"] = dy.sum(1), (dy * y).sum(1)
        y = y * (1 + s["scale"])[:, None] + s["shift"][:, None]
        g = g * (1 + s["scale"])[:, None]
    if s["weight"] is not None:
        r["dbias"], r["dweight"] = g.sum((0, 1)), (g * n).sum((0, 1))
        g = g * s["weight"]
    dx = (g - g.mean(2, keepdim=True) - n * (g * n).mean(2, keepdim=True)) * rstd
    return {"y": y.to(t), "dx": dx.to(t), **r}


def _plain_rmsnorm_rope(s):
    x, dy, t = s["x"].float(), s["dy"].float(), s["x"].dtype
    rstd = (x.square().mean(2, keepdim=True) + 1e-6).rsqrt()
    n = x * rstd
    y, g = n * s["weight"], dy
    if s["cos"] is not None:
        cos, sin = s["cos"][None, :, None], s["sin"][None, :, None]
        a, b = y.unflatten(2, (-1, 64, 2)).unbind(4)
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), 4).flatten(2)
        a, b = dy.unflatten(2, (-1, 64, 2)).unbind(4)
        g = torch.stack((a * cos + b * sin, b * cos - a * sin), 4).flatten(2)
    dweight = (g * n).sum((0, 1))
    g = g * s["weight"]
    dx = (g - n * (g * n).mean(2, keepdim=True)) * rstd
    return {"y": y.to(t), "dx": dx.to(t), "dweight": dweight}


# ---------------------------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------------------------
def _own(s):
    from dax_b200 import ops

    if s["op"] == "attention":
        lens = {"q_lens": s["q_lens"], "k_lens": s["k_lens"]}
        out, lse = ops.attention_lse(s["q"], s["k"], s["v"], **lens)
        if not s["backward"]:
            return out, lse
        return (out, lse, *ops.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **lens))
    if s["op"] == "layernorm":
        y, mean, rstd = ops.layernorm_modulate(s["x"], ln_weight=s["weight"], ln_bias=s["bias"], shift=s["shift"], scale=s["scale"])
        r = ops.layernorm_modulate_backward(s["dy"], s["x"], mean, rstd, ln_weight=s["weight"], ln_bias=s["bias"], scale=s["scale"])
        r = dict(zip(("dx", "dweight", "dbias", "dshift", "dscale"), r))
        return {"y": y, **{k: v for k, v in r.items() if v is not None}}
    y, rstd = ops.rmsnorm_rope(s["x"], s["weight"], rope_cos=s["cos"], rope_sin=s["sin"])
    dx, dweight = ops.rmsnorm_rope_backward(s["dy"], s["x"], rstd, s["weight"], rope_cos=s["cos"], rope_sin=s["sin"])
    return {"y": y, "dx": dx, "dweight": dweight}


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "layernorm": _plain_layernorm, "rmsnorm_rope": _plain_rmsnorm_rope}[state["op"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    B = case["B"]
    if case["op"] == "attention":
        H, Sq, Sk = case["H"], case["Sq"], case["Sk"]
        q_lens, k_lens = _lens(B, Sq, case["q_min"]) or [Sq] * B, _lens(B, Sk, case["k_min"]) or [Sk] * B
        pairs, queries, keys = sum(a * b for a, b in zip(q_lens, k_lens)) * H, sum(q_lens) * H, sum(k_lens) * H
        # two products forward, five more backward; q, k, v (and dout) read, everything written in full
        if not case["backward"]:
            return {"bytes": (queries + 2 * keys + B * H * Sq) * HEAD * e + B * H * Sq * 4, "flops": 4 * HEAD * pairs}
        return {"bytes": (2 * queries + 2 * keys + 2 * B * H * (Sq + Sk)) * HEAD * e + B * H * Sq * 4, "flops": 14 * HEAD * pairs}
    n = B * case["S"] * case["D"]
    if case["op"] == "layernorm":
        vectors = (4 * case["D"] if case["affine"] else 0) + (4 * B * case["D"] if case["modulate"] else 0)
        return {"bytes": 4 * n * e + 4 * vectors, "flops": 20 * n}
    return {"bytes": 4 * n * e + 8 * case["D"] + (512 * case["S"] if case["rotate"] else 0), "flops": 20 * n}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_head(q, k, v, dout, backward):
    """One head, valid tokens only: the softmax and the gradients of sum(out * dout)."""
    w = torch.softmax(torch.einsum("id,jd->ij", q, k) / math.sqrt(HEAD), 1)
    lse = torch.logsumexp(torch.einsum("id,jd->ij", q, k) / math.sqrt(HEAD), 1)
    out = torch.einsum("ij,jd->id", w, v)
    if not backward:
        return out, lse
    dw = torch.einsum("id,jd->ij", dout, v)
    if k.shape[0] == 1:  # the softmax of one key is constant
        da = torch.zeros_like(dw)
    else:
        da = w * (dw - torch.einsum("id,id->i", dout, out)[:, None]) / math.sqrt(HEAD)
    return out, lse, torch.einsum("ij,jd->id", da, k), torch.einsum("ij,id->jd", da, q), torch.einsum("ij,id->jd", w, dout)


def _exact_attention(case, s):
    B, H, Sq, Sk = case["B"], case["H"], case["Sq"], case["Sk"]
    zeros = lambda S: torch.zeros(B, H, S, HEAD, dtype=torch.float64, device="cuda")  # noqa: E731
    got = [zeros(Sq), torch.full((B, H, Sq), -math.inf, dtype=torch.float64, device="cuda")]
    got += [zeros(Sq), zeros(Sk), zeros(Sk)] if case["backward"] else []
    n_q, n_k = _lens(B, Sq, case["q_min"]) or [Sq] * B, _lens(B, Sk, case["k_min"]) or [Sk] * B
    for b in range(B):
        if n_q[b] == 0 or n_k[b] == 0:
            continue
        for h in range(H):
            q, dout = (s[n][b, h, : n_q[b]].double() for n in ("q", "dout"))
            k, v = (s[n][b, h, : n_k[b]].double() for n in ("k", "v"))
            for to, value in zip(got, _exact_head(q, k, v, dout, case["backward"])):
                to[b, h, : value.shape[0]] = value
    return tuple(got)


def _exact_layernorm(s):
    x, dy = s["x"].double(), s["dy"].double()
    D = x.shape[2]
    std = torch.sqrt(x.var(2, correction=0, keepdim=True) + 1e-6)
    n = (x - x.mean(2, keepdim=True)) / std
    w = s["weight"].double() if s["weight"] is not None else torch.ones(D, dtype=torch.float64, device="cuda")
    b = s["bias"].double() if s["bias"] is not None else torch.zeros(D, dtype=torch.float64, device="cuda")
    m = 1 + s["scale"].double()[:, None] if s["scale"] is not None else 1.0
    y = (n * w + b) * m + (s["shift"].double()[:, None] if s["shift"] is not None else 0.0)
    dn = dy * m * w
    dx = dn / std - (dn.sum(2, keepdim=True) + n * torch.einsum("bsd,bsd->bs", dn, n)[..., None]) / (D * std)
    r = {"y": y, "dx": dx}
    if s["weight"] is not None:
        r["dweight"], r["dbias"] = torch.einsum("bsd,bsd->d", dy * m, n), (dy * m).sum((0, 1))
    if s["scale"] is not None:
        r["dscale"], r["dshift"] = torch.einsum("bsd,bsd->bd", dy, n * w + b), dy.sum(1)
    return r


def _exact_rmsnorm_rope(s):
    x, dy, w = s["x"].double(), s["dy"].double(), s["weight"].double()
    D = x.shape[2]
    rms = torch.sqrt(torch.einsum("bsd,bsd->bs", x, x)[..., None] / D + 1e-6)
    n = x / rms
    y, back = n * w, dy
    if s["cos"] is not None:  # a pair of channels as a complex number, turned by the table's angle and back
        turn = torch.complex(s["cos"].double(), s["sin"].double())[None, :, None]
        y = torch.view_as_real(torch.view_as_complex(y.unflatten(2, (-1, 64, 2)).contiguous()) * turn).flatten(2)
        back = torch.view_as_real(torch.view_as_complex(dy.unflatten(2, (-1, 64, 2)).contiguous()) * turn.conj()).flatten(2)
    dn = back * w
    dx = dn / rms - n * torch.einsum("bsd,bsd->bs", dn, n)[..., None] / (D * rms)
    return {"y": y, "dx": dx, "dweight": torch.einsum("bsd,bsd->d", back, n)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    return _exact_layernorm(s) if case["op"] == "layernorm" else _exact_rmsnorm_rope(s)
