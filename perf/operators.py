"""Workloads of the operators that training a token tower needs around its matrix products and attention cores:

  embed, embed_grad   token rows scaled and added to positions; the gradient of the table (and of the positions) by sorted tokens
  norm, norm_grad     x_new = res_scale * x + gate * post(y), h = pre(x_new) in one pass, with every gradient
  act8, act8_wgrad    an activation kept in 8 bits (e4m3 with a power-of-two scale for 128 channels) and its use in the backward pass

`run` computes them in elementary torch operations in 32 bits, or, with `own`, through the package's entry points.  Sizes are those of the
package's own towers (caption batches of 77 tokens in 768 channels over 49 408 rows, clips of 4097 tokens in 1024 / 4096 channels, 13 query
rows in 512 / 2048 channels) and, for the long packed batches, generic ones.
"""
import math

import torch

own = False

GROUP = 128                      # channels that share one scale
E4M3_MAX = 448.0                 # 1.75 * 2^8
QUICKGELU, RELU = "quickgelu", "relu"


def listed():
    return [
        # one new token for each of 32 sequences: the lookup of a decoding step
        {"name": "embed, one token each", "kind": "embed", "seqs": 32, "length": 1, "dim": 768, "rows": 49408, "table": "f32", "out": "bf16", "scale": 27.712812921102035,
         "pos": True, "ids": "zipf"},
        # the text tower's input for 2048 captions
        {"name": "embed, captions", "kind": "embed", "seqs": 2048, "length": 77, "dim": 768, "rows": 49408, "table": "f32", "out": "f32", "scale": 1.0, "pos": True,
         "ids": "captions"},
        # the table's gradient for 32 clips with five captions each: most ids are padding, start and end marks stand in every row
        {"name": "embed grad, captions", "kind": "embed_grad", "seqs": 160, "length": 77, "dim": 768, "rows": 49408, "grad": "f32", "scale": 1.0, "pos": True,
         "ids": "captions", "skip": False},
        # a packed batch of long sequences, gradients in bf16
        {"name": "embed grad, packed", "kind": "embed_grad", "seqs": 64, "length": 2048, "dim": 1024, "rows": 49408, "grad": "bf16", "scale": 32.0, "pos": False,
         "ids": "zipf", "skip": False},
        # the decoder's 13 query rows of 32 clips under a scalar tanh gate
        {"name": "norm, query rows", "kind": "norm", "groups": 32, "each": 13, "dim": 512, "x": "f32", "y": "f32", "h": "f32", "gate": "scalar", "tanh": True, "res": 1.0,
         "post": False, "pre": True, "rms": False},
        # a block's end on the vision tower's stream: norms before and after, one gate for each channel
        {"name": "norm, clips", "kind": "norm", "groups": 32, "each": 4097, "dim": 1024, "x": "f32", "y": "bf16", "h": "bf16", "gate": "channel", "tanh": False, "res": 1.0,
         "post": True, "pre": True, "rms": False},
        # its backward pass for a caption batch, a gate row for each caption, root-mean-square norms
        {"name": "norm grad, captions", "kind": "norm_grad", "groups": 160, "each": 77, "dim": 768, "x": "bf16", "y": "bf16", "h": "bf16", "gate": "group", "tanh": False,
         "res": 0.7071067811865476, "post": True, "pre": True, "rms": True},
        # and on the vision tower's stream
        {"name": "norm grad, clips", "kind": "norm_grad", "groups": 32, "each": 4097, "dim": 1024, "x": "f32", "y": "bf16", "h": "bf16", "gate": "channel", "tanh": False,
         "res": 1.0, "post": True, "pre": True, "rms": False},
        # the decoder's FFN rows: forward with the checkpoint, then the backward that reads it
        {"name": "act8, query rows", "kind": "act8", "tokens": 416, "dim": 2048, "type": "bf16", "act": RELU},
        # eight clips through the vision tower's MLP
        {"name": "act8, clips", "kind": "act8", "tokens": 32776, "dim": 4096, "type": "bf16", "act": QUICKGELU},
        # weight gradient of a projection of 32 captions from the 8-bit copy of its input
        {"name": "act8 wgrad, captions", "kind": "act8_wgrad", "tokens": 2464, "dim": 768, "outs": 768},
        # and of an MLP's second product over sixteen clips
        {"name": "act8 wgrad, clips", "kind": "act8_wgrad", "tokens": 65552, "dim": 4096, "outs": 1024},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "norm", "norm_grad", "act8", "act8_wgrad"])
    dim = rng.choice([rng.randrange(1, 600), 8 * rng.randrange(1, 128), 128 * rng.randrange(1, 9)])
    if kind in ("embed", "embed_grad"):
        seqs = _log(rng, 1, 2048)
        length = _log(rng, 1, min(2048, 131072 // seqs))
        case = {"kind": kind, "seqs": seqs, "length": length, "dim": dim, "rows": _log(rng, 4, 60000), "scale": rng.choice([1.0, math.sqrt(dim)]), "pos": rng.random() < 0.5,
                "ids": rng.choice(["zipf", "captions"])}
        if kind == "embed":
            return {**case, "table": rng.choice(["f32", "bf16"]), "out": rng.choice(["f32", "bf16"])}
        return {**case, "grad": rng.choice(["f32", "bf16"]), "skip": rng.random() < 0.5}
    if kind in ("norm", "norm_grad"):
        groups = _log(rng, 1, 64)
        post = rng.random() < 0.6
        return {"kind": kind, "groups": groups, "each": _log(rng, 1, 131072 // groups), "dim": dim, "x": rng.choice(["f32", "bf16"]), "y": rng.choice(["f32", "bf16"]),
                "h": rng.choice(["f32", "bf16"]), "gate": rng.choice(["none", "scalar", "channel", "group"]), "tanh": rng.random() < 0.3, "res": rng.choice([1.0, 0.7071067811865476]),
                "post": post, "pre": not post or rng.random() < 0.8, "rms": rng.random() < 0.5}
    if kind == "act8":
        dim = rng.choice([rng.randrange(1, 600), 8 * rng.randrange(1, 256), 128 * rng.randrange(1, 33)])
        return {"kind": kind, "tokens": _log(rng, 1, 32776), "dim": dim, "type": rng.choice(["f32", "bf16"]), "act": rng.choice([QUICKGELU, RELU])}
    dim = rng.choice([rng.randrange(1, 600), 128 * rng.randrange(1, 9), 512 * rng.randrange(1, 9)])
    return {"kind": kind, "tokens": _log(rng, 1, 65552), "dim": dim, "outs": rng.choice([rng.randrange(1, 300), 64 * rng.randrange(1, 17)])}


TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "bf16": 2}


def work(case):
    kind, d = case["kind"], case["dim"]
    if kind in ("embed", "embed_grad"):
        n, pos = case["seqs"] * case["length"], case["length"] * d * 4 if case["pos"] else 0
        distinct = _distinct(case)
        if kind == "embed":
            return {"bytes": 8 * n + distinct * d * BYTES[case["table"]] + pos + n * d * BYTES[case["out"]], "flops": 2 * n * d}
        return {"bytes": 8 * n + n * d * BYTES[case["grad"]] + case["rows"] * d * 4 + pos, "flops": 2 * n * d}
    if kind in ("norm", "norm_grad"):
        rows = case["groups"] * case["each"]
        bx, by, bh = BYTES[case["x"]], BYTES[case["y"]], BYTES[case["h"]] if case["pre"] else 0
        if kind == "norm":
            return {"bytes": rows * d * (2 * bx + by + bh), "flops": rows * d * (4 + 8 * case["post"] + 8 * case["pre"])}
        return {"bytes": rows * d * (3 * bx + 2 * by + bh), "flops": rows * d * (8 + 20 * case["post"] + 20 * case["pre"])}
    if kind == "act8":
        n, b = case["tokens"] * d, BYTES[case["type"]]
        return {"bytes": n * (4 * b + 1) + case["tokens"] * -(-d // GROUP) * 4, "flops": n * 30}
    k, m = case["tokens"], case["outs"]
    return {"bytes": k * (2 * m + d) + k * -(-d // GROUP) * 4 + 4 * m * d, "flops": 2 * k * m * d}


def _distinct(case):
    """How many table rows a batch names in the mean: rank k is drawn with the weight log((k + 2) / (k + 1)) (see _ids)."""
    v, n = case["rows"], case["seqs"] * (min(case["length"], 12) if case["ids"] == "captions" else case["length"])
    k = torch.arange(v, dtype=torch.float64)
    return float((1 - torch.exp(n * torch.log1p(-torch.log((k + 2) / (k + 1)) / math.log(v + 1)))).sum())


def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _ids(g, case):
    """Token ids [seqs, length]: word frequencies fall as 1 / rank; a caption is a start mark, 5 to 20 words, an end mark, and zeros."""
    s, n, v = case["seqs"], case["length"], case["rows"]
    u = torch.rand(s, n, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.clamp((torch.exp(u * math.log(v + 1)) - 1).long(), 0, v - 1)
    if case["ids"] != "captions":
        return ids, torch.ones(s, n, 1, device="cuda")
    end = 1 + torch.randint(5, 21, (s, 1), generator=g, device="cuda")
    t = torch.arange(n, device="cuda")[None, :]
    ids = torch.where(t == 0, v - 2, torch.where(t < end, ids, torch.where(t == end, v - 1, 0)))
    return ids, (t <= end).float()[:, :, None]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, d = case["kind"], case["dim"]
    s = {"case": case}
    if kind in ("embed", "embed_grad"):
        s["ids"], used = _ids(g, case)
        n = case["length"]
        if kind == "embed":
            s["table"] = _randn(g, case["rows"], d, dtype=TYPES[case["table"]], scale=0.02)
            s["pos"] = _randn(g, n, d, scale=0.01) if case["pos"] else None
        else:
            # nothing behind a caption's end mark reaches the loss
            s["dy"] = (_randn(g, case["seqs"], n, d) * used).to(TYPES[case["grad"]])
    elif kind in ("norm", "norm_grad"):
        rows = case["groups"] * case["each"]
        x = _randn(g, rows, d, scale=2.0)
        y = _randn(g, rows, d, dtype=TYPES[case["y"]]) + 0.25
        s["y"] = y.to(TYPES[case["y"]])
        shape = {"none": None, "scalar": (1,), "channel": (d,), "group": (case["groups"], d)}[case["gate"]]
        s["gate"] = None if shape is None else _randn(g, *shape, scale=0.1) + 0.5
        for name in ("post", "pre"):
            gamma, beta = 1 + _randn(g, d, scale=0.1), _randn(g, d, scale=0.1)
            s[name] = (gamma, None if case["rms"] else beta, 1e-5) if case[name] else None
        if kind == "norm":
            s["x"] = x.to(TYPES[case["x"]])
        else:
            s["x_new"] = x.to(TYPES[case["x"]])
            # a loss that pulls the stream towards or away from the branch: its gradient has a part along the branch
            s["dx_new"] = (_randn(g, rows, d) + 0.25 * s["y"].float()).to(TYPES[case["x"]])
            s["dh"] = _randn(g, rows, d, dtype=TYPES[case["h"]]) if case["pre"] else None
    elif kind == "act8":
        # pre-activations: a spread that differs from token to token, and a few channels that stand out
        u = _randn(g, case["tokens"], d) * torch.exp(_randn(g, case["tokens"], 1, scale=0.5)) * torch.exp(_randn(g, 1, d, scale=0.5)) - 0.5
        s["u"] = u.to(TYPES[case["type"]])
        s["da"] = _randn(g, case["tokens"], d, dtype=TYPES[case["type"]])
    else:
        u = _randn(g, case["tokens"], d, dtype=torch.bfloat16)
        s["q"], s["scale"] = _to_e4m3(u.float())
        s["dy"] = _randn(g, case["tokens"], case["outs"], dtype=torch.bfloat16)
    return s


def run(s):
    kind = s["case"]["kind"]
    if own:
        return _OWN[kind](s, s["case"])
    return _PLAIN[kind](s, s["case"])


# ---- the package's entry points ------------------------------------------------------------------------------------------------------
def _own_ops():
    from helping_hand_for_egocentric_videos_amd import ops
    return ops


def _own_act(ops, case):
    return ops.ACT_QUICKGELU if case["act"] == QUICKGELU else ops.ACT_RELU


def _own_embed(s, case):
    return _own_ops().embed_tokens(s["ids"], s["table"], scale=case["scale"], pos=s["pos"], out_dtype=TYPES[case["out"]])


def _own_embed_grad(s, case):
    return _own_ops().embed_tokens_bwd(s["ids"], s["dy"], case["rows"], scale=case["scale"], skip_id=0 if case["skip"] else None, pos_grad=case["pos"])


def _own_norm(s, case):
    return _own_ops().residual_norm(s["x"], s["y"], gate=s["gate"], gate_tanh=case["tanh"], res_scale=case["res"], post=s["post"], pre=s["pre"], rms=case["rms"],
                                    out_dtype=TYPES[case["h"]])


def _own_norm_grad(s, case):
    return tuple(_own_ops().residual_norm_bwd(s["x_new"], s["y"], s["dx_new"], s["dh"], gate=s["gate"], gate_tanh=case["tanh"], res_scale=case["res"], post=s["post"],
                                              pre=s["pre"], rms=case["rms"]))


def _own_act8(s, case):
    ops = _own_ops()
    a, q, scale = ops.act8(s["u"], _own_act(ops, case))
    return a, q, scale, ops.act8_bwd(q, scale, s["da"], _own_act(ops, case))


def _own_act8_wgrad(s, case):
    return _own_ops().gemm_tn_act8(s["dy"], s["q"], s["scale"], colsum=True)


_OWN = {"embed": _own_embed, "embed_grad": _own_embed_grad, "norm": _own_norm, "norm_grad": _own_norm_grad, "act8": _own_act8, "act8_wgrad": _own_act8_wgrad}


# ---- the plain forms -----------------------------------------------------------------------------------------------------------------
def _embed(s, case):
    x = s["table"][s["ids"]].float() * case["scale"]
    if s["pos"] is not None:
        x = x + s["pos"]
    return x.to(TYPES[case["out"]])


def _embed_grad(s, case):
    ids, dy = s["ids"].reshape(-1), s["dy"].float()
    flat = dy.reshape(ids.numel(), -1)
    if case["skip"]:
        flat = flat * (ids != 0)[:, None]
    dw = torch.zeros(case["rows"], case["dim"], device="cuda").index_add_(0, ids, flat) * case["scale"]
    return (dw, dy.sum(0)) if case["pos"] else dw


def _normed(v, gamma, beta, eps, rms):
    if not rms:
        v = v - v.mean(-1, keepdim=True)
    n = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * gamma
    return n if beta is None else n + beta


def _gate_rows(s, case):
    """The gate as a factor that broadcasts over [groups, each, dim], or None."""
    if s["gate"] is None:
        return None
    g = torch.tanh(s["gate"]) if case["tanh"] else s["gate"]
    return g[:, None, :] if case["gate"] == "group" else g


def _norm(s, case):
    rms = case["rms"]
    p = s["y"].float()
    if s["post"] is not None:
        p = _normed(p, *s["post"], rms)
    g = _gate_rows(s, case)
    if g is not None:
        p = (p.view(case["groups"], case["each"], -1) * g).view(p.shape)
    x = s["x"].float() * case["res"] + p
    return x.to(TYPES[case["x"]]), _normed(x, *s["pre"], rms).to(TYPES[case["h"]]) if s["pre"] is not None else None


def _normed_grad(v, dn, gamma, eps, rms):
    """(gradient of v, of gamma, of beta) of a norm whose output has the gradient dn."""
    c = v if rms else v - v.mean(-1, keepdim=True)
    r = torch.rsqrt((c * c).mean(-1, keepdim=True) + eps)
    xh = c * r
    k = dn * gamma
    dv = k - xh * (k * xh).mean(-1, keepdim=True)
    if not rms:
        dv = dv - k.mean(-1, keepdim=True)
    return dv * r, (dn * xh).sum(0), None if rms else dn.sum(0)


def _norm_grad(s, case):
    rms = case["rms"]
    dx, y = s["dx_new"].float(), s["y"].float()
    dg2 = db2 = dg1 = db1 = dgate = None
    if s["pre"] is not None:
        gamma, _, eps = s["pre"]
        d, dg2, db2 = _normed_grad(s["x_new"].float(), s["dh"].float(), gamma, eps, rms)
        dx = dx + d
    p = _normed(y, *s["post"], rms) if s["post"] is not None else y
    dp = dx
    g = _gate_rows(s, case)
    if g is not None:
        cube = (case["groups"], case["each"], case["dim"])
        t = (dx * p).view(cube)
        dgate = {"scalar": lambda: t.sum().view(1), "channel": lambda: t.sum((0, 1)), "group": lambda: t.sum(1)}[case["gate"]]()
        if case["tanh"]:
            dgate = dgate * (1 - torch.tanh(s["gate"]) ** 2)
        dp = (dx.view(cube) * g).view(dx.shape)
    if s["post"] is not None:
        gamma, _, eps = s["post"]
        dp, dg1, db1 = _normed_grad(y, dp, gamma, eps, rms)
    return (dx * case["res"]).to(TYPES[case["x"]]), dp.to(TYPES[case["y"]]), dgate, dg1, db1, dg2, db2


def _to_e4m3(u):
    """(e4m3 values, scales [tokens, groups]) of u fp32: 128 channels share the smallest power of two that brings them to 448 or below."""
    t, d = u.shape
    n = -(-d // GROUP)
    v = torch.nn.functional.pad(u, (0, n * GROUP - d)).view(t, n, GROUP)
    top = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)
    k = torch.where(top > 0, torch.clamp(e - 9 + (m > 0.875).int(), -117, 120), 0)
    q = (v * _power(-k)[:, :, None]).to(torch.float8_e4m3fn)
    return q.view(t, n * GROUP)[:, :d].contiguous(), _power(k)


def _power(k):
    """2^k in fp32 for whole -126 <= k <= 127, from the exponent's bits (a power function may be off by a step)."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _of_e4m3(q, scale):
    return q.float() * scale.repeat_interleave(GROUP, 1)[:, :q.shape[1]]


def _act8(s, case):
    u, t = s["u"].float(), TYPES[case["type"]]
    q, scale = _to_e4m3(u)
    v, da = _of_e4m3(q, scale), s["da"].float()
    if case["act"] == RELU:
        return torch.where(u < 0, 0.0, u).to(t), q, scale, (da * (v > 0)).to(t)
    sig = 1 / (1 + torch.exp(-1.702 * v))
    return (u / (1 + torch.exp(-1.702 * u))).to(t), q, scale, (da * (sig * (1 + 1.702 * v * (1 - sig)))).to(t)


def _act8_wgrad(s, case):
    dy = s["dy"].float()
    return dy.t() @ _of_e4m3(s["q"], s["scale"]), dy.sum(0)


_PLAIN = {"embed": _embed, "embed_grad": _embed_grad, "norm": _norm, "norm_grad": _norm_grad, "act8": _act8, "act8_wgrad": _act8_wgrad}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["kind"]](s, case)


def _exact_embed(s, case):
    flat = s["ids"].reshape(-1)
    x = torch.index_select(s["table"].double(), 0, flat).mul_(case["scale"]).view(case["seqs"], case["length"], case["dim"])
    return x if s["pos"] is None else x.add_(s["pos"].double()[None])


def _exact_embed_grad(s, case):
    """Prefix sums along the sorted tokens: a row's gradient is the difference of two of them."""
    flat = s["ids"].reshape(-1)
    order = torch.argsort(flat, stable=True)
    sums = torch.cumsum(s["dy"].reshape(flat.numel(), -1)[order].double(), 0)
    sums = torch.cat([torch.zeros_like(sums[:1]), sums])
    v = torch.arange(case["rows"], device="cuda")
    at = flat[order].contiguous()
    dw = (sums[torch.searchsorted(at, v, right=True)] - sums[torch.searchsorted(at, v)]).mul_(case["scale"])
    if case["skip"]:
        dw[0] = 0
    return (dw, s["dy"].double().sum(0)) if case["pos"] else dw


def _exact_block(case, x, y, gate, post, pre):
    def norm(v, gamma, beta, eps):
        var = (v ** 2).mean(-1, keepdim=True) if case["rms"] else v.var(-1, unbiased=False, keepdim=True)
        out = gamma * (v if case["rms"] else v - v.mean(-1, keepdim=True)) / (var + eps).sqrt()
        return out if beta is None else out + beta

    b = y if post is None else norm(y, *post)
    if gate is not None:
        a = gate.tanh() if case["tanh"] else gate
        b = b * (a.repeat_interleave(case["each"], 0) if case["gate"] == "group" else a)
    x_new = x * case["res"] + b
    return x_new, None if pre is None else norm(x_new, *pre)


def _double(v, grad=False):
    return None if v is None else v.double().requires_grad_(grad)


def _exact_norm(s, case):
    post, pre = (None if p is None else (p[0].double(), _double(p[1]), p[2]) for p in (s["post"], s["pre"]))
    return _exact_block(case, s["x"].double(), s["y"].double(), _double(s["gate"]), post, pre)


def _exact_norm_grad(s, case):
    """Derivatives of the forward definition, taken by torch in 64 bits, at the x that gives this x_new."""
    y, gate = _double(s["y"], True), _double(s["gate"], True)
    post, pre = (None if p is None else (_double(p[0], True), _double(p[1], True), p[2]) for p in (s["post"], s["pre"]))
    with torch.no_grad():
        branch, _ = _exact_block(case, torch.zeros_like(y), y, gate, post, None)
        x = (s["x_new"].double() - branch) / case["res"]
        del branch
    x.requires_grad_(True)
    x_new, h = _exact_block(case, x, y, gate, post, pre)
    leaves = [x, y, gate] + [t for p in (post, pre) for t in ((None, None) if p is None else p[:2])]
    outs, grads = [x_new], [s["dx_new"].double()]
    if h is not None:
        outs.append(h)
        grads.append(s["dh"].double())
    found = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], grads))
    return tuple(None if t is None else next(found) for t in leaves)


def _exact_values(u):
    """(values in units of their scale, scales), both in 64 bits: the grid of e4m3 has 8 steps to a power of two, and steps of 2^-9 at its lower end."""
    t, d = u.shape
    n = -(-d // GROUP)
    v = torch.zeros(t, n * GROUP, dtype=torch.float64, device=u.device)
    v[:, :d] = u
    v = v.view(t, n, GROUP)
    top = v.abs().amax(-1)
    def power(k):
        return ((k.long() + 1023) << 52).view(torch.float64)

    k = torch.ceil(torch.log2(torch.where(top > 0, top, E4M3_MAX) / E4M3_MAX))
    k = torch.where(top > E4M3_MAX * power(k), k + 1, torch.where(top <= E4M3_MAX * power(k - 1), k - 1, k)).clamp_(-117, 120)
    k = torch.where(top > 0, k, 0.0)
    v = v / power(k)[:, :, None]
    w = v.abs().clamp_min(2.0 ** -6)
    e = torch.floor(torch.log2(w))
    step = power(torch.where(w < power(e), e - 1, torch.where(w >= power(e + 1), e + 1, e)) - 3)
    return (torch.round(v / step) * step).view(t, n * GROUP)[:, :d], power(k)


def _exact_act8(s, case):
    u = s["u"].double()
    q, scale = _exact_values(u)
    v = q * scale.repeat_interleave(GROUP, 1)[:, :case["dim"]]
    with torch.enable_grad():
        w = v.requires_grad_(True)
        out = torch.relu(w) if case["act"] == RELU else w * torch.sigmoid(1.702 * w)
        du, = torch.autograd.grad(out, w, s["da"].double())
    a = torch.relu(u) if case["act"] == RELU else u * torch.sigmoid(1.702 * u)
    return a, q.detach(), scale, du


def _exact_act8_wgrad(s, case):
    """Summed over slices of the tokens, so that one slice at a time is held in 64 bits."""
    dw = torch.zeros(case["outs"], case["dim"], dtype=torch.float64, device="cuda")
    for i in range(0, case["tokens"], 8192):
        q = s["q"][i:i + 8192].double()
        for j in range(s["scale"].shape[1]):
            q[:, GROUP * j:GROUP * (j + 1)] *= s["scale"][i:i + 8192, j:j + 1].double()
        dw += s["dy"][i:i + 8192].double().t() @ q
    return dw, s["dy"].double().sum(0)


_EXACT = {"embed": _exact_embed, "embed_grad": _exact_embed_grad, "norm": _exact_norm, "norm_grad": _exact_norm_grad, "act8": _exact_act8, "act8_wgrad": _exact_act8_wgrad}
