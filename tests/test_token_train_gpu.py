"""GPU tests of the operators that train a token stream (ops.embed_tokens, residual_norm, act8 and their gradients) against plain implementations in 64 bits.

Tolerances are bounds, not measurements.  U = 2^-24 is fp32's largest relative rounding, a value stored in bf16 is off by at most 2^-8 of itself more.
A sum of n terms taken in any order is off by at most n U (to first order) of the sum of the terms' magnitudes; the magnitudes are taken from the 64-bit result,
element by element."""
import pytest
import torch

from helping_hand_for_egocentric_videos_amd import ops
from _record import record

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16


def rnd(*shape, seed=0, scale=1.0, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def rints(lo, hi, shape, seed=0, dtype=torch.int64):
    return torch.randint(lo, hi, shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def stored(ref, dtype):
    """What rounding to the output's type may add."""
    return ref.abs() * (2.0 ** -8 if dtype == BF16 else U)


def within(got, ref, bound, what):
    """|got - ref| <= bound element by element (64 bits), and the same places finite."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    if got.numel() == 0:
        return
    err = (got.double() - ref).abs()
    worst = float((err / (bound + 1e-300)).max())
    record("test_token_train_gpu", what, worst, 1.0)
    assert worst <= 1.0, "%s: %.3g times the bound (largest error %.3g)" % (what, worst, float(err.max()))


# ---- embedding -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [1, 3, 8, 77, 128, 768, 1030, 2052])
@pytest.mark.parametrize("wt,ot", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
def test_embed_tokens(dim, wt, ot):
    V, S, L = 211, 5, 13
    w, pos, ids = rnd(V, dim, seed=1, dtype=wt), rnd(L + 2, dim, seed=2), rints(0, V, (S, L), seed=3)
    for scale, p, i in ((1.0, None, ids), (dim ** 0.5, pos, ids), (-0.3, pos, ids.int()), (2.0, pos[4:5], ids[:, 4:5].contiguous())):
        got = ops.embed_tokens(i, w, scale=scale, pos=p, out_dtype=ot)
        a = w.double()[i.long()] * scale
        ref = a if p is None else a + p.double()[:i.shape[1]]
        assert got.dtype == ot
        # one rounding of the scale to fp32, of the product and of the sum
        within(got, ref, 2 * U * a.abs() + U * ref.abs() + stored(ref, ot) + 1e-44, "embed dim %d" % dim)


def test_embed_tokens_equals_the_stock_lookup_bit_for_bit():
    w, pos, ids = rnd(300, 768, seed=1), rnd(77, 768, seed=2), rints(0, 300, (9, 77), seed=3)
    assert torch.equal(ops.embed_tokens(ids, w, pos=pos), torch.nn.functional.embedding(ids, w) + pos)


def test_embed_tokens_odd_addresses_and_unknown_ids():
    V, D = 50, 64
    w = rnd(V * D + 1, seed=1)[1:].view(V, D)                       # 4-byte aligned rows
    ids = torch.tensor([[0, -1, 49, 50, 2 ** 40, -2 ** 63, 7]], device=DEV)
    got = ops.embed_tokens(ids, w)
    for t, i in enumerate(ids[0].tolist()):
        if 0 <= i < V:
            assert torch.equal(got[0, t], w[i])
        else:
            assert torch.isnan(got[0, t]).all()
    assert ops.embed_tokens(ids[:, :0], w).shape == (1, 0, D)
    assert ops.embed_tokens(ids[:0], w).shape == (0, 7, D)
    assert ops.embed_tokens(ids[0, :1], w, out_dtype=BF16).shape == (1, D)


def embed_grad_ref(ids, dy, V, scale, skip):
    """On the host: one thread adds in order (64-bit atomics on one row take minutes)."""
    flat, d = ids.reshape(-1).long().cpu(), dy.cpu().double().reshape(ids.numel(), -1)
    use = (flat >= 0) & (flat < V) & (flat != (-1 if skip is None else skip))
    flat, d = flat[use], d[use]
    dw = torch.zeros(V, d.shape[1], dtype=torch.float64).index_add_(0, flat, d) * scale
    mag = torch.zeros_like(dw).index_add_(0, flat, d.abs()) * abs(scale)
    n = torch.bincount(flat, minlength=V).double()
    return dw.to(DEV), ((n + 4)[:, None] * U * mag).to(DEV)


@pytest.mark.parametrize("S,L,V,dim,kind", [
    (1, 1, 1, 1, "random"), (1, 1, 9, 768, "random"), (1, 33, 5, 3, "random"), (160, 77, 49408, 768, "captions"), (7, 31, 1, 64, "random"),
    (3, 1000, 260, 132, "random"), (64, 65, 70000, 40, "random"), (5, 1024, 300, 8, "one"), (9, 77, 500, 1028, "sorted"), (2, 3000, 1000, 1, "two"),
    (1100, 300, 1 << 20, 4, "random"), (1, 262145, 3, 2, "random"), (700, 500, 65535, 5, "captions"), (1, 32, 8, 16, "one"), (1, 64, 8, 16, "halves")])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_embed_tokens_bwd(S, L, V, dim, kind, dt):
    ids = rints(0, V, (S, L), seed=4)
    if kind == "captions":                                          # start mark, words, end mark, zeros
        end = rints(3, 20, (S, 1), seed=5)
        t = torch.arange(L, device=DEV)[None]
        ids = torch.where(t == 0, V - 2, torch.where(t < end, ids, torch.where(t == end, V - 1, 0)))
    elif kind == "one":
        ids = torch.full((S, L), V - 1, device=DEV)
    elif kind == "two":
        ids = (ids > V // 3).long() * (V - 1)
    elif kind == "sorted":
        ids = ids.reshape(-1).sort().values.view(S, L)
    elif kind == "halves":                                          # a run that ends where a chunk of the list does
        ids = (torch.arange(S * L, device=DEV) // 32).view(S, L)
    dy = rnd(S, L, dim, seed=6, dtype=dt)
    for scale, skip, i in ((1.0, None, ids), (-2.5, 0, ids.int())):
        got, dpos = ops.embed_tokens_bwd(i, dy, V, scale=scale, skip_id=skip, pos_grad=True)
        ref, bound = embed_grad_ref(i, dy, V, scale, skip)
        within(got, ref, bound, "embed grad %s" % kind)
        assert not got[ref == 0].any()                              # rows that nothing points at: zeros, not left-overs
        within(dpos, dy.double().sum(0), (S + 2) * U * dy.double().abs().sum(0), "pos grad")
        again, dpos2 = ops.embed_tokens_bwd(i, dy, V, scale=scale, skip_id=skip, pos_grad=True)
        assert torch.equal(got, again) and torch.equal(dpos, dpos2)
    out = rnd(V, dim, seed=7)
    before = out.clone()
    res = ops.embed_tokens_bwd(ids, dy, V, scale=0.5, out=out)
    assert res.data_ptr() == out.data_ptr()
    ref, bound = embed_grad_ref(ids, dy, V, 0.5, None)
    within(out, before.double() + ref, bound + U * (before.double().abs() + ref.abs()), "embed grad, accumulated")
    assert torch.equal(out[ref == 0], before[ref == 0])


def test_embed_tokens_bwd_without_rows_and_odd_addresses():
    V, D = 40, 12
    ids = torch.tensor([[-1, 40, 2 ** 33, -7]], device=DEV)
    assert not ops.embed_tokens_bwd(ids, rnd(1, 4, D), V).any()
    for shape in ((0, 5), (3, 0)):
        e, dpos = ops.embed_tokens_bwd(ids.new_zeros(shape), rnd(*shape, D), V, pos_grad=True)
        assert e.shape == (V, D) and not e.any() and dpos.shape == (shape[1], D) and not dpos.any()
    dy = rnd(3 * 5 * D + 1, seed=2, dtype=BF16)[1:].view(3, 5, D)    # 2-byte aligned
    i = rints(0, V, (3, 5), seed=1)
    ref, bound = embed_grad_ref(i, dy, V, 1.0, None)
    within(ops.embed_tokens_bwd(i, dy, V), ref, bound, "embed grad, odd address")
    out = torch.zeros(V * D + 1, device=DEV)[1:].view(V, D)
    within(ops.embed_tokens_bwd(i, dy, V, out=out), ref, bound + U * ref.abs(), "embed grad, odd out")


def test_embed_tokens_bwd_infinities_stay_in_their_rows():
    dy = rnd(4, 8, 64, seed=1)
    dy[1, 3], dy[2, 5, 7] = float("inf"), float("nan")
    ids = torch.arange(32, device=DEV).view(4, 8)
    got = ops.embed_tokens_bwd(ids, dy, 40)
    assert torch.isinf(got[11]).all() and torch.isnan(got[21, 7])
    got[11] = got[21] = 0
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("S,L,dim", [(1, 1, 3), (7, 73, 96), (60, 17, 516), (40, 60, 541), (9, 900, 64), (160, 77, 768), (3, 4100, 33), (0, 5, 8), (4, 0, 8)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_embed_tokens_bwd_of_the_positions_alone(S, L, dim, dt):
    """A frozen table: the bits of the joint call's dpos, without its [V, D] gradient.  (One launch, both sorts' sizes, odd widths, no tokens.)"""
    V = 49408
    ids, dy = rints(-1, V + 1, (S, L), seed=1), rnd(S, L, dim, seed=2, dtype=dt)
    _, want = ops.embed_tokens_bwd(ids, dy, V, pos_grad=True)
    none, got = ops.embed_tokens_bwd(ids, dy, V, pos_grad=True, weight_grad=False)
    assert none is None and torch.equal(got, want)
    within(got, dy.double().sum(0), (S + 2) * U * dy.double().abs().sum(0), "pos grad alone")


def test_a_frozen_table_with_trained_positions():
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import token_stream as ts
    V, D, S, L = 49408, 256, 40, 60
    emb = ts.TokenEmbedding(V, D).to(DEV).requires_grad_(False)
    pos, ids, cot = nn.Parameter(rnd(L + 3, D, seed=1)), rints(0, V, (S, L), seed=2), rnd(S, L, D, seed=3)
    for trained in (False, True):
        emb.weight.requires_grad_(trained)
        emb.weight.grad = pos.grad = None
        out = emb(ids, pos, scale=3.0)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out.backward(cot)
        torch.cuda.synchronize()
        assert trained or torch.cuda.max_memory_allocated() - before < V * D * 4 // 2
        assert (emb.weight.grad is not None) == trained
        within(pos.grad[:L], cot.double().sum(0), (S + 2) * U * cot.double().abs().sum(0), "frozen table, pos grad")
        assert not pos.grad[L:].any()
    ref, bound = embed_grad_ref(ids, cot, V, 3.0, None)
    within(emb.weight.grad, ref, bound, "trained table")


# ---- the end of a residual block -------------------------------------------------------------------------------------------------------
def block_ref(x, y, gate, tanh, res, post, pre, rms, groups):
    """The definition in the inputs' type (64 bits): (x_new, h)."""
    def norm(v, gamma, beta, eps):
        c = v if rms else v - v.mean(-1, keepdim=True)
        n = c / (c.square().mean(-1, keepdim=True) + eps).sqrt() * gamma
        return n if beta is None else n + beta

    p = y if post is None else norm(y, *post)
    if gate is not None:
        g = gate.tanh() if tanh else gate
        p = p * (g.repeat_interleave(x.shape[0] // groups, 0) if g.dim() == 2 and g.shape[0] > 1 else g)
    x_new = res * x + p
    return x_new, None if pre is None else norm(x_new, *pre)


def make_block(rows, cols, gate, post, pre, rms, xt, yt, seed=0, groups=1, spread=1.0):
    s = dict(x=rnd(rows, cols, seed=seed + 1, scale=2.0, dtype=xt), y=(rnd(rows, cols, seed=seed + 2, scale=spread) + 0.3).to(yt))
    s["gate"] = {"none": None, "scalar": rnd(1, seed=3) + 0.5, "channel": rnd(cols, seed=3), "group": rnd(groups, cols, seed=3)}[gate]
    for i, name in enumerate(("post", "pre")):
        on = post if name == "post" else pre
        s[name] = (1 + 0.2 * rnd(cols, seed=10 + i), None if rms else 0.2 * rnd(cols, seed=20 + i), 1e-5 if name == "post" else 1e-6) if on else None
    return s


def dbl(v, grad=False):
    return None if v is None else v.double().requires_grad_(grad)


def dnorm(n, grad=False):
    return None if n is None else (dbl(n[0], grad), dbl(n[1], grad), n[2])


def norm_error(v, e, n, rms, ref):
    """Bound on the error of a norm of v in fp32 whose input is off by e (element by element), n = (gamma, beta, eps): a mean is off by at most M U of the mean
    magnitude, with M = 48 above the depth of any sum here (16 or fewer terms in a lane, 6 + 2 exchanges, the divisions), and so on through the formula."""
    M = 48 * U
    c = v if rms else v - v.mean(-1, keepdim=True)
    r = 1 / (c.square().mean(-1, keepdim=True) + n[2]).sqrt()
    de = e + (0 if rms else e.mean(-1, keepdim=True) + M * v.abs().mean(-1, keepdim=True) + U * v.abs())
    xh = (c * r).abs()
    dr = M + r * (de.square().mean(-1, keepdim=True)).sqrt()         # relative error of r
    return n[0].abs() * (r * de + xh * dr) + 8 * U * (n[0].abs() * xh + ref.abs())


CASES = [(1, 1, "none"), (9, 2, "channel"), (12, 3, "group"), (33, 6, "scalar"), (50, 1023, "channel"), (5, 4093, "none"), (3, 5, "scalar"), (7, 64, "channel"), (37, 255, "group"), (64, 256, "none"), (40, 257, "group"), (416, 512, "scalar"), (130, 768, "group"),
         (77, 1000, "channel"), (33, 1024, "channel"), (9, 1025, "scalar"), (12, 2048, "group"), (5, 2051, "channel"), (3, 4096, "none"), (2, 4095, "group")]


@pytest.mark.parametrize("rows,cols,gate", CASES)
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("rms,xt,yt,ht", [(False, F32, BF16, BF16), (True, BF16, F32, F32)])
def test_residual_norm(rows, cols, gate, post, pre, rms, xt, yt, ht):
    groups = {37: 37, 40: 8, 130: 10, 12: 3, 2: 2}.get(rows, 1)
    s = make_block(rows, cols, gate, post, pre, rms, xt, yt, groups=groups)
    tanh, res = cols % 2 == 0, 0.75 if cols % 3 else 1.0
    x0 = s["x"].clone()
    x_new, h = ops.residual_norm(s["x"], s["y"], gate=s["gate"], gate_tanh=tanh, res_scale=res, post=s["post"], pre=s["pre"], rms=rms, out_dtype=ht)
    assert torch.equal(s["x"], x0) and x_new.dtype == xt
    y, g, po, pr = s["y"].double(), dbl(s["gate"]), dnorm(s["post"]), dnorm(s["pre"])
    rx, rh = block_ref(s["x"].double(), y, g, tanh, res, po, pr, rms, groups)
    branch, _ = block_ref(torch.zeros_like(y), y, g, tanh, res, po, None, rms, groups)
    e = 0
    if post:
        only, _ = block_ref(torch.zeros_like(y), y, None, False, res, po, None, rms, groups)
        gg = 1.0 if g is None else (g.tanh() if tanh else g).abs()
        gg = gg.repeat_interleave(rows // groups, 0) if g is not None and g.dim() == 2 and groups > 1 else gg
        e = gg * norm_error(y, torch.zeros_like(y), po, rms, only)
    e = e + 8 * U * (branch.abs() + (res * s["x"].double()).abs() + rx.abs())      # tanh (4 steps), products, the sum
    within(x_new, rx, e + stored(rx, xt), "residual_norm x_new")
    if pre:
        assert h.dtype == ht
        within(h, rh, norm_error(rx, e, pr, rms, rh) + stored(rh, ht), "residual_norm h")
    else:
        assert h is None
    same, h2 = ops.residual_norm(s["x"], s["y"], gate=s["gate"], gate_tanh=tanh, res_scale=res, post=s["post"], pre=s["pre"], rms=rms, out_dtype=ht, out=s["x"])
    assert same.data_ptr() == s["x"].data_ptr() and torch.equal(same, x_new) and (h is None or torch.equal(h, h2))


@pytest.mark.parametrize("rows,cols,gate", CASES + [(3000, 64, "channel"), (2600, 200, "group"), (9000, 24, "scalar"), (4000, 1024, "channel")])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("rms,xt,yt,ht", [(False, F32, BF16, BF16), (True, BF16, F32, F32), (False, BF16, BF16, F32)])
def test_residual_norm_bwd(rows, cols, gate, post, pre, rms, xt, yt, ht):
    groups = {37: 37, 40: 8, 130: 10, 12: 3, 2: 2, 2600: 1300}.get(rows, 1)
    s = make_block(rows, cols, gate, post, pre, rms, xt, yt, groups=groups)
    tanh, res = cols % 2 == 0, 0.75 if cols % 3 else 1.0
    dxn, dh = rnd(rows, cols, seed=31, dtype=xt), rnd(rows, cols, seed=32, dtype=ht) if pre else None
    got = ops.residual_norm_bwd(s["x"], s["y"], dxn, dh, gate=s["gate"], gate_tanh=tanh, res_scale=res, post=s["post"], pre=s["pre"], rms=rms)
    again = ops.residual_norm_bwd(s["x"], s["y"], dxn, dh, gate=s["gate"], gate_tanh=tanh, res_scale=res, post=s["post"], pre=s["pre"], rms=rms)
    for a, b in zip(got, again):
        assert (a is None) == (b is None) and (a is None or torch.equal(a, b))
    # autograd of the definition, at the x that gives this x_new
    y, g, po, pr = dbl(s["y"], True), dbl(s["gate"], True), dnorm(s["post"], True), dnorm(s["pre"], True)
    with torch.no_grad():
        branch, _ = block_ref(torch.zeros(rows, cols, dtype=torch.float64, device=DEV), y, g, tanh, res, po, None, rms, groups)
    x = ((s["x"].double() - branch) / res).requires_grad_(True)
    rx, rh = block_ref(x, y, g, tanh, res, po, pr, rms, groups)
    leaves = [x, y, g] + [t for n in (po, pr) for t in ((None, None) if n is None else n[:2])]
    outs, grads = ([rx], [dxn.double()]) if rh is None else ([rx, rh], [dxn.double(), dh.double()])
    found = iter(torch.autograd.grad(outs, [t for t in leaves if t is not None], grads))
    refs = [None if t is None else next(found) for t in leaves]
    # magnitudes of the terms that the formulas add, element by element: d = dx_new + r (k - mean k - xh mean(k xh)), dy the same of g o d
    M = 160 * U                                                      # above all roundings on a term's way: two statistics (48 each), two row means, products

    def parts(v, k, n):
        c = v if rms else v - v.mean(-1, keepdim=True)
        r = 1 / (c.square().mean(-1, keepdim=True) + n[2]).sqrt()
        xh = (c * r).abs() + r * (0 if rms else v.abs().mean(-1, keepdim=True))      # (its error: the mean's, and v's own rounding)
        return r * (k + (0 if rms else k.mean(-1, keepdim=True)) + xh * (k * xh).mean(-1, keepdim=True) * 3), xh
    with torch.no_grad():
        D = dxn.double().abs()
        if pre:
            t, xh2 = parts(rx, dh.double().abs() * pr[0].abs(), pr)
            D = D + t
        gg = torch.ones((), dtype=torch.float64, device=DEV) if g is None else (g.tanh() if tanh else g).abs()
        gg = gg.repeat_interleave(rows // groups, 0) if g is not None and g.dim() == 2 and groups > 1 else gg
        P, Y, xh1 = y.abs(), gg * D, None
        if post:
            t, xh1 = parts(y, gg * D * po[0].abs(), po)
            Y = t
            P = po[0].abs() * xh1 + (0 if po[1] is None else po[1].abs())
        within(got.dx, refs[0], M * res * D + stored(refs[0], xt), "residual_norm dx")
        within(got.dy, refs[1], 2 * M * Y + stored(refs[1], yt), "residual_norm dy")
        N = M + (rows + 64) * U                                      # a column sum over the rows
        if g is not None:
            T = D * P
            T = T.sum().view(1) if gate == "scalar" else T.sum(0) if gate == "channel" or groups == 1 else T.view(groups, -1, cols).sum(1)
            n = N + cols * U if gate == "scalar" else N
            within(got.dgate, refs[2], (2 * n * T).view_as(refs[2]) + 1e-30, "residual_norm dgate")
        for name, ref, mag in (("dpost_gamma", refs[3], (lambda: gg * D * xh1)), ("dpost_beta", refs[4], (lambda: gg * D)), ("dpre_gamma", refs[5], (lambda: dh.double().abs() * xh2)),
                               ("dpre_beta", refs[6], (lambda: dh.double().abs()))):
            v = getattr(got, name)
            assert (v is None) == (ref is None), name
            if ref is not None:
                within(v, ref, 2 * N * (mag() * torch.ones_like(rx)).sum(0) + 1e-30, "residual_norm " + name)


@pytest.mark.parametrize("rows,cols,groups", [(16504, 1024, 4), (17003, 1000, 1), (8402, 2048, 2), (33500, 512, 1), (16801, 1023, 1), (24002, 770, 2),
                                              (104002, 1024, 2), (215000, 512, 1), (430001, 256, 1)])
@pytest.mark.parametrize("post,pre", [(True, True), (False, True), (True, False)])
def test_residual_norm_of_large_calls(rows, cols, groups, post, pre):
    """Over 96 MB of outputs the non-temporal kernels, over 600 MB of gradients four rows at a time, against the same rows in calls of a few thousand (whose kernels the tests above hold to their
    definition).  Rows are independent, so that they agree bit for bit up to the order of a sum over a row's waves, which is the same; column sums to their bound."""
    gate = "group" if groups > 1 else "channel"
    s = make_block(rows, cols, gate, post, pre, False, F32, BF16, groups=groups)
    kw = dict(res_scale=0.75, post=s["post"], pre=s["pre"], gate_tanh=True)
    dxn, dh = rnd(rows, cols, seed=31), rnd(rows, cols, seed=32, dtype=BF16) if pre else None
    x_new, h = ops.residual_norm(s["x"], s["y"], gate=s["gate"], **kw)
    got = ops.residual_norm_bwd(s["x"], s["y"], dxn, dh, gate=s["gate"], **kw)
    sums = None
    cut = lambda t, i, j: None if t is None else t[i:j].contiguous()  # noqa: E731
    each = rows // groups
    for k in range(groups):
        for i in range(k * each, (k + 1) * each, 2100):
            j = min(i + 2100, (k + 1) * each)
            g = s["gate"][k] if groups > 1 else s["gate"]
            a, b = ops.residual_norm(cut(s["x"], i, j), cut(s["y"], i, j), gate=g, **kw)
            assert torch.equal(a, x_new[i:j]) and (h is None or torch.equal(b, h[i:j]))
            p = ops.residual_norm_bwd(cut(s["x"], i, j), cut(s["y"], i, j), cut(dxn, i, j), cut(dh, i, j), gate=g, **kw)
            assert torch.equal(p.dx, got.dx[i:j]) and torch.equal(p.dy, got.dy[i:j])
            add = [None if t is None else t.double() for t in p[2:]]
            if groups > 1:
                rest = torch.zeros(groups, cols, dtype=torch.float64, device=DEV)
                rest[k] = add[0]
                add[0] = rest
            sums = add if sums is None else [None if t is None else t + v for t, v in zip(sums, add)]
    for name, t, v in zip(got._fields[2:], got[2:], sums):
        assert (t is None) == (v is None)
        if t is not None:                                           # both sides add about `rows` terms of a size near 1 (xh, dh, d, gammas) in fp32
            assert float((t.double() - v).abs().max()) <= 2 * (rows + 64) * U * 40 * rows ** 0.5, name


def test_large_outputs_of_embed_and_act8():
    """Over 96 MB: the non-temporal kernels give what calls on a part of the rows give."""
    w, pos, ids = rnd(1000, 1024, seed=1), rnd(77, 1024, seed=2), rints(0, 1000, (420, 77), seed=3)
    for ot in (F32, BF16):
        for wt in (F32, BF16):
            n = 420 if ot == F32 else 840
            i = ids.repeat(n // 420, 1)
            big = ops.embed_tokens(i, w.to(wt), scale=3.0, pos=pos, out_dtype=ot)
            assert big.numel() * big.element_size() > 96 << 20
            assert torch.equal(big[-3:], ops.embed_tokens(i[-3:], w.to(wt), scale=3.0, pos=pos, out_dtype=ot))
            assert torch.equal(big[:100], ops.embed_tokens(i[:100], w.to(wt), scale=3.0, pos=pos, out_dtype=ot))
    for dt, rows, cols in ((F32, 13000, 2048), (BF16, 26000, 2056)):
        u, da = rnd(rows, cols, seed=4, dtype=dt), rnd(rows, cols, seed=5, dtype=dt)
        a, q, sc = ops.act8(u, ops.ACT_QUICKGELU)
        du, a2 = ops.act8_bwd(q, sc, da, ops.ACT_QUICKGELU, want_out=True)
        for i in (slice(0, 50), slice(rows - 50, rows)):
            b, r, t = ops.act8(u[i].contiguous(), ops.ACT_QUICKGELU)
            assert torch.equal(a[i], b) and torch.equal(q[i].view(torch.uint8), r.view(torch.uint8)) and torch.equal(sc[i], t)
            dv, b2 = ops.act8_bwd(r, t, da[i].contiguous(), ops.ACT_QUICKGELU, want_out=True)
            assert torch.equal(du[i], dv) and torch.equal(a2[i], b2)
    dy = rnd(340, 77, 2048, seed=6, dtype=BF16)                      # a gradient over 96 MB with positions: read past the cache
    assert dy.numel() * 2 > 96 << 20
    i = rints(0, 5000, (340, 77), seed=7)
    dw, dpos = ops.embed_tokens_bwd(i, dy, 5000, pos_grad=True)
    ref, bound = embed_grad_ref(i, dy, 5000, 1.0, None)
    within(dw, ref, bound, "embed grad, large")
    within(dpos, dy.double().sum(0), 342 * U * dy.double().abs().sum(0), "pos grad, large")


def test_residual_norm_bwd_against_differences():
    """A directional derivative of the kernels' own forward (fp32 in and out) against the gradients: central differences of step t are off by t^2 / 6 of the third
    derivative (below 50 of the sizes here: unit rows, gammas near 1) and by the forward's rounding / t."""
    rows, cols = 24, 96
    s = make_block(rows, cols, "channel", True, True, False, F32, F32)
    cx, ch = rnd(rows, cols, seed=41), rnd(rows, cols, seed=42)
    loss = lambda x, y, gate, post, pre: sum((a.double() * c.double()).sum() for a, c in zip(ops.residual_norm(x, y, gate=gate, gate_tanh=True, res_scale=0.8, post=post, pre=pre, out_dtype=F32), (cx, ch)))  # noqa: E731
    x_new, _ = ops.residual_norm(s["x"], s["y"], gate=s["gate"], gate_tanh=True, res_scale=0.8, post=s["post"], pre=s["pre"], out_dtype=F32)
    g = ops.residual_norm_bwd(x_new, s["y"], cx, ch, gate=s["gate"], gate_tanh=True, res_scale=0.8, post=s["post"], pre=s["pre"])
    base = [s["x"], s["y"], s["gate"], s["post"][0], s["post"][1], s["pre"][0], s["pre"][1]]
    dirs = [rnd(*t.shape, seed=50 + i) for i, t in enumerate(base)]
    t = 2.0 ** -8

    def at(k, sign):
        v = [b + sign * t * d if i == k else b for i, (b, d) in enumerate(zip(base, dirs))]
        return loss(v[0], v[1], v[2], (v[3], v[4], 1e-5), (v[5], v[6], 1e-6))
    for k, (grad, d) in enumerate(zip(g, dirs)):
        num = float((at(k, 1) - at(k, -1)) / (2 * t))
        ana = float((grad.double() * d.double()).sum())
        size = float((grad.double() * d.double()).abs().sum())
        assert abs(num - ana) <= (50 * t * t / 6 + 64 * U / t) * size + 64 * U / t * (rows * cols) ** 0.5, (k, num, ana)


def test_residual_norm_without_dx_new_without_rows_and_with_infinities():
    s = make_block(6, 128, "channel", True, True, False, F32, BF16)
    dh = rnd(6, 128, seed=9, dtype=BF16)
    kw = dict(gate=s["gate"], post=s["post"], pre=s["pre"])
    a = ops.residual_norm_bwd(s["x"], s["y"], None, dh, **kw)
    b = ops.residual_norm_bwd(s["x"], s["y"], torch.zeros_like(s["x"]), dh, **kw)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for gate in ("scalar", "channel"):
        e = make_block(0, 128, gate, True, True, False, F32, BF16)
        assert ops.residual_norm(e["x"], e["y"], gate=e["gate"], post=e["post"], pre=e["pre"])[1].shape == (0, 128)
        for t in ops.residual_norm_bwd(e["x"], e["y"], None, dh[:0], gate=e["gate"], post=e["post"], pre=e["pre"])[2:]:
            assert not t.any()
    x = s["x"].clone()
    x[2, 5], x[4, 100] = float("inf"), float("nan")
    _, h = ops.residual_norm(x, s["y"], **kw)
    _, clean = ops.residual_norm(s["x"], s["y"], **kw)
    assert torch.isnan(h[4]).all() and torch.isnan(h[2, 5])
    keep = [0, 1, 3, 5]
    assert torch.equal(h[keep], clean[keep])
    const = torch.full((3, 100), 7.25, device=DEV)                   # a row without variance: the norm gives its beta
    beta = rnd(100, seed=1)
    _, h = ops.residual_norm(const, torch.zeros_like(const), pre=(torch.ones(100, device=DEV), beta, 1e-5), out_dtype=F32)
    assert float((h - beta).abs().max()) <= 48 * U * 7.25 / 1e-5 ** 0.5


# ---- activations in 8 bits -------------------------------------------------------------------------------------------------------------
def act8_ref(u):
    """(values in units of the scale, scale) by whole-number arithmetic on the exponents, in 64 bits."""
    rows, cols = u.shape
    G = -(-cols // 128)
    v = torch.zeros(rows, G * 128, dtype=torch.float64)
    v[:, :cols] = u.detach().cpu().double()
    v = v.view(rows, G, 128)
    top = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(-1)
    m, e = torch.frexp(top)
    k = torch.where(top > 0, (e - 9 + (m > 0.875).int()).clamp(-117, 120), 0)
    w = torch.ldexp(v, -k[..., None])
    _, ew = torch.frexp(w.abs().clamp_min(2.0 ** -6))
    step = torch.ldexp(torch.ones_like(w), ew - 4)
    q = torch.where(torch.isfinite(w), torch.round(w / step) * step, float("nan"))
    return q.view(rows, G * 128)[:, :cols], torch.ldexp(torch.ones_like(top), k)


def act_ref(v, act):
    if act == ops.ACT_QUICKGELU:
        s = 1 / (1 + torch.exp(-1.702 * v))
        return v * s, s * (1 + 1.702 * v * (1 - s))
    if act == ops.ACT_RELU:
        return v.clamp_min(0), (v > 0).double()
    return v, torch.ones_like(v)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (5, 127), (33, 128), (7, 129), (416, 2048), (19, 1000), (64, 4096), (3, 136), (2, 4104)])
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_QUICKGELU, ops.ACT_RELU])
def test_act8(rows, cols, dt, act):
    u = (rnd(rows, cols, seed=1) * torch.exp(3 * rnd(rows, 1, seed=2))).to(dt)
    da = rnd(rows, cols, seed=3, dtype=dt)
    a, q, s = ops.act8(u, act)
    qr, sr = act8_ref(u)
    assert torch.equal(q.double().cpu(), qr) and torch.equal(s.double().cpu(), sr)
    none, q2, s2 = ops.act8(u, act, want_out=False)
    assert none is None and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    # exp within 4 steps and its argument (1.702 rounded, the product) within 2 U of itself, which exp turns into |1.702 v| times as much
    slack = lambda v: (16 + 4 * (1.702 * v).abs().clamp_max(100)) * U  # noqa: E731
    # a reciprocal below fp32's smallest normal number, 2^-126, is zero: a sigmoid there (v below -51.3) loses at most 2^-126 of what multiplies it
    tiny = 2.0 ** -125
    ud = u.double()
    ra, _ = act_ref(ud, act)
    within(a, ra, (slack(ud) * ra.abs() if act == ops.ACT_QUICKGELU else 0) + stored(ra, dt) * (act == ops.ACT_QUICKGELU) + tiny * (1 + ud.abs()), "act8 a")
    v = qr.to(DEV) * sr.to(DEV).repeat_interleave(128, 1)[:, :cols]
    rv, slope = act_ref(v, act)
    du, a2 = ops.act8_bwd(q, s, da, act, want_out=True)
    du2 = ops.act8_bwd(q, s, da, act)
    assert torch.equal(du, du2)
    ref = da.double() * slope
    mag = da.double().abs() * (slope.abs() if act != ops.ACT_QUICKGELU else (lambda g: g * (1 + 1.702 * v.abs() * (1 - g)) + g)(1 / (1 + torch.exp(-1.702 * v))))
    within(du, ref, slack(v) * mag + stored(ref, dt) + tiny * (1 + da.double().abs() * (1 + 1.702 * v.abs())), "act8 du")
    within(a2, rv, slack(v) * rv.abs() + stored(rv, dt) + tiny * (1 + v.abs()), "act8 a again")


def test_act8_borders_of_the_scale():
    rows = [448.0, 448.0 + 2 ** -14, 449.0, 1.75, 1.75 * (1 + 2 ** -23), 2.0, 1.0, 2.0 ** -126, 2.0 ** -140, 2.0 ** -149, 3.4e38, 2.0 ** 127, 1.75 * 2.0 ** 127, 0.0, 240.0, 464.0, 2.0 ** -118, 1e-30]
    u = torch.zeros(len(rows), 130)
    for i, t in enumerate(rows):
        u[i, :128] = t * torch.linspace(-1, 1, 128)
        u[i, 7], u[i, 128], u[i, 129] = t, -t, t / 3
    _, q, s = ops.act8(u.to(DEV), want_out=False)
    qr, sr = act8_ref(u)
    assert torch.equal(s.double().cpu(), sr) and torch.equal(q.double().cpu(), qr)
    assert float(q.double().abs().max()) <= 448
    # every value that e4m3 has, and every middle between two: ties go to the even one
    code = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    grid = code[torch.isfinite(code)].unique()
    vals = torch.cat([grid, (grid[1:] + grid[:-1]) / 2])
    pad = (-len(vals)) % 126
    blocks = torch.cat([vals, vals.new_zeros(pad)]).view(-1, 126)
    blocks = torch.cat([blocks, blocks.new_full((len(blocks), 2), 448.0)], 1).float()
    _, q, s = ops.act8(blocks.to(DEV), want_out=False)
    qr, sr = act8_ref(blocks)
    assert (s == 1).all() and torch.equal(q.double().cpu(), qr)


def test_act8_infinities_and_nan_touch_nothing_else():
    u = rnd(4, 300, seed=1)
    _, q0, s0 = ops.act8(u, want_out=False)
    v = u.clone()
    v[0, 3], v[1, 130], v[2, 299] = float("inf"), float("-inf"), float("nan")
    v[3, :128] = float("nan")
    a, q, s = ops.act8(v, ops.ACT_RELU)
    bad = ~torch.isfinite(v)
    assert torch.isnan(q.float()[bad]).all() and torch.isfinite(q.float()[~bad]).all() and float(s[3, 0]) == 1
    qr, sr = act8_ref(v)
    assert torch.equal(s.double().cpu(), sr) and torch.equal(torch.nan_to_num(q.double().cpu()), torch.nan_to_num(qr))
    assert float(a[0, 3]) == float("inf") and float(a[1, 130]) == 0 and torch.isnan(a[2, 299])
    du = ops.act8_bwd(q, s, torch.ones_like(v), ops.ACT_QUICKGELU)
    assert torch.isnan(du[bad]).all() and torch.isfinite(du[~bad]).all()
    for shape in ((0, 64),):
        a, q, s = ops.act8(torch.zeros(shape, device=DEV), ops.ACT_RELU)
        assert a.shape == shape and q.shape == shape and s.shape == (0, 1) and ops.act8_bwd(q, s, a, ops.ACT_RELU).shape == shape
    odd = rnd(5 * 64 + 1, seed=3, dtype=BF16)[1:].view(5, 64)         # 2-byte aligned
    a, q, s = ops.act8(odd, ops.ACT_RELU)
    b, r, t = ops.act8(odd.clone(), ops.ACT_RELU)
    assert torch.equal(a, b) and torch.equal(q.view(torch.uint8), r.view(torch.uint8)) and torch.equal(s, t)


@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_QUICKGELU, ops.ACT_RELU])
@pytest.mark.parametrize("dt", [F32, BF16])
@pytest.mark.parametrize("cols", [128, 131, 5])
def test_act8_bwd_shows_what_was_infinite_or_nan(act, dt, cols):
    """A checkpoint holds infinities and NaN as NaN, and so does every gradient (and activation) that uses them, whatever the activation; their neighbours are as without them."""
    u, da = rnd(6, cols, seed=1, dtype=dt), rnd(6, cols, seed=2, dtype=dt).abs() + 0.5
    bad = torch.zeros(6, cols, dtype=torch.bool, device=DEV)
    v = u.clone()
    for r, c, t in ((0, 0, "inf"), (1, 3, "-inf"), (2, cols - 1, "nan"), (4, 2, "inf")):
        v[r, c], bad[r, c], u[r, c] = float(t), True, 0              # (zero: counts for no scale either)
    _, q, s = ops.act8(v, act)
    _, q0, s0 = ops.act8(u, act)
    assert torch.equal(s, s0)
    du, a = ops.act8_bwd(q, s, da, act, want_out=True)
    du0, a0 = ops.act8_bwd(q0, s0, da, act, want_out=True)
    assert torch.isnan(du[bad]).all() or act == ops.ACT_NONE
    assert torch.isnan(a[bad]).all()
    assert torch.equal(du[~bad], du0[~bad]) and torch.equal(a[~bad], a0[~bad])
    if act == ops.ACT_NONE:                                          # (a slope of one whatever the value)
        assert torch.equal(du, da)


@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_QUICKGELU, ops.ACT_RELU])
def test_act8_bwd_at_the_ends_of_the_range(act):
    """Finite activations up to fp32's largest.  From 1.9375 * 2^127 on (248 of a scale of 2^120: e4m3's middle between 240 and 256) a value rounds to 2^128, infinity in fp32;
    the slope there is that of the far end, 1 or 0, and no other value is infinite."""
    top = 3.402823466e38
    border = 1.9375 * 2.0 ** 127
    below = float(torch.tensor(border).nextafter(torch.tensor(0.0)))
    vals = [top, border, below, 3e38, 2.9e38, 2.5e38, 2e38, 1.9e38, 1e38, 2.0 ** 100, 1e10, 200.0, 128.0, 60.0, 52.0]
    u = torch.tensor([[v, -v] for v in vals], device=DEV)
    da = torch.full_like(u, 0.75)
    _, q, s = ops.act8(u, act)
    qr, sr = act8_ref(u)
    assert torch.equal(q.double().cpu(), qr) and torch.equal(s.double().cpu(), sr)
    du, a = ops.act8_bwd(q, s, da, act, want_out=True)
    v = (qr * sr).to(DEV)                                            # 64 bits: finite
    assert (v.abs() >= 2.0 ** 128).sum() == 4
    rv, slope = act_ref(v, act)
    pos = torch.where(v.abs() >= 2.0 ** 128, float("inf"), rv.abs()) * torch.sign(v)
    if act == ops.ACT_NONE:
        assert torch.equal(du, da) and torch.equal(a.double(), pos)
    else:
        assert torch.equal(du[:, 0], da[:, 0])                       # (the slope at 52 and above is 1 to fp32)
        assert (du[:, 1].abs() <= 2.0 ** -60).all()                  # e^(-1.702 * 52) < 2^-127, times 90
        assert torch.equal(a[:, 0].double(), pos[:, 0]) and (a[:, 1].abs() <= 2.0 ** -60).all()


def values(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, :q.shape[1]]


def check_wgrad(dy, q, s, what):
    dw, db = ops.gemm_tn_act8(dy, q, s, colsum=True)
    K = dy.shape[0]
    v, d = values(q, s), dy.double()
    # exact products, K of them added in fp32 (the matrix core may truncate where an addition rounds: 2 U each)
    within(dw, d.t() @ v, 2 * (K + 8) * U * (d.abs().t() @ v.abs()) + 1e-38, what)
    within(db, d.sum(0), 2 * (K + 8) * U * d.abs().sum(0) + 1e-38, what + " db")
    rel = float((dw.double() - d.t() @ v).norm() / ((d.t() @ v).norm() + 1e-300))
    assert rel <= 4 * U * max(K, 16) ** 0.5, (what, rel)             # independent roundings grow as the root of their number
    assert torch.equal(ops.gemm_tn_act8(dy, q, s), dw)
    return dw, db


@pytest.mark.parametrize("K,M,N", [(1, 1, 1), (1, 128, 128), (64, 128, 128), (63, 8, 16), (65, 130, 144), (2464, 768, 768), (513, 256, 384), (1000, 77, 131), (4097, 128, 2048), (77, 512, 128),
                                   (130, 1000, 40), (3, 264, 272), (8200, 200, 136), (257, 129, 1000)])
def test_gemm_tn_act8(K, M, N):
    u = rnd(K, N, seed=1, dtype=BF16) * torch.exp(2 * rnd(K, 1, seed=2)).to(BF16)
    _, q, s = ops.act8(u, want_out=False)
    check_wgrad(rnd(K, M, seed=3, dtype=BF16), q, s, "act8 wgrad")


@pytest.mark.parametrize("K,M,N", [(102000, 264, 272), (205001, 136, 400), (16503, 1030, 1037), (68000, 512, 520), (40961, 768, 1024), (4200, 4100, 4099), (700, 3600, 3500)])
def test_gemm_tn_act8_in_large_tiles(K, M, N):
    """Enough tokens and outputs for the 256 x 256 tiles: slices that end inside a tile, slices without a token, ragged outputs, unaligned rows."""
    tiles = -(-M // 256) * -(-N // 256)
    assert tiles >= 192 or tiles * -(-K // 1024) >= 400
    u = rnd(K, N, seed=1, dtype=BF16) * torch.exp(rnd(K, 1, seed=2)).to(BF16)
    _, q, s = ops.act8(u, want_out=False)
    check_wgrad(rnd(K, M, seed=3, dtype=BF16), q, s, "act8 wgrad, large tiles")


def test_gemm_tn_act8_takes_every_code_and_scale_exactly():
    """dy = unit rows: the product is the operand itself."""
    codes = torch.arange(256, dtype=torch.uint8)
    codes = codes[torch.isfinite(codes.view(torch.float8_e4m3fn).float())]
    q = codes.repeat(2)[:256].repeat(64, 1).to(DEV).view(torch.float8_e4m3fn)
    k = torch.arange(64) * 3 - 117
    s = torch.ldexp(torch.ones(64), torch.stack([k, 117 - k], 1).T.contiguous()).T.contiguous().clamp(2.0 ** -117, 2.0 ** 100).to(DEV)
    dw = ops.gemm_tn_act8(torch.eye(64, device=DEV, dtype=BF16), q, s)
    assert torch.equal(dw.double(), values(q, s))


def test_gemm_tn_act8_views_bounds_and_empty():
    K, M, N = 300, 136, 144
    base, dyb = rnd(K, 3 * 256, seed=1), rnd(K, 400, seed=2, dtype=BF16)
    _, q, s = ops.act8(base, want_out=False)
    dy = dyb[:, 8:8 + M]
    big = q[:, 256:256 + N]                                         # the columns of a wider checkpoint, with their scales
    sc = s[:, 2:4].contiguous()
    a = ops.gemm_tn_act8(dy, big, sc)
    b = ops.gemm_tn_act8(dy.contiguous(), big.contiguous(), sc)
    assert torch.equal(a, b)
    c = ops.gemm_tn_act8(dyb[:, 3:3 + M], big, sc)                   # 2-byte aligned rows
    assert torch.equal(c, ops.gemm_tn_act8(dyb[:, 3:3 + M].contiguous(), big, sc))
    out = torch.full((M, N), 7.0, device=DEV)
    assert ops.gemm_tn_act8(dy, big, sc, out=out).data_ptr() == out.data_ptr() and torch.equal(out, a)
    dw, db = ops.gemm_tn_act8(dy[:0], big[:0], sc[:0], colsum=True)
    assert dw.shape == (M, N) and not dw.any() and not db.any()
    pad = torch.full((M + 1, N), 3.0, device=DEV)
    ops.gemm_tn_act8(dy, big, sc, out=pad[:M])
    assert (pad[M] == 3).all()


def placed(t, offset, junk):
    """t's values in a buffer that is `junk` before and behind them, `offset` elements from its (aligned) begin."""
    raw = torch.full((t.numel() + offset + 32,), junk, dtype=torch.uint8 if t.element_size() == 1 else torch.int16, device=DEV)
    raw[offset:offset + t.numel()] = t.contiguous().view(-1).view(raw.dtype)
    return raw[offset:offset + t.numel()].view(t.dtype).view(t.shape)


@pytest.mark.parametrize("K,M,N", [(1, 3, 5), (33, 7, 21), (63, 129, 131), (101, 40, 1001), (1101, 77, 145), (16503, 1031, 1037)])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_gemm_tn_act8_any_address_and_nan_around_the_operands(K, M, N, offset):
    """Rows that begin at every byte, in buffers whose other bytes are NaN: nothing but the operands counts."""
    _, q, s = ops.act8(rnd(K, N, seed=1, dtype=BF16), want_out=False)
    dy = rnd(K, M, seed=3, dtype=BF16)
    want = check_wgrad(dy, q, s, "act8 wgrad")
    got = ops.gemm_tn_act8(placed(dy, offset, 0x7fff), placed(q, offset, 0x7f), s, colsum=True)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("rows,cols", [(5, 3), (9, 130), (33, 1001), (64, 768)])
def test_act8_at_any_address(rows, cols):
    for dt in (F32, BF16):
        u, da = rnd(rows * cols + 1, seed=4, dtype=dt), rnd(rows * cols + 1, seed=5, dtype=dt)
        a, q, s = ops.act8(u[1:].view(rows, cols), ops.ACT_QUICKGELU)
        for x, y in zip((a, q, s), ops.act8(u[1:].clone().view(rows, cols), ops.ACT_QUICKGELU)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        du, b = ops.act8_bwd(placed(q, 1, 0x7f), s, da[1:].view(rows, cols), ops.ACT_QUICKGELU, want_out=True)
        for x, y in zip((du, b), ops.act8_bwd(q, s, da[1:].clone().view(rows, cols), ops.ACT_QUICKGELU, want_out=True)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("S,L,V,dim", [(3, 50, 9, 2), (5, 77, 30, 7), (40, 60, 12, 541), (64, 77, 40, 1031)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_embed_tokens_bwd_adds_once_where_pieces_share_channels(S, L, V, dim, dt):
    """Whole numbers, whose sums are exact in any order: rows of a width that no wide access divides, added to what is there, equal the stock sum."""
    ids, dy = rints(0, V, (S, L), seed=4), rints(-8, 9, (S, L, dim), seed=5).to(dt)
    out = rints(-100, 100, (V, dim), seed=6).to(F32)
    want = out.double().index_add(0, ids.view(-1), dy.view(-1, dim).double())
    assert torch.equal(ops.embed_tokens_bwd(ids, dy, V, out=out).double(), want)
    dw, dpos = ops.embed_tokens_bwd(ids, dy, V, pos_grad=True)
    assert torch.equal(dw.double(), torch.zeros(V, dim, dtype=torch.float64, device=DEV).index_add(0, ids.view(-1), dy.view(-1, dim).double()))
    assert torch.equal(dpos.double(), dy.double().sum(0))


@pytest.mark.parametrize("S,L,V,dim", [(1, 512, 40, 768), (512, 1, 3, 2052), (16, 32, 49408, 12), (7, 73, 33000, 1), (3, 171, 700000, 3), (2, 9, 4, 70000), (1, 1, 40000000, 4),
                                       (513, 1, 60, 5), (64, 64, 300, 33), (17, 241, 20, 8), (3, 1366, 49408, 16), (128, 64, 2000, 12), (8193, 1, 70, 4),
                                       (91, 101, 9000, 5), (30, 1000, 29999, 3), (8, 128, 700, 33), (1, 1024, 60, 512), (32, 32, 9, 1024), (13, 77, 60, 516), (41, 25, 90, 64), (5, 2000, 9999, 770)])
@pytest.mark.parametrize("dt", [F32, BF16])
def test_embed_tokens_bwd_of_few_tokens(S, L, V, dim, dt):
    """One launch (up to 512 or 1024 tokens), a sort by counting (8192) and just over, tables of many rows or wide ones: whole numbers, so that the stock sums are exact."""
    ids = rints(-2, V + 2, (S, L), seed=4)
    ids[0, 0] = V - 1
    if S * L > 100:
        ids[:, L // 2:] = min(5, V - 1)                             # one id has most of the tokens
    dy = rints(-8, 9, (S, L, dim), seed=5).to(dt)
    known = (ids >= 0) & (ids < V) & (ids != 1)
    want = torch.zeros(V, dim, device=DEV)
    want.index_add_(0, ids[known], dy[known].float() * 0.5)
    for i in (ids, ids.int()):
        dw, dpos = ops.embed_tokens_bwd(i, dy, V, scale=0.5, skip_id=1, pos_grad=True)
        assert torch.equal(dw, want) and torch.equal(dpos, dy.float().sum(0))
    out = torch.full((V, dim), 3.0, device=DEV)
    ops.embed_tokens_bwd(ids, dy, V, scale=0.5, skip_id=1, out=out)
    assert torch.equal(out, want + 3)


# ---- streams, graphs, the operators together -------------------------------------------------------------------------------------------
def one_pass(t):
    """Embedding, the end of a block, an activation and its checkpoint, and their backward passes: every output."""
    x = ops.embed_tokens(t["ids"], t["w"], scale=2.0, pos=t["pos"])
    x2 = x.view(-1, x.shape[-1])
    xn, h = ops.residual_norm(x2, t["y"], gate=t["gate"], gate_tanh=True, res_scale=0.9, post=t["post"], pre=t["pre"])
    a, q, s = ops.act8(h, ops.ACT_QUICKGELU)
    du = ops.act8_bwd(q, s, t["da"], ops.ACT_QUICKGELU)
    dw, db = ops.gemm_tn_act8(t["da"], q, s, colsum=True)
    g = ops.residual_norm_bwd(xn, t["y"], None, du, gate=t["gate"], gate_tanh=True, res_scale=0.9, post=t["post"], pre=t["pre"])
    de, dpos = ops.embed_tokens_bwd(t["ids"], g.dx.view(*t["ids"].shape, -1), t["w"].shape[0], scale=2.0, pos_grad=True)
    return [x, xn, h, a, q.view(torch.uint8), s, du, dw, db, de, dpos, *g]


def pass_inputs(seed, S=20):
    L, V, D = 77, 500, 256
    s = make_block(S * L, D, "group", True, True, False, F32, BF16, seed=seed, groups=S)
    return dict(ids=rints(0, V, (S, L), seed=seed), w=rnd(V, D, seed=seed + 1), pos=rnd(L, D, seed=seed + 2), y=s["y"], gate=s["gate"], post=s["post"], pre=s["pre"],
                da=rnd(S * L, D, seed=seed + 3, dtype=BF16))


@pytest.mark.parametrize("S", [5, 20, 130])                        # (a gradient without a sort, one by counting, one by digits with the zeros beside the sums)
def test_graph_replays_equal_eager_passes(S):
    static = pass_inputs(0, S)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            one_pass(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = one_pass(static)
    for seed in (0, 7, 3, 7):
        new = pass_inputs(seed, S)
        for k, v in new.items():
            for dst, src in zip(static[k], v) if isinstance(v, tuple) else ((static[k], v),):
                if isinstance(dst, torch.Tensor):
                    dst.copy_(src)
        eager = one_pass(new)
        for o in outs:                                              # nothing of the last replay may be taken for this one's
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(outs, eager)):
            assert torch.equal(a, b), (seed, i)


@pytest.mark.parametrize("S", [5, 20, 130])
def test_two_streams_at_once(S):
    a, b = pass_inputs(1, S), pass_inputs(2, S)
    want = [one_pass(a), one_pass(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for k, t in ((0, a), (1, b)):
            with torch.cuda.stream(streams[k]):
                got[k] = one_pass(t)
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(x, y) for x, y in zip(got[k], want[k]))


def test_a_block_trains_like_its_definition():
    """Embedding, pre-norm, MLP with 8-bit checkpoints, post-norm with a gate, all under autograd, against the same computed in 64 bits with the checkpoints' rounding put in
    where the kernels have it: what is left is the bf16 rounding of the matrix products' operands and results."""
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import token_stream as ts
    torch.manual_seed(0)
    S, L, V, D, H = 6, 24, 90, 128, 256
    emb = ts.TokenEmbedding(V, D, padding_idx=0).to(DEV)
    pos = nn.Parameter(0.3 * torch.randn(L + 4, D, device=DEV))
    pre, post = nn.LayerNorm(D).to(DEV), nn.LayerNorm(D).to(DEV)
    fc1, fc2 = nn.Linear(D, H).to(DEV), nn.Linear(H, D).to(DEV)
    gate = nn.Parameter(torch.tensor([0.4], device=DEV))
    ids = rints(0, V, (S, L), seed=1)
    cot = rnd(S * L, D, seed=2)
    x = emb(ids, pos, scale=D ** 0.5)
    flat = x.view(S * L, D)
    zero = torch.zeros_like(flat)
    x1, h = ts.residual_norm(flat, zero, pre=pre)
    y = ts.mlp_act8(h, fc1, fc2)
    x2, _ = ts.residual_norm(x1, y, gate=gate, post=post, gate_tanh=True, res_scale=0.8)
    (x2 * cot).sum().backward()
    leaves = [emb.weight, pos, pre.weight, pre.bias, post.weight, post.bias, fc1.weight, fc1.bias, fc2.weight, fc2.bias, gate]
    P = [t.detach().double().requires_grad_(True) for t in leaves]

    class Ckpt(torch.autograd.Function):                            # act(u), with the slope at the value that the checkpoint holds
        @staticmethod
        def forward(ctx, u):
            q, sc = act8_ref(u.float())
            ctx.save_for_backward((q * sc.repeat_interleave(128, 1)[:, :q.shape[1]]).to(u.device))
            return act_ref(u, ops.ACT_QUICKGELU)[0]

        @staticmethod
        def backward(ctx, da):
            return da * act_ref(ctx.saved_tensors[0], ops.ACT_QUICKGELU)[1]
    w = torch.where((ids == 0)[..., None], P[0][ids].detach(), P[0][ids])
    rx = (w * D ** 0.5 + P[1][:L]).view(S * L, D)
    rh = nn.functional.layer_norm(rx, (D,), P[2], P[3], pre.eps)
    ry = Ckpt.apply(rh @ P[6].t() + P[7]) @ P[8].t() + P[9]
    rx2 = rx * 0.8 + torch.tanh(P[10]) * nn.functional.layer_norm(ry, (D,), P[4], P[5], post.eps)
    (rx2 * cot.double()).sum().backward()
    assert float((x2.detach().double() - rx2.detach()).norm() / rx2.detach().norm()) <= 8 * 2.0 ** -8
    for name, t, p in zip("emb pos pre.g pre.b post.g post.b w1 b1 w2 b2 gate".split(), leaves, P):
        rel = float((t.grad.double() - p.grad).norm() / p.grad.norm())
        record("test_token_train_gpu", "block grad " + name, rel, 0.06)
        # at most 8 roundings to bf16 (2^-8 each) on the way, and the checkpoints' own (2^-4 of an element, independent: 2^-4 / sqrt 3 of a sum over
        # random signs, of the MLP's part alone, which the 64-bit side has only for fc1's output)
        assert rel <= 8 * 2.0 ** -8 + (2.0 ** -4 / 3 ** 0.5 if name in ("w1", "w2") else 0), (name, rel)
    assert not emb.weight.grad[0].any() and not pos.grad[L:].any()


def test_long_lists_pass_32_bits():
    """Element offsets above 2^31: 2^21 + 64 rows of 1024 channels in bf16 (4.3 GB)."""
    n, D, V = (1 << 21) + 64, 1024, 2000
    w = rnd(V, D, seed=1, dtype=BF16)
    ids = (torch.arange(n, device=DEV) * 7 % V).view(1, n)
    x = ops.embed_tokens(ids, w)
    for r in (0, 1 << 20, (1 << 21) - 1, n - 1):
        assert torch.equal(x[0, r], w[ids[0, r]])
    dy = torch.zeros(1, n, D, device=DEV, dtype=BF16)
    dy[0, -1], dy[0, 5] = 1, 2
    dw = ops.embed_tokens_bwd(ids, dy, V)
    want = torch.zeros(V, device=DEV).index_add_(0, ids[0, [n - 1, 5]], torch.tensor([1.0, 2.0], device=DEV))
    assert torch.equal(dw, want[:, None].expand(V, D))
    del dy, dw
    x2 = x.view(n, D)
    xn, h = ops.residual_norm(x2, x2, pre=(torch.ones(D, device=DEV), None, 1e-5), rms=True)
    small, hs = ops.residual_norm(x2[-64:].clone(), x2[-64:].clone(), pre=(torch.ones(D, device=DEV), None, 1e-5), rms=True)
    assert torch.equal(xn[-64:], small) and torch.equal(h[-64:], hs)
    del xn, h
    _, q, s = ops.act8(x2, want_out=False)
    _, qs, ss = ops.act8(x2[-64:].clone(), want_out=False)
    assert torch.equal(q[-64:].view(torch.uint8), qs.view(torch.uint8)) and torch.equal(s[-64:], ss)
    g = torch.zeros(n, 8, device=DEV, dtype=BF16)
    g[-64:] = rnd(64, 8, seed=3, dtype=BF16)
    got, ref = ops.gemm_tn_act8(g, q, s).double(), g[-64:].double().t() @ values(qs, ss)
    assert float((got - ref).abs().max()) <= 2 * 80 * U * float((g[-64:].double().abs().t() @ values(qs, ss).abs()).max())


def test_encode_text_looks_its_tokens_up_with_embed_tokens(monkeypatch):
    """CLIP.encode_text takes the operator, and its features are those of the stock lookup bit for bit (strided ids too)."""
    from helping_hand_for_egocentric_videos_amd import TINY4, synth
    from helping_hand_for_egocentric_videos_amd.model import LaviLa
    model = LaviLa.build_backbone(TINY4, synth.encoder_state(TINY4, seed=4))
    text = synth.make_batch(TINY4, 2, seed=9)["text"].to(DEV)
    calls = []
    real = ops.embed_tokens
    monkeypatch.setattr(ops, "embed_tokens", lambda *a, **k: calls.append(1) or real(*a, **k))
    cls, fmap = model.encode_text(text)
    assert calls == [1]
    wide = torch.zeros((text.shape[0], 2 * text.shape[1]), dtype=text.dtype, device=DEV)
    wide[:, ::2] = text
    assert torch.equal(model.encode_text(wide[:, ::2])[1], fmap)
    monkeypatch.setattr(ops, "embed_tokens", lambda ids, w, pos: torch.nn.functional.embedding(ids, w) + pos)
    cls2, fmap2 = model.encode_text(text)
    assert torch.equal(cls, cls2) and torch.equal(fmap, fmap2)
