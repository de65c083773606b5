"""GPU tests of the token-stream operators in the forms that tests/test_token_train_gpu.py does not take: every type triple of residual_norm, LayerNorms without beta and
root-mean-square norms with it, operands at odd addresses, the kernels that take four rows at a time, and the autograd forms' other branches.  Bounds are that file's."""
import itertools

import pytest
import torch
from torch import nn

import test_token_train_gpu as T
from test_token_train_gpu import BF16, DEV, F32, U, rints, rnd, stored, within
from helping_hand_for_egocentric_videos_amd import ops
from helping_hand_for_egocentric_videos_amd.model import token_stream as ts

pytestmark = pytest.mark.gpu
TRIPLES = list(itertools.product((F32, BF16), repeat=3))
NORMS = [(True, True), (False, True), (True, False), (False, False)]


def name(v):
    return {F32: "f32", BF16: "bf16"}.get(v) if isinstance(v, torch.dtype) else None


@pytest.fixture
def other_betas(monkeypatch):
    """make_block with a beta exactly where it has none: root-mean-square norms with beta, LayerNorms without."""
    real = T.make_block

    def make(rows, cols, gate, post, pre, rms, *a, **k):
        s = real(rows, cols, gate, post, pre, rms, *a, **k)
        for i, which in enumerate(("post", "pre")):
            if s[which] is not None:
                s[which] = (s[which][0], 0.2 * rnd(cols, seed=20 + i) if rms else None, s[which][2])
        return s
    monkeypatch.setattr(T, "make_block", make)


@pytest.fixture
def odd_addresses(monkeypatch):
    """Every input one element behind an aligned address."""
    def odd(*shape, **k):
        t = rnd(*shape, **k)
        raw = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        raw[1:] = t.reshape(-1)
        return raw[1:].view(t.shape)
    real = T.make_block

    def make(*a, **k):
        s = real(*a, **k)
        shift = lambda v: None if v is None else tuple(shift(x) for x in v) if isinstance(v, tuple) else v if isinstance(v, float) else odd_copy(v)  # noqa: E731
        return {k_: shift(v) for k_, v in s.items()}

    def odd_copy(t):
        raw = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        raw[1:] = t.reshape(-1)
        got = raw[1:].view(t.shape)
        assert got.data_ptr() % 16 != 0
        return got
    monkeypatch.setattr(T, "make_block", make)
    monkeypatch.setattr(T, "rnd", odd)


SHAPES = [(37, 255, "group"), (130, 768, "group"), (33, 1024, "channel"), (4100, 64, "scalar")]


@pytest.mark.parametrize("rows,cols,gate", SHAPES)
@pytest.mark.parametrize("post,pre", NORMS)
@pytest.mark.parametrize("xt,yt,ht", TRIPLES, ids=name)
def test_residual_norm_of_every_type(rows, cols, gate, post, pre, xt, yt, ht):
    rms = (xt, yt, ht).count(BF16) % 2 == 1
    T.test_residual_norm(rows, cols, gate, post, pre, rms, xt, yt, ht)
    T.test_residual_norm_bwd(rows, cols, gate, post, pre, rms, xt, yt, ht)


@pytest.mark.parametrize("rows,cols,gate", SHAPES + [(5, 3, "channel"), (416, 512, "none")])
@pytest.mark.parametrize("post,pre", NORMS[:3])
@pytest.mark.parametrize("rms", [False, True])
def test_residual_norm_without_beta_and_rms_norms_with_it(rows, cols, gate, post, pre, rms, other_betas):
    for xt, yt, ht in ((F32, BF16, BF16), (BF16, BF16, BF16)):
        T.test_residual_norm(rows, cols, gate, post, pre, rms, xt, yt, ht)
        T.test_residual_norm_bwd(rows, cols, gate, post, pre, rms, xt, yt, ht)


@pytest.mark.parametrize("rows,cols,gate", SHAPES + [(12, 3, "group"), (9, 1028, "channel")])
@pytest.mark.parametrize("post,pre", NORMS)
@pytest.mark.parametrize("xt,yt,ht", [(F32, BF16, BF16), (BF16, F32, F32), (BF16, BF16, BF16)], ids=name)
def test_residual_norm_at_odd_addresses(rows, cols, gate, post, pre, xt, yt, ht, odd_addresses):
    """Widths that wide accesses divide too: the address alone asks for the other form."""
    T.test_residual_norm(rows, cols, gate, post, pre, False, xt, yt, ht)
    T.test_residual_norm_bwd(rows, cols, gate, post, pre, False, xt, yt, ht)


# ---- four rows at a time ---------------------------------------------------------------------------------------------------------------
def term_sums(x_new, y, d, dh, gate, tanh, post, pre, rms, rows_of):
    """Sums over `rows_of(t)` of the magnitudes of what the parameters' gradients add up, in 64 bits: (dgate, dpost_gamma, dpost_beta, dpre_gamma, dpre_beta)."""
    def xhat(v, eps):
        c = v if rms else v - v.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    g = 1.0 if gate is None else (gate.double().tanh() if tanh else gate.double()).abs()
    d, y, out = d.double().abs(), y.double(), [None] * 5
    p = y.abs()
    if post is not None:
        xh = xhat(y, post[2]).abs()
        p = post[0].double().abs() * xh + (0 if post[1] is None else post[1].double().abs())
        out[1], out[2] = (g * d * xh).sum(0), (g * d).sum(0)
    out[0] = (d * p).sum(0)
    if pre is not None:
        out[3], out[4] = (dh.double().abs() * xhat(x_new.double(), pre[2]).abs()).sum(0), dh.double().abs().sum(0)
    return out


def large_block(cols, gate, post, pre, rms, xt, yt, ht, groups, beta):
    """Inputs of a call whose gradients are over 600 MB, with a number of rows in each group that four does not divide."""
    size = lambda t: 4 if t == F32 else 2  # noqa: E731
    each = (600 << 20) // (cols * (size(xt) + size(yt)) * groups) // 4 * 4 + 7
    rows = each * groups
    assert rows * cols * (size(xt) + size(yt)) > 600 << 20
    g = torch.Generator(device=DEV).manual_seed(5)
    big = lambda t, scale=1.0: (torch.randn(rows, cols, generator=g, device=DEV) * scale).to(t)  # noqa: E731
    s = dict(x=big(xt, 2.0), y=big(yt) + 0.25, dxn=big(xt), dh=big(ht) if pre else None)
    s["gate"] = {"none": None, "scalar": rnd(1, seed=3) + 0.5, "channel": rnd(cols, seed=3), "group": rnd(groups, cols, seed=3)}[gate]
    for i, which in enumerate(("post", "pre")):
        on = post if which == "post" else pre
        s[which] = (1 + 0.2 * rnd(cols, seed=10 + i), 0.2 * rnd(cols, seed=20 + i) if beta else None, 1e-5) if on else None
    return s, rows, each


FOUR = []                                                             # every kernel that takes four rows: a type triple with and without either norm (dh's type counts only with pre)
for k, ((post, pre), types) in enumerate(itertools.product(NORMS, TRIPLES)):
    if pre or types[2] == F32:
        gate = ("scalar", "none", "channel", "group")[(k + k // 4) % 4]
        FOUR.append((post, pre, *types, gate, k % 3 == 1, (200, 512, 1024, 772)[(k + k // 8) % 4], k % 2 == 0))


@pytest.mark.parametrize("post,pre,xt,yt,ht,gate,rms,cols,beta", FOUR, ids=name)
def test_residual_norm_bwd_of_four_rows_adds_every_row_once(post, pre, xt, yt, ht, gate, rms, cols, beta):
    """Gradients that are zero but in a few rows -- each group's first and last ones, the remainder that four does not divide among them -- so that the column sums have few terms and
    a row that is lost, added twice or added to another group's shows at its full size.  Rows without a gradient add exact zeros.  Against a call on those rows alone (a kernel of two
    rows at a time, which other tests hold to its definition): row by row equal, the sums to the error of adding that many terms in any order."""
    groups = 3 if gate == "group" else 1
    s, rows, each = large_block(cols, gate, post, pre, rms, xt, yt, ht, groups, beta)
    some = torch.cat([torch.arange(9), torch.tensor([each // 3, each // 2 + 1]), torch.arange(each - 9, each)])
    idx = torch.cat([some + k * each for k in range(groups)]).to(DEV)
    keep = torch.zeros(rows, 1, dtype=torch.bool, device=DEV)
    keep[idx] = True
    for n in ("dxn", "dh"):
        if s[n] is not None:
            s[n].masked_fill_(~keep, 0)
    kw = dict(gate=s["gate"], gate_tanh=k_tanh(gate), res_scale=0.75, post=s["post"], pre=s["pre"], rms=rms)
    got = ops.residual_norm_bwd(s["x"], s["y"], s["dxn"], s["dh"], **kw)
    few = {n: None if s[n] is None else s[n][idx].contiguous() for n in ("x", "y", "dxn", "dh")}
    part = ops.residual_norm_bwd(few["x"], few["y"], few["dxn"], few["dh"], **kw)
    assert torch.equal(got.dx[idx], part.dx) and torch.equal(got.dy[idx], part.dy)
    assert not got.dx.masked_fill(keep, 0).any() and not got.dy.masked_fill(keep, 0).any()
    n = len(some)
    d = part.dx.double() / 0.75 * (1 + 2.0 ** -7)                     # (bf16: the stored d is within a rounding of the one that was added)
    for g in range(groups):
        cut = slice(g * n, (g + 1) * n)
        gr = s["gate"][g] if gate == "group" else s["gate"]
        mags = term_sums(few["x"][cut], few["y"][cut], d[cut], None if few["dh"] is None else few["dh"][cut], gr, k_tanh(gate), s["post"], s["pre"], rms, None)
        total = mags if g == 0 else [None if a is None else a + b for a, b in zip(total, mags)]
        if gate == "group":
            # n rows and gamma S1 + beta S0, on both sides; tanh's slope (at most one) to 8 steps
            within(got.dgate[g], part.dgate[g].double(), 2 * (n + 24) * U * mags[0] + 1e-30, "four rows, dgate of a group")
    if gate in ("scalar", "channel"):
        mag = total[0].sum().view(1) if gate == "scalar" else total[0]
        within(got.dgate, part.dgate.double(), 2 * (len(idx) + (cols if gate == "scalar" else 0) + 24) * U * mag + 1e-30, "four rows, dgate")
    for i, field in enumerate(("dpost_gamma", "dpost_beta", "dpre_gamma", "dpre_beta")):
        a, b = getattr(got, field), getattr(part, field)
        assert (a is None) == (b is None)
        if a is not None:
            within(a, b.double(), 2 * (len(idx) + 24) * U * total[1 + i] + 1e-30, "four rows, " + field)


def k_tanh(gate):
    return gate in ("scalar", "group")


@pytest.mark.parametrize("post,pre,gate,rms,cols,types", [(True, True, "scalar", False, 1024, (F32, BF16, BF16)), (True, True, "group", True, 512, (BF16, BF16, BF16)),
                                                           (False, True, "channel", False, 256, (F32, F32, F32)), (True, False, "none", True, 1000, (BF16, F32, F32))])
def test_residual_norm_bwd_of_four_rows_sums_all_rows(post, pre, gate, rms, cols, types):
    """Dense gradients, against 64-bit sums of calls on about 2000 rows each.  A workgroup of the large call adds at most DEPTH rows, one after the other, and 16 terms or fewer
    follow each of the two times that partial rows are joined; the small calls add no more."""
    xt, yt, ht = types
    groups = 2 if gate == "group" else 1
    s, rows, each = large_block(cols, gate, post, pre, rms, xt, yt, ht, groups, True)
    kw = dict(gate_tanh=k_tanh(gate), res_scale=0.75, post=s["post"], pre=s["pre"], rms=rms)
    got = ops.residual_norm_bwd(s["x"], s["y"], s["dxn"], s["dh"], gate=s["gate"], **kw)
    blocks = 256 * (8 // -(-cols // 256))                             # resident workgroups
    DEPTH = -(-rows // blocks) + 8 + -(-blocks // 64) + 32            # a workgroup's rows, and the joining launch's sums over the workgroups by 64 lanes and 16 waves
    cut = lambda t, i, j: None if t is None else t[i:j].contiguous()  # noqa: E731
    sums, mags = None, None
    for k in range(groups):
        gr = s["gate"][k] if groups > 1 else s["gate"]
        for i in range(k * each, (k + 1) * each, 2000):
            j = min(i + 2000, (k + 1) * each)
            p = ops.residual_norm_bwd(cut(s["x"], i, j), cut(s["y"], i, j), cut(s["dxn"], i, j), cut(s["dh"], i, j), gate=gr, **kw)
            assert torch.equal(p.dx, got.dx[i:j]) and torch.equal(p.dy, got.dy[i:j])
            m = term_sums(s["x"][i:j], s["y"][i:j], p.dx.double() / 0.75 * (1 + 2.0 ** -7), cut(s["dh"], i, j), gr, k_tanh(gate), s["post"], s["pre"], rms, None)
            a = [None if t is None else t.double() for t in p[2:]]
            if gate == "scalar":
                m[0] = m[0].sum().view(1)
            if groups > 1:
                for v in (a, m):
                    rest = torch.zeros(groups, cols, dtype=torch.float64, device=DEV)
                    rest[k] = v[0]
                    v[0] = rest
            sums = a if sums is None else [None if t is None else t + v for t, v in zip(sums, a)]
            mags = m if mags is None else [None if t is None else t + v for t, v in zip(mags, m)]
    extra = cols if gate == "scalar" else 0
    for i, (field, t, v) in enumerate(zip(got._fields[2:], got[2:], sums)):
        assert (t is None) == (v is None)
        if t is not None:
            within(t, v, 2 * (DEPTH + 64 + (extra if i == 0 else 0)) * U * mags[i] + 1e-30, "all rows, " + field)


# ---- autograd --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rms,bias", [(False, True), (False, False), (True, False)])
@pytest.mark.parametrize("used", ["both", "x_new", "h"])
@pytest.mark.parametrize("xt,ht", [(F32, BF16), (BF16, F32)], ids=name)
def test_residual_norm_whose_outputs_go_unused(rms, bias, used, xt, ht):
    """The gradients under autograd are those of ops.residual_norm_bwd with zeros for an output that nothing uses -- both norms, LayerNorms without bias and RMSNorms."""
    rows, cols = 30, 96
    make = lambda i: nn.RMSNorm(cols, eps=1e-5) if rms else nn.LayerNorm(cols, bias=bias)  # noqa: E731
    post, pre = make(0).to(DEV), make(1).to(DEV)
    with torch.no_grad():
        for i, m in enumerate((post, pre)):
            m.weight.copy_(1 + 0.2 * rnd(cols, seed=10 + i))
            if getattr(m, "bias", None) is not None:
                m.bias.copy_(0.2 * rnd(cols, seed=20 + i))
    x, y = rnd(rows, cols, seed=1, dtype=xt).requires_grad_(True), rnd(rows, cols, seed=2, dtype=BF16).requires_grad_(True)
    gate = nn.Parameter(rnd(cols, seed=3))
    cx, ch = rnd(rows, cols, seed=4, dtype=xt), rnd(rows, cols, seed=5, dtype=ht)
    x_new, h = ts.residual_norm(x, y, gate=gate, post=post, pre=pre, gate_tanh=True, res_scale=0.8, rms=rms, out_dtype=ht)
    assert x_new.dtype == xt and h.dtype == ht
    terms = [(x_new * cx).float().sum()] * (used in ("both", "x_new")) + [(h * ch).float().sum()] * (used in ("both", "h"))
    leaves = [x, y, gate, post.weight, getattr(post, "bias", None), pre.weight, getattr(pre, "bias", None)]
    sum(terms).backward()
    norm = lambda m: (m.weight.detach(), None if getattr(m, "bias", None) is None else m.bias.detach(), m.eps)  # noqa: E731
    want = ops.residual_norm_bwd(x_new.detach(), y.detach(), cx if used != "h" else torch.zeros_like(cx), ch if used != "x_new" else torch.zeros_like(ch), gate=gate.detach(),
                                 gate_tanh=True, res_scale=0.8, post=norm(post), pre=norm(pre), rms=rms)
    for leaf, ref in zip(leaves, want):
        assert (leaf is None) == (ref is None)
        if leaf is not None:
            assert leaf.grad.dtype == leaf.dtype and torch.equal(leaf.grad, ref)


@pytest.mark.parametrize("ot", [None, F32], ids=name)
def test_a_bf16_table_under_autograd(ot):
    V, D, S, L = 300, 96, 11, 70
    emb = ts.TokenEmbedding(V, D, padding_idx=3).to(DEV).to(BF16)
    pos, ids = nn.Parameter(rnd(L, D, seed=1)), rints(0, V, (S, L), seed=2)
    out = emb(ids, pos, scale=2.5, out_dtype=ot)
    assert out.dtype == (BF16 if ot is None else ot)
    ref = 2.5 * emb.weight.detach().double()[ids] + pos.detach().double()
    within(out.detach(), ref, 2 * U * (2.5 * emb.weight.detach().double()[ids]).abs() + U * ref.abs() + stored(ref, out.dtype), "bf16 table")
    cot = rnd(S, L, D, seed=3, dtype=out.dtype)
    out.backward(cot)
    dw, bound = T.embed_grad_ref(ids, cot, V, 2.5, 3)
    assert emb.weight.grad.dtype == BF16 and pos.grad.dtype == F32 and not emb.weight.grad[3].any()
    within(emb.weight.grad, dw, bound + 2.0 ** -8 * (dw.abs() + bound), "bf16 table's gradient")
    within(pos.grad, cot.double().sum(0), (S + 2) * U * cot.double().abs().sum(0), "bf16 table, pos grad")


@pytest.mark.parametrize("rows", [0, 1, 77, 520])
@pytest.mark.parametrize("act", [ops.ACT_QUICKGELU, ops.ACT_RELU])
@pytest.mark.parametrize("biases", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("xt", [F32, BF16], ids=name)
def test_mlp_act8_of_every_form(rows, act, biases, xt):
    """Against 64-bit products of operands that are rounded where the kernels round them (bf16 operands and results, e4m3 checkpoints): what is left is roundings that fall
    the other way because a product was summed in fp32, a bf16 step (2^-7 of an element) each, which cannot move all elements: below one bf16 step of the norm."""
    D, H, O = 128, 384, 256
    torch.manual_seed(0)
    fc1, fc2 = nn.Linear(D, H, bias=biases[0]).to(DEV), nn.Linear(H, O, bias=biases[1]).to(DEV)
    x = rnd(rows, D, seed=1, dtype=xt).requires_grad_(True)
    y = ts.mlp_act8(x, fc1, fc2, act)
    assert y.shape == (rows, O) and y.dtype == F32
    dy = rnd(rows, O, seed=2)
    y.backward(dy)
    b = lambda t: t.detach().to(BF16).double()  # noqa: E731
    bias = lambda m: 0 if m.bias is None else m.bias.detach().double()  # noqa: E731

    def held(t):
        q, s = T.act8_ref(t.float())
        return (q * s.repeat_interleave(128, 1)[:, :q.shape[1]]).to(DEV)
    xb = b(x)
    u = b(xb @ b(fc1.weight).t() + bias(fc1))
    a = b(T.act_ref(u, act)[0])
    ry = a @ b(fc2.weight).t() + bias(fc2)
    v = held(u)
    av, slope = T.act_ref(v, act)
    du = b(b(b(dy) @ b(fc2.weight)) * slope)
    refs = [ry, b(du @ b(fc1.weight)) if xt == BF16 else du @ b(fc1.weight), du.t() @ held(xb), du.sum(0), b(dy).t() @ b(av), b(dy).sum(0)]
    for what, t, ref in zip("y dx dw1 db1 dw2 db2".split(), [y.detach(), x.grad, fc1.weight.grad, fc1.bias.grad if biases[0] else None, fc2.weight.grad,
                                                            fc2.bias.grad if biases[1] else None], refs):
        if t is None:
            continue
        assert t.shape == ref.shape
        err, size = float((t.double() - ref).norm()), float(ref.norm())
        T.record("test_token_train_forms_gpu", "mlp " + what, err / (size + 1e-300), 2.0 ** -7)
        assert err <= 2.0 ** -7 * size, (what, err, size)


# ---- graphs that run at once -----------------------------------------------------------------------------------------------------------
def mlp_pass(rows, seed):
    """An MLP's forward and backward pass over fresh inputs of its own -> (what runs it, the tensors that it reads)."""
    D, H = 512, 1024
    torch.manual_seed(seed)
    fc1, fc2 = nn.Linear(D, H).to(DEV), nn.Linear(H, D).to(DEV)
    x, dy = rnd(rows, D, seed=seed, dtype=BF16).requires_grad_(True), rnd(rows, D, seed=seed + 1)

    def run():
        y = ts.mlp_act8(x, fc1, fc2)
        return [y.detach(), *torch.autograd.grad(y, [x, fc1.weight, fc1.bias, fc2.weight, fc2.bias], dy)]
    return run, (x, dy)


def captured(run):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run()
    return graph, outs


@pytest.mark.parametrize("rows", [640, 65536])
def test_captured_mlps_that_run_at_once(rows):
    """Two graphs, captured one after the other on torch's one capture stream and replayed side by side on two others (65 536 rows: products of 1024 tiles, more than there are
    workgroups), with eager passes between: each replay gives the eager results' bits."""
    runs = [mlp_pass(rows, seed) for seed in (1, 5)]
    graphs = [captured(run) for run, _ in runs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for k, (_, (x, dy)) in enumerate(runs):
            with torch.no_grad():
                x.copy_(rnd(rows, x.shape[1], seed=10 * turn + k, dtype=BF16))
                dy.copy_(rnd(rows, dy.shape[1], seed=10 * turn + k + 5))
            for o in graphs[k][1]:
                o.zero_()
        torch.cuda.synchronize()
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (run, _), (_, outs) in zip(runs, graphs):
            for i, (got, want) in enumerate(zip(outs, run())):
                assert torch.equal(got, want), (turn, i)
