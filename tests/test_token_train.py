"""CPU-side checks of the operators that train a token stream: what the C ABI and the Python side refuse before anything is launched."""
import ctypes

import pytest
import torch

from helping_hand_for_egocentric_videos_amd import _lib, ops


def test_embed_tokens_refusals():
    L = _lib.lib()
    f = lambda ids=16, idb=8, w=16, wd=0, o=16, od=0, s=2, n=3, v=5, d=8: L.hh_embed_tokens_fwd(ids, idb, w, wd, None, o, od, s, n, v, d, 1.0, None)  # noqa: E731
    assert f(s=0) == 0                                               # nothing to do: no launch, no pointer read
    assert f(d=0) == -1 and f(v=0) == -1 and f(n=0) == -1 and f(s=-1) == -1 and f(d=(1 << 20) + 1) == -1 and f(v=1 << 31) == -1 and f(s=1 << 20, n=1 << 10) == -1
    assert b"hh_embed_tokens_fwd" in L.hh_last_error_string()
    assert f(idb=2) == -2 and f(wd=2) == -2 and f(od=7) == -2
    assert f(ids=None) == -5 and f(w=None) == -5 and f(o=None) == -5
    b = lambda ids=16, idb=8, dy=16, dd=0, dw=16, s=2, n=3, v=5, d=8, ws=16: L.hh_embed_tokens_bwd(ids, idb, dy, dd, dw, 1, None, s, n, v, d, 1.0, -1, ws, None)  # noqa: E731
    assert b(d=0) == -1 and b(idb=1) == -2 and b(dd=3) == -2 and b(dw=None) == -5 and b(ids=None) == -5 and b(dy=None) == -5 and b(s=2000, ws=None) == -5 and b(s=2000, ws=8) == -5
    assert L.hh_workspace_bytes_embed_tokens_bwd(2, 0, 5, 8) == -1 and L.hh_workspace_bytes_embed_tokens_bwd(1 << 30, 1, 5, 8) == -1
    assert L.hh_workspace_bytes_embed_tokens_bwd(2, 3, 5, 8) == 0         # few tokens: one launch
    assert L.hh_workspace_bytes_embed_tokens_bwd(160, 77, 49408, 768) >= 4 * 4 * 160 * 77


def test_residual_norm_refusals():
    L = _lib.lib()

    def desc(**kw):
        d = _lib.ResidualNorm()
        d.rows, d.groups, d.cols, d.res_scale = 6, 1, 64, 1.0
        d.x = d.y = d.x_new = d.dx = d.dy = d.workspace = 16
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)
    for fn, name in ((L.hh_residual_norm_fwd, b"hh_residual_norm_fwd"), (L.hh_residual_norm_bwd, b"hh_residual_norm_bwd")):
        assert fn(None, None) == -1
        assert fn(desc(cols=0), None) == -1 and fn(desc(cols=4097), None) == -1 and fn(desc(rows=-1), None) == -1
        assert name in L.hh_last_error_string()
        assert fn(desc(gate_kind=4), None) == -3 and fn(desc(groups=0), None) == -1 and fn(desc(groups=4, gate_kind=3, gate=16), None) == -1
        assert fn(desc(groups=2), None) == -1                        # groups without a gate for each
        assert fn(desc(groups=65001, rows=65001, gate_kind=3, gate=16), None) == -1
        assert fn(desc(x_dtype=2), None) == -2 and fn(desc(y_dtype=-1), None) == -2 and fn(desc(h_dtype=5), None) == -2
        assert fn(desc(y=None), None) == -5 and fn(desc(x_new=None), None) == -5
        assert fn(desc(gate=16), None) == -5 and fn(desc(gate_kind=1), None) == -5
        assert fn(desc(post_beta=16), None) == -5 and fn(desc(pre_beta=16), None) == -5
    assert L.hh_residual_norm_fwd(desc(x=None), None) == -5
    assert L.hh_residual_norm_fwd(desc(h=16), None) == -5 and L.hh_residual_norm_fwd(desc(pre_gamma=16), None) == -5
    assert L.hh_residual_norm_fwd(desc(rows=0), None) == 0
    assert L.hh_residual_norm_bwd(desc(dx=None), None) == -5 and L.hh_residual_norm_bwd(desc(dy=None), None) == -5
    assert L.hh_residual_norm_bwd(desc(dh=16), None) == -5 and L.hh_residual_norm_bwd(desc(workspace=None), None) == -5
    assert L.hh_residual_norm_bwd(desc(gate=16, gate_kind=2), None) == -5       # a gate without its gradient's place
    assert L.hh_residual_norm_bwd(desc(dpost_gamma=16), None) == -5 and L.hh_residual_norm_bwd(desc(dpre_beta=16), None) == -5
    assert L.hh_workspace_bytes_residual_norm_bwd(6, 64, 4) == -1 and L.hh_workspace_bytes_residual_norm_bwd(6, 4097, 1) == -1
    assert L.hh_workspace_bytes_residual_norm_bwd(0, 64, 1) == 0
    assert ctypes.sizeof(_lib.ResidualNorm) == L.hh_abi_sizeof(b"hh_residual_norm")


def test_act8_refusals():
    L = _lib.lib()
    f = lambda u=16, dt=0, q=16, s=16, r=2, c=8, act=0: L.hh_act8_fwd(u, dt, None, q, s, r, c, act, None)  # noqa: E731
    assert f(r=0) == 0 and f(r=-1) == -1 and f(c=0) == -1 and f(dt=2) == -2 and f(act=3) == -3 and f(u=None) == -5 and f(q=None) == -5 and f(s=None) == -5
    assert f(r=1 << 45) == -1
    b = lambda q=16, s=16, da=16, du=16, dt=0, r=2, c=8, act=0: L.hh_act8_bwd(q, s, da, du, None, dt, r, c, act, None)  # noqa: E731
    assert b(r=0) == 0 and b(c=-3) == -1 and b(dt=9) == -2 and b(act=-1) == -3 and b(q=None) == -5 and b(s=None) == -5 and b(da=None) == -5 and b(du=None) == -5
    g = lambda dy=16, ld=8, q=16, ldq=16, s=16, dw=16, M=8, N=16, K=64, ws=16: L.hh_gemm_tn_act8(dy, ld, q, ldq, s, dw, None, M, N, K, ws, None)  # noqa: E731
    assert g(M=0) == -1 and g(N=0) == -1 and g(K=-1) == -1 and g(ld=7) == -1 and g(ldq=15) == -1 and g(ld=(1 << 24) + 8) == -1 and g(K=(1 << 30) + 1) == -1
    assert g(dy=None) == -5 and g(q=None) == -5 and g(s=None) == -5 and g(dw=None) == -5 and g(dw=8) == -5 and g(K=4096, ws=None) == -5
    assert L.hh_workspace_bytes_gemm_tn_act8(0, 16, 64) == -1 and L.hh_workspace_bytes_gemm_tn_act8(8, 16, 64) == 0      # (one slice)
    assert L.hh_workspace_bytes_gemm_tn_act8(128, 128, 1 << 16) >= 2 * 128 * 128 * 4


def test_cpu_tensors_and_wrong_types_are_refused():
    f = torch.zeros(4, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embed_tokens(torch.zeros(2, 2, dtype=torch.int64), f)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.embed_tokens_bwd(torch.zeros(2, 2, dtype=torch.int64), torch.zeros(2, 2, 8), 4)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.residual_norm(f, f)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.residual_norm_bwd(f, f, f)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.act8(f)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.act8_bwd(f.to(torch.float8_e4m3fn), f[:, :1], f, ops.ACT_RELU)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.gemm_tn_act8(f.bfloat16(), f.to(torch.float8_e4m3fn), f[:, :1].contiguous())
    with pytest.raises(ValueError, match="unit inner stride"):
        ops.gemm_tn_act8(f.bfloat16().t(), f.to(torch.float8_e4m3fn), f)
    with pytest.raises(ValueError, match="rows that do not overlap"):
        ops.gemm_tn_act8(torch.zeros(1, 8, dtype=torch.bfloat16).expand(4, 8), f.to(torch.float8_e4m3fn), f)


def test_pinned_matrix_products_keep_their_distances(tmp_path):
    """gemm_tn8.hip's matrix instructions in inline asm are opaque to hipcc: in what it makes of them, no vector instruction writes a source of one right before it, nothing
    but them touches an accumulator inside the loop, and behind the last one every accumulator is read only after 16 wait states of its own (s_nop 15)."""
    import os
    import re
    import subprocess
    from helping_hand_for_egocentric_videos_amd import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path / "gemm_tn8.s")
    subprocess.run([build.HIPCC] + build.FLAGS + ["--cuda-device-only", "-S", os.path.join(build.CSRC, "gemm_tn8.hip"), "-o", out], check=True, capture_output=True)
    text = open(out).read()

    def regs(token):
        m = re.match(r"([va])\[(\d+):(\d+)\]$", token)
        if m:
            return {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)}
        return {token} if re.match(r"[va]\d+$", token) else set()
    found = 0
    for body in re.findall(r"^_Z15gemm_tn8_kernelILi8E.*?\.end_amdhsa_kernel", text, re.S | re.M):
        insts = []
        for line in body.split("\n"):
            line = line.split(";")[0].strip()
            if re.match(r"[a-z]+_", line):
                op, _, rest = line.partition(" ")
                insts.append((op, [t.split()[0] for t in re.split(r",\s*", rest) if t]))
        at = [i for i, (op, _) in enumerate(insts) if op.startswith("v_mfma")]
        assert len(at) == 4 * 64
        found += 1
        for i in at:
            sources = set().union(*[regs(t) for t in insts[i][1][1:3]])
            for op, args in insts[max(0, i - 6):i]:
                assert not (op.startswith("v_") and not op.startswith("v_mfma") and args and regs(args[0]) & sources), (op, args, insts[i])
        for op, args in insts[at[0]:at[-1] + 1]:
            assert op.startswith("v_mfma") or not any(t.startswith("a") and regs(t) for t in args), (op, args)
        nops = [i for i, (op, args) in enumerate(insts) if op == "s_nop" and args == ["15"]]
        assert len(nops) >= 64 and nops[0] > at[-1]
        for op, args in insts[at[-1] + 1:nops[0]]:              # (the zeros of a slice without tokens are written here)
            assert not any(regs(t) and t.startswith("a") for t in args[1:]), (op, args)
    assert found == 2


def test_norm_modules_that_the_residual_does_not_take_are_refused():
    """A norm without weights would be left out, one of the other kind computed as if it were not."""
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import token_stream as ts
    x = torch.zeros(2, 8)
    for norm, rms in ((nn.LayerNorm(8, elementwise_affine=False), False), (nn.RMSNorm(8, elementwise_affine=False), True)):
        with pytest.raises(ValueError, match="no weight"):
            ts.residual_norm(x, x, post=norm, rms=rms)
    for norm, rms in ((nn.RMSNorm(8), False), (nn.LayerNorm(8), True)):
        for where in ("post", "pre"):
            with pytest.raises(TypeError, match=where):
                ts.residual_norm(x, x, rms=rms, **{where: norm})


def test_residual_norm_without_rows_still_needs_the_parameters_it_reads():
    """The backward pass of no rows writes the parameters' gradients, a tanh gate's from the gate's values: a gate that is not there is refused as it is with rows."""
    L = _lib.lib()
    for gate_kind, dgate in ((1, 16), (2, 16), (3, 16)):
        for tanh in (0, 1):
            d = _lib.ResidualNorm()
            d.rows, d.groups, d.cols, d.res_scale, d.gate_kind, d.gate_tanh, d.dgate = 0, 1, 64, 1.0, gate_kind, tanh, dgate
            assert L.hh_residual_norm_bwd(ctypes.byref(d), None) == -5 and L.hh_residual_norm_fwd(ctypes.byref(d), None) == -5
    for beta in ("post_beta", "pre_beta"):
        d = _lib.ResidualNorm()
        d.rows, d.groups, d.cols, d.res_scale = 0, 1, 64, 1.0
        setattr(d, beta, 16)
        assert L.hh_residual_norm_bwd(ctypes.byref(d), None) == -5 and L.hh_residual_norm_fwd(ctypes.byref(d), None) == -5


def text_tower(monkeypatch):
    """A CLIP on the CPU whose encode_text ends behind the embedding, and a list of the lookups that ops.embed_tokens made."""
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import LaviLa
    torch.manual_seed(0)
    clip = LaviLa.CLIP(embed_dim=8, vision_width=8, vision_model=nn.Identity(), context_length=9, vocab_size=40, transformer_width=16, transformer_heads=2, transformer_layers=1)
    clip.requires_grad_(False)
    calls = []
    monkeypatch.setattr(LaviLa, "_require_gpu", lambda x, who: None)
    monkeypatch.setattr(clip.transformer, "forward_frozen", lambda x, final_ln, owns_x: x)
    monkeypatch.setattr(ops, "embed_tokens", lambda ids, w, pos: calls.append(1) or torch.nn.functional.embedding(ids, w) + pos)
    return clip, calls


def test_encode_text_calls_a_token_embedding_that_does_more_than_a_lookup(monkeypatch):
    from torch import nn
    clip, calls = text_tower(monkeypatch)
    text = torch.randint(0, 40, (3, 7))
    run = lambda: clip.encode_text(text, apply_project=False, want_cls=False)[1]  # noqa: E731
    plain = clip.token_embedding(text) + clip.positional_embedding[:7]
    assert torch.equal(run(), plain) and calls == [1]

    stock = clip.token_embedding
    for register, hook in ((stock.register_forward_hook, lambda m, i, o: o * 2), (stock.register_forward_pre_hook, lambda m, i: (i[0] * 0,))):
        handle = register(hook)
        want = stock(text) + clip.positional_embedding[:7]
        assert not torch.equal(want, plain) and torch.equal(run(), want) and calls == [1]
        handle.remove()
    handle = nn.modules.module.register_module_forward_hook(lambda m, i, o: o + 1 if m is stock else None)
    assert torch.equal(run(), stock(text) + clip.positional_embedding[:7]) and calls == [1]
    handle.remove()

    class Adapter(nn.Embedding):
        def forward(self, ids):
            return super().forward(ids) * 3
    clip.token_embedding = Adapter(40, 16, _weight=stock.weight.data)
    assert torch.equal(run(), 3 * stock(text) + clip.positional_embedding[:7]) and calls == [1]

    class Wrapper(nn.Module):                                        # no table of its own name
        def __init__(self):
            super().__init__()
            self.inner = stock

        def forward(self, ids):
            return self.inner(ids) - 1
    clip.token_embedding = Wrapper()
    assert torch.equal(run(), stock(text) - 1 + clip.positional_embedding[:7]) and calls == [1]

    bounded = nn.Embedding(40, 16, max_norm=0.01, _weight=stock.weight.data.clone())
    clip.token_embedding = bounded
    assert float((run() - clip.positional_embedding[:7]).norm(dim=-1).max()) <= 0.0101 and calls == [1]

    patched = nn.Embedding(40, 16, _weight=stock.weight.data)
    patched.forward = lambda ids: stock(ids) * 5
    clip.token_embedding = patched
    assert torch.equal(run(), stock(text) * 5 + clip.positional_embedding[:7]) and calls == [1]


def test_encode_text_takes_tables_that_the_operator_does_not(monkeypatch):
    """Transposed storage, another type, a tensor subclass, one row of positions for all: as the stock operations have it."""
    from torch import nn
    clip, calls = text_tower(monkeypatch)
    text = torch.randint(0, 40, (3, 7))
    run = lambda: clip.encode_text(text, apply_project=False, want_cls=False)[1]  # noqa: E731
    w, pos = clip.token_embedding.weight.data, clip.positional_embedding.data
    want = clip.token_embedding(text) + pos[:7]
    clip.token_embedding.weight = nn.Parameter(w.t().contiguous().t(), requires_grad=False)
    assert torch.equal(run(), want) and not calls

    class Sub(torch.Tensor):
        pass
    clip.token_embedding.weight = nn.Parameter(w.as_subclass(Sub), requires_grad=False)
    assert torch.equal(run().as_subclass(torch.Tensor), want) and not calls
    clip.token_embedding.weight = nn.Parameter(w.double(), requires_grad=False)
    assert run().dtype == torch.float64 and not calls
    clip.token_embedding.weight = nn.Parameter(w, requires_grad=False)
    clip.positional_embedding = nn.Parameter(pos.t().contiguous().t(), requires_grad=False)
    assert torch.equal(run(), want) and not calls
    clip.positional_embedding = nn.Parameter(pos[:1].clone(), requires_grad=False)
    assert torch.equal(run(), clip.token_embedding(text) + pos[:1]) and not calls
    clip.positional_embedding = nn.Parameter(pos, requires_grad=False)
    assert torch.equal(run(), want) and calls == [1]


def test_non_temporal_embedding_kernels_store_past_the_caches(tmp_path):
    """embed_tokens.hip's forward kernels for large outputs, of every type: in what hipcc makes of them each wide store is non-temporal, and none in the kernels for small outputs."""
    import os
    import re
    import subprocess
    from helping_hand_for_egocentric_videos_amd import build
    if not os.path.exists(build.HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path / "embed_tokens.s")
    subprocess.run([build.HIPCC] + build.FLAGS + ["--cuda-device-only", "-S", os.path.join(build.CSRC, "embed_tokens.hip"), "-o", out], check=True, capture_output=True)
    found = set()
    for name, body in re.findall(r"^(_Z16embed_fwd_kernel\w+):(.*?)\.end_amdhsa_kernel", open(out).read(), re.S | re.M):
        nt = re.search(r"Lb([01])E", name)[1] == "1"
        wide = re.findall(r"global_store_dwordx[24][^\n]*", body)
        assert wide and all((" nt" in line) == nt for line in wide), (name, wide)
        found.add(name)
    assert len(found) == 8


def test_positions_alone_refusals(monkeypatch):
    """Without a place for the table's gradient there has to be one for the positions'; dy and the workspace are needed as ever, ids are not read."""
    L = _lib.lib()
    b = lambda ids=16, dy=16, dw=None, dpos=16, s=2, ws=16: L.hh_embed_tokens_bwd(ids, 8, dy, 0, dw, 0, dpos, s, 3, 5, 8, 1.0, -1, ws, None)  # noqa: E731
    assert b(dpos=None) == -5 and b(dy=None) == -5 and b(s=2000, ws=None) == -5 and b(s=2000, ws=8) == -5
    assert b(dw=16, ids=None) == -5
    monkeypatch.setattr(ops, "_here", lambda *t: 0)
    ids, dy = torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3, 8)
    for kw in ({}, {"pos_grad": True, "out": torch.zeros(4, 8)}):
        with pytest.raises(ValueError, match="weight_grad=False"):
            ops.embed_tokens_bwd(ids, dy, 4, weight_grad=False, **kw)


def test_calls_that_a_launch_has_no_room_for_are_refused_as_shapes():
    """A launch counts its threads in 32 bits.  One row under the limit is not tried here: it would be launched."""
    L = _lib.lib()
    f = lambda s, d, wd=0, od=0: L.hh_embed_tokens_fwd(16, 8, 16, wd, None, 16, od, s, 1, 5, d, 1.0, None)  # noqa: E731
    assert f(1 << 26, 768) == -1 and b"too many tokens" in L.hh_last_error_string()
    assert f(1 << 26, 129, 0, 1) == -1 and f(1 << 26, 129, 1, 0) == -1 and f(1 << 26, 257, 1, 1) == -1 and f(1 << 27, 129, 1, 1) == -1 and f(1 << 29, 30) == -1

    def norm(rows, cols):
        d = _lib.ResidualNorm()
        d.rows, d.groups, d.cols, d.res_scale = rows, 1, cols, 1.0
        d.x = d.y = d.x_new = 16
        return L.hh_residual_norm_fwd(ctypes.byref(d), None)
    assert norm(1 << 28, 8) == -1 and b"too many rows" in L.hh_last_error_string()
    assert norm(1 << 24, 4096) == -1 and norm((1 << 31) - 1, 256) == -1 and norm(1 << 40, 1) == -1 and norm((1 << 63) - 1, 1) == -1
    for fn, args in ((L.hh_act8_fwd, lambda r, c: (16, 1, None, 16, 16, r, c, 0, None)), (L.hh_act8_bwd, lambda r, c: (16, 16, 16, 16, None, 1, r, c, 0, None))):
        for rows, cols in ((1 << 28, 128), (1 << 28, 1), (1 << 24, 2047), (1 << 23, 2049), ((1 << 63) - 1, 4096)):
            assert fn(*args(rows, cols)) == -1, (rows, cols)
            assert b"too many rows" in L.hh_last_error_string()


def test_sizes_over_32_bits_are_refused_before_they_are_cut_off(monkeypatch):
    """The library takes widths and lengths as 32-bit integers, of which ctypes keeps the lowest bits: 2^32 + 64 channels would be worked on as 64."""
    monkeypatch.setattr(ops, "_here", lambda *t: 0)
    monkeypatch.setattr(_lib, "lib", lambda: pytest.fail("reached the library"))
    wide = lambda dtype, *shape: torch.zeros((), dtype=dtype).expand(shape)  # noqa: E731
    n = (1 << 32) + 64
    ids, f, b, q, i64 = torch.zeros(1, 1, dtype=torch.int64), torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.int64
    calls = [lambda: ops.embed_tokens(wide(i64, 1, n), wide(b, 4, 1)), lambda: ops.embed_tokens(ids, wide(b, 4, n)),
             lambda: ops.embed_tokens_bwd(wide(i64, 1, n), wide(b, 1, n, 1), 4), lambda: ops.embed_tokens_bwd(ids, wide(b, 1, 1, n), 4),
             lambda: ops.residual_norm(wide(b, 1, n), wide(b, 1, n)), lambda: ops.residual_norm_bwd(wide(b, 1, n), wide(b, 1, n), wide(b, 1, n)),
             lambda: ops.act8(wide(b, 1, n)), lambda: ops.act8_bwd(wide(q, 1, n), wide(f, 1, n // 128 + 1), wide(b, 1, n), 0)]
    for call in calls:
        with pytest.raises(ValueError, match="over 2"):
            call()
    # (an expanded row has no unit inner stride: a storage that nothing touches)
    dy = torch.empty(1, n, dtype=b)
    with pytest.raises(ValueError, match="over 2"):
        ops.gemm_tn_act8(dy, torch.zeros(1, 8).to(q), torch.ones(1, 1))


def test_modules_that_are_not_what_the_autograd_forms_compute_are_refused():
    """Their weights have the right sizes and names: they were taken for a LayerNorm, or for a plain Linear."""
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import token_stream as ts

    class OwnNorm(nn.Module):                                        # a root-mean-square norm of the user's
        def __init__(self):
            super().__init__()
            self.weight, self.eps = nn.Parameter(torch.ones(8)), 1e-6
    x = torch.zeros(2, 8)
    for norm in (nn.BatchNorm1d(8), nn.GroupNorm(2, 8), OwnNorm()):
        for rms in (False, True):
            with pytest.raises(TypeError, match="post"):
                ts.residual_norm(x, x, post=norm, rms=rms)

    class LowRank(nn.Linear):
        def forward(self, x):
            return super().forward(x) + 1

    class Wrapper(nn.Module):
        def __init__(self):
            super().__init__()
            self.base = nn.Linear(128, 128)
            self.weight, self.bias = self.base.weight, self.base.bias
    plain = nn.Linear(128, 128)
    for other in (LowRank(128, 128), Wrapper()):
        for fcs in ((plain, other), (other, plain)):
            with pytest.raises(TypeError, match="must be nn.Linear"):
                ts.mlp_act8(torch.zeros(2, 128), *fcs)


def test_casts_and_the_mlp_refuse_other_types(monkeypatch):
    """The casts read four bytes (two) for each value whatever the tensor's type was: a half-precision input or weight was read past its end."""
    from torch import nn
    from helping_hand_for_egocentric_videos_amd.model import token_stream as ts
    monkeypatch.setattr(ops, "_chk", lambda *t: None)
    monkeypatch.setattr(ops, "_here", lambda *t: 0)
    monkeypatch.setattr(_lib, "lib", lambda: pytest.fail("reached the library"))
    for dtype in (torch.float16, torch.float64, torch.int32, torch.uint8):
        for cast in (ops.to_bf16, ops.to_f32):
            with pytest.raises(TypeError, match="unsupported dtype"):
                cast(torch.zeros(4, 8, dtype=dtype))
    for dtype in (torch.float16, torch.float64):
        with pytest.raises(TypeError, match="unsupported dtype"):
            ts.mlp_act8(torch.zeros(4, 128, dtype=dtype), nn.Linear(128, 128), nn.Linear(128, 128))
    for x in (torch.zeros(4, 8), torch.zeros(4, 8, dtype=torch.bfloat16)):
        assert (ops.to_bf16 if x.dtype == torch.bfloat16 else ops.to_f32)(x) is x
