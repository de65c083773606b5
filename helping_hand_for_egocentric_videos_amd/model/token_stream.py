"""Autograd of the operators that a trainable token tower needs around its matrix products and attention cores (ops.embed_tokens, ops.residual_norm,
ops.act8): the embedding with the gradient of its table by sorted tokens, the end of a residual block, and an MLP that keeps its activations in 8
bits.  The reference trains none of its towers (run/train.py:89 freezes the backbone), and this package's towers stay frozen: their attention cores have no backward
pass here.  These are pieces for a user's own trained tower or block, next to the decoder's attention and products: `CLIP.encode_text`'s lookup (LaviLa.py:660-663), the
residual of `SpaceTimeBlock` with the tanh gate that the reference has there (LaviLa.py:305-390), `Mlp` (LaviLa.py:175-190).

Once differentiable.  Under graph capture, as for any autograd function: no eager graph of the same parameters may be alive when a backward pass is captured (drop
earlier outputs and losses first), and gradients should be None or already allocated outside the capture."""
import torch
from torch import nn
from torch.autograd.function import once_differentiable

from .. import ops


class _EmbedTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, pos, scale, skip_id, out_dtype):
        ids = ids.contiguous()
        out = ops.embed_tokens(ids, weight.detach().contiguous(), scale=scale, pos=None if pos is None else pos.detach().contiguous(), out_dtype=out_dtype)
        ctx.save_for_backward(ids)
        ctx.shape, ctx.dtype, ctx.scale, ctx.skip_id = weight.shape, weight.dtype, scale, skip_id
        ctx.pos_rows = None if pos is None else pos.shape[0]
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        want_pos = ctx.pos_rows is not None and ctx.needs_input_grad[2]
        if not (ctx.needs_input_grad[1] or want_pos):
            return (None,) * 6
        got = ops.embed_tokens_bwd(ids, dy.contiguous(), ctx.shape[0], scale=ctx.scale, skip_id=ctx.skip_id, pos_grad=want_pos, weight_grad=ctx.needs_input_grad[1])
        dw, dpos = got if want_pos else (got, None)
        if want_pos and dpos.shape[0] < ctx.pos_rows:
            dpos = torch.cat([dpos, dpos.new_zeros((ctx.pos_rows - dpos.shape[0], dpos.shape[1]))])
        return None, dw.to(ctx.dtype) if ctx.needs_input_grad[1] else None, dpos, None, None, None


def embed_tokens(ids, weight, pos=None, scale=1.0, skip_id=None, out_dtype=None):
    """scale * weight[ids] + pos with gradients of weight [V, D] and pos fp32 [P, D] (ops.embed_tokens)."""
    return _EmbedTokens.apply(ids, weight, pos, float(scale), skip_id, out_dtype)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, gate, post_gamma, post_beta, pre_gamma, pre_beta, opts):
        x, y = x.contiguous(), y.contiguous()
        p = [None if t is None else t.detach().float().contiguous() for t in (gate, post_gamma, post_beta, pre_gamma, pre_beta)]
        post = None if p[1] is None else (p[1], p[2], opts["post_eps"])
        pre = None if p[3] is None else (p[3], p[4], opts["pre_eps"])
        x_new, h = ops.residual_norm(x.detach(), y.detach(), gate=p[0], gate_tanh=opts["gate_tanh"], res_scale=opts["res_scale"], post=post, pre=pre, rms=opts["rms"],
                                     out_dtype=opts["out_dtype"])
        ctx.save_for_backward(x_new, y, *p)
        ctx.opts, ctx.dtypes = opts, [None if t is None else t.dtype for t in (gate, post_gamma, post_beta, pre_gamma, pre_beta)]
        ctx.set_materialize_grads(False)
        return x_new, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dx_new, dh):
        x_new, y, gate, pg, pb, ng, nb = ctx.saved_tensors
        if dx_new is None and dh is None:
            return (None,) * 8
        o = ctx.opts
        if ng is not None and dh is None:                # h went unused: a gradient of zeros for it
            dh = torch.zeros(x_new.shape, dtype=o["out_dtype"], device=x_new.device)
        g = ops.residual_norm_bwd(x_new, y, None if dx_new is None else dx_new.contiguous(), None if dh is None else dh.contiguous(), gate=gate, gate_tanh=o["gate_tanh"],
                                  res_scale=o["res_scale"], post=None if pg is None else (pg, pb, o["post_eps"]), pre=None if ng is None else (ng, nb, o["pre_eps"]), rms=o["rms"])
        return (g.dx, g.dy, *(None if t is None else t.to(d) for t, d in zip(g[2:], ctx.dtypes)), None)


def _norm_of(m, rms, which):
    if m is None:
        return None, None, 0.0
    if not isinstance(m, nn.RMSNorm if rms else nn.LayerNorm):
        raise TypeError("residual_norm: %s is a %s, with rms=%s" % (which, type(m).__name__, rms))
    if m.weight is None:
        raise ValueError("residual_norm: %s has no weight (elementwise_affine=False)" % which)
    return m.weight, getattr(m, "bias", None), torch.finfo(torch.float32).eps if m.eps is None else m.eps


def residual_norm(x, y, gate=None, post=None, pre=None, *, gate_tanh=False, res_scale=1.0, rms=False, out_dtype=torch.bfloat16):
    """(x_new, h) of ops.residual_norm with every gradient; post / pre: nn.LayerNorm (nn.RMSNorm with rms) modules with weights, or None."""
    (pg, pb, pe), (ng, nb, ne) = _norm_of(post, rms, "post"), _norm_of(pre, rms, "pre")
    opts = {"gate_tanh": gate_tanh, "res_scale": float(res_scale), "rms": rms, "out_dtype": out_dtype, "post_eps": pe, "pre_eps": ne}
    return _ResidualNorm.apply(x, y, gate, pg, pb, ng, nb, opts)


class _MlpAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w1, b1, w2, b2, act):
        f = lambda b: None if b is None else b.detach().float().contiguous()  # noqa: E731
        xb = ops.to_bf16(x.detach().contiguous())
        _, qx, sx = ops.act8(xb, want_out=False)
        u = ops.gemm(xb, ops.to_bf16(w1.detach().contiguous()), f(b1))
        a, qu, su = ops.act8(u, act)
        y = ops.gemm(a, ops.to_bf16(w2.detach().contiguous()), f(b2), out_dtype=torch.float32)
        ctx.save_for_backward(qx, sx, qu, su, w1, w2)
        ctx.act, ctx.x_dtype, ctx.dtypes = act, x.dtype, [None if t is None else t.dtype for t in (w1, b1, w2, b2)]
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        qx, sx, qu, su, w1, w2 = ctx.saved_tensors
        dyb = ops.to_bf16(dy.contiguous())
        da = ops.gemm(dyb, ops.transpose_bf16(w2.detach().contiguous()))
        du, a = ops.act8_bwd(qu, su, da, ctx.act, want_out=True)
        dw2, db2 = ops.gemm_tn(dyb, a, colsum=True)
        dw1, db1 = ops.gemm_tn_act8(du, qx, sx, colsum=True)
        dx = ops.gemm(du, ops.transpose_bf16(w1.detach().contiguous()), out_dtype=torch.float32).to(ctx.x_dtype) if ctx.needs_input_grad[0] else None
        return (dx, *(None if d is None else t.to(d) for t, d in zip((dw1, db1, dw2, db2), ctx.dtypes)), None)


def mlp_act8(x, fc1, fc2, act=ops.ACT_QUICKGELU):
    """fc2(act(fc1(x))) for x fp32 / bf16 [rows, D] -> fp32 [rows, D_out] with bf16 products, keeping x and fc1's output as 8-bit checkpoints for the backward pass (1.03
    bytes for a value of either; fc2's input, which has the width of fc1's output, is taken again from that and not kept).  fc1, fc2: nn.Linear whose widths are multiples of 128 (ops.gemm, ops.gemm_tn)."""
    if x.dim() != 2:
        raise ValueError("mlp_act8: x must be [rows, D]")
    for m in (fc1, fc2):                             # (its weight and bias are used, and nothing else that it may do)
        if not isinstance(m, nn.Linear) or type(m).forward is not nn.Linear.forward:
            raise TypeError("mlp_act8: fc1 and fc2 must be nn.Linear, got %s" % type(m).__name__)
    return _MlpAct8.apply(x, fc1.weight, fc1.bias, fc2.weight, fc2.bias, act)


class TokenEmbedding(nn.Embedding):
    """nn.Embedding (same arguments and state dict) whose lookup and gradient are ops.embed_tokens / ops.embed_tokens_bwd; forward(ids, pos=None, scale=1.0).  max_norm,
    scale_grad_by_freq and sparse gradients are refused."""

    def forward(self, ids, pos=None, scale=1.0, out_dtype=None):
        if self.max_norm is not None or self.scale_grad_by_freq or self.sparse:
            raise NotImplementedError("TokenEmbedding: max_norm, scale_grad_by_freq and sparse are not built")
        return embed_tokens(ids, self.weight, pos, scale, self.padding_idx, out_dtype)
