"""The operators as a training step uses them: a teacher's pass reduced to its top logits, a student's step with the fused
feed-forward block and the distillation loss, eagerly, captured, and as thunks over spilling cells."""
import numpy as np
import pytest
import torch

from cacti_b200 import capi, llama_step as LS, ops
from cacti_b200.host import binding as H
from oracle import llama_oracle
from oracle import ref_chain as R
from tests.gpu_util import dev, host
from tests.tolerances import assert_close

pytestmark = pytest.mark.gpu

CFG = LS.LlamaShape(layers=2, d_model=200, heads=2, head_dim=100, ffn=96, vocab=160, seq=128)
B = 2


def _params(cuda, seed):
    return LS.init_weights(CFG, cuda, seed=seed, std=0.08)


def _np_params(P):
    out = {k: host(v) for k, v in P.items() if k != "layers"}
    out["layers"] = [{k: host(v) for k, v in L.items()} for L in P["layers"]]
    return out


def _tokens(seed):
    return dev(R.uniform_int(seed, B * CFG.seq, CFG.vocab))


def test_step_with_the_fused_feed_forward_block(cuda):
    """Held to the composed oracle at the tolerance of the unfused step: both are chains of about forty 16-bit roundings."""
    P = _params(cuda, 1)
    tok, tgt = _tokens(3), _tokens(4)
    ref_loss, ref_g = llama_oracle.step(_np_params(P), host(tok), host(tgt), CFG)
    grads = LS.zeros_like_params(P)
    step = LS.TrainStep(CFG, P, B, ffn="fused")
    loss = step.forward_backward(tok, tgt, grads)
    torch.cuda.synchronize()
    assert host(step.status)[0] == 0
    assert abs(float(loss) - float(ref_loss)) < 2e-3 * abs(float(ref_loss))
    for name in ("lm_head", "head_norm", "embed"):
        assert_close(host(grads[name]), ref_g[name], "float16", name, rtol=2e-2, floor_frac=1.0)
    for li in range(CFG.layers):
        for name, g in grads["layers"][li].items():
            assert_close(host(g), ref_g["layers"][li][name], "float16", f"fused ffn layer {li} {name}", rtol=2e-2, floor_frac=1.0)
    with pytest.raises(ValueError):
        LS.TrainStep(CFG, P, B, ffn="sometimes")


@pytest.mark.parametrize("weight", [1.0, 0.5])
def test_student_step_against_a_teacher(cuda, weight):
    """The step's loss and its output head's gradient are those of the operators called one by one on its logits."""
    teacher_step = LS.TrainStep(CFG, _params(cuda, 7), B, ffn="fused")
    P = _params(cuda, 1)
    tok, tgt = _tokens(3), _tokens(4)
    teacher = teacher_step.teacher_topk(tok, 16, temperature=2.0, weight=weight)
    assert teacher.values.shape == (B * CFG.seq, 16) and teacher.lse is not None
    step, grads = LS.TrainStep(CFG, P, B, ffn="fused"), LS.zeros_like_params(P)
    loss = step.forward_backward(tok, tgt, grads, teacher=teacher)
    nf, _, logits = step._forward(tok, [])
    T = B * CFG.seq
    want, dlogits = torch.zeros(1, device=cuda), None
    if weight < 1:
        want, _, dlogits, _ = ops.softmax_nll_fwd_bwd(logits, tgt, w_scalar=(1 - weight) / T)
    soft, rows, dlogits, _ = ops.distill_topk_fwd_bwd(logits, teacher.values, teacher.indices, teacher.lse, 2.0, w_scalar=weight / T,
                                                      dlogits=dlogits, beta=int(dlogits is not None))
    torch.cuda.synchronize()
    assert torch.equal(loss, want + soft) and (rows >= 0).all() and host(step.status)[0] == 0
    assert torch.equal(grads["lm_head"], ops.gemm(dlogits, nf, True, False))
    assert all(torch.isfinite(g).all() and g.any() for _, g in LS.flat_params(grads))
    # a student that is its own teacher has nothing to learn: q = p on the list and in the bucket.  The teacher's f16 logits are the
    # student's, its lse is rounded to f32 (2^-24 of at most 16): p - q is off by 2^-20 relative, the loss by as much
    same = LS.TrainStep(CFG, P, B, ffn="fused")
    own = same.teacher_topk(tok, 16, temperature=2.0)
    loss = same.forward_backward(tok, tgt, grads, teacher=own)
    assert abs(float(loss)) < 2.0 ** -19


def test_launches_of_the_losses_are_counted(cuda):
    """Two kernels a loss (rows, sum), one more that adds a mixed step's two sums."""
    P, tok, tgt = _params(cuda, 1), _tokens(3), _tokens(4)
    step, grads = LS.TrainStep(CFG, P, B), LS.zeros_like_params(P)
    counts = []
    for weight in (None, 1.0, 0.5):
        teacher = None if weight is None else LS.TrainStep(CFG, P, B).teacher_topk(tok, 16, weight=weight)
        step.forward_backward(tok, tgt, grads, teacher=teacher)
        counts.append(step.launches)
    assert counts[1] == counts[0] and counts[2] == counts[0] + 3


def test_captured_student_step(cuda):
    P = _params(cuda, 1)
    toks, tgts = [_tokens(3), _tokens(5)], [_tokens(4), _tokens(6)]
    teacher_step = LS.TrainStep(CFG, _params(cuda, 7), B, ffn="fused")
    eager = []
    for tok, tgt in zip(toks, tgts):
        grads = LS.zeros_like_params(P)
        teacher = teacher_step.teacher_topk(tok, 20, weight=0.75)
        loss = LS.TrainStep(CFG, P, B, ffn="fused").forward_backward(tok, tgt, grads, teacher=teacher)
        eager.append((loss.clone(), [g.clone() for _, g in LS.flat_params(grads)]))
    grads = LS.zeros_like_params(P)
    step = LS.TrainStep(CFG, P, B, ffn="fused")
    tok, tgt = toks[0].clone(), tgts[0].clone()
    gs = LS.GraphedStep(lambda: step.forward_backward(tok, tgt, grads, teacher=teacher_step.teacher_topk(tok, 20, weight=0.75)))
    for i in (0, 1, 0):
        tok.copy_(toks[i]), tgt.copy_(tgts[i])
        loss = gs.replay()
        torch.cuda.synchronize()
        assert torch.equal(loss, eager[i][0])
        assert all(torch.equal(g, w) for (_, g), w in zip(LS.flat_params(grads), eager[i][1]))
    assert host(step.status)[0] == 0


def test_thunks_over_spilling_cells(cuda):
    """The same operators through the host shim, its soft limit below what the cells take together: same bits."""
    t, d, f, v, k = 200, 256, 520, 4000, 24
    f16, i32 = capi.R_16F, capi.R_32I
    arr = dict(x=R.normal(1, (t, d), np.float16), wg=R.normal(2, (f, d), np.float16, 0.06), wu=R.normal(3, (f, d), np.float16, 0.06),
               dh=R.normal(4, (t, f), np.float16), logits=R.normal(5, (t, v), np.float16, 2.0), teacher=R.normal(6, (t, v), np.float16, 2.0))
    g = {n: dev(a) for n, a in arr.items()}
    h, gate, up = ops.gated_ffn_fwd(g["x"], g["wg"], g["wu"], save=True)
    bwd = ops.gated_ffn_bwd(g["dh"], g["x"], g["wg"], g["wu"], gate, up)
    top = ops.logits_topk(g["teacher"], k, 1.5)
    loss, _, dl, _ = ops.distill_topk_fwd_bwd(g["logits"], *top, 1.5, w_scalar=0.25, want_rows=False)
    ctx = H.Ctx(cuda=True, arena_bytes=16 << 20, soft_limit=6 << 20)
    L, hd = ctx.L, ctx.h
    c = {n: ctx.cell(a) for n, a in arr.items()}
    new = lambda like: ctx.cell(nbytes=like.numel() * like.element_size())
    ch, cg, cu, cx, cwg, cwu = new(h), new(gate), new(up), new(bwd[0]), new(bwd[1]), new(bwd[2])
    cv, ci, ce, cl, cd = new(top[0]), new(top[1]), new(top[2]), ctx.cell(nbytes=4), new(dl)
    st = ctx.cell(np.zeros(1, np.uint32))
    assert L.cbh_thunk_gated_ffn_fwd(hd, H.APPLY, ch, cg, cu, c["x"], c["wg"], c["wu"], t, d, f, f16) == 0
    assert L.cbh_thunk_logits_topk(hd, H.APPLY, cv, ci, ce, c["teacher"], t, v, k, 1.5, f16) == 0
    assert L.cbh_thunk_gated_ffn_bwd(hd, H.APPLY, H.APPLY, cx, cwg, cwu, c["dh"], c["x"], c["wg"], c["wu"], cg, cu, t, d, f, f16) == 0
    assert L.cbh_thunk_distill_topk(hd, H.APPLY, cl, cd, c["logits"], cv, f16, ci, i32, ce, k, 1.5, 0.25, t, v, f16, st) == 0
    for cell, want in ((ch, h), (cg, gate), (cu, up), (cx, bwd[0]), (cwg, bwd[1]), (cwu, bwd[2]), (cv, top[0]), (ci, top[1]), (ce, top[2]),
                       (cl, loss), (cd, dl)):
        w = host(want)
        assert np.array_equal(ctx.get(cell, w), w)
    assert ctx.get(st, np.zeros(1, np.uint32))[0] == 0
    assert ctx.stats()["spills"] > 0 and ctx.stats()["hard_oom"] == 0
    # Accumulate mode adds to what the cells hold; modes the thunks do not have are refused
    assert L.cbh_thunk_distill_topk(hd, H.ACCUMULATE, H.NO_CELL, cd, c["logits"], cv, f16, ci, i32, H.NO_CELL, k, 1.5, 0.25, t, v, f16, H.NO_CELL) == 0
    acc = ops.distill_topk_fwd_bwd(g["logits"], top[0], top[1], None, 1.5, w_scalar=0.25, dlogits=dl.clone(), beta=1)[2]
    assert np.array_equal(ctx.get(cd, host(acc)), host(acc))
    assert L.cbh_thunk_gated_ffn_fwd(hd, H.ACCUMULATE, ch, -1, -1, c["x"], c["wg"], c["wu"], t, d, f, f16) == capi.ERR_INVALID_VALUE
    assert L.cbh_thunk_logits_topk(hd, H.ACCUMULATE, cv, ci, ce, c["teacher"], t, v, k, 1.5, f16) == capi.ERR_INVALID_VALUE
    assert L.cbh_thunk_gated_ffn_fwd(hd, H.APPLY, ch, H.NO_CELL, H.NO_CELL, c["x"], c["wg"], c["wu"], t, d, f, f16) == 0
    assert np.array_equal(ctx.get(ch, host(h)), host(h))
    ctx.close()
