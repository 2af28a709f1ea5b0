"""Argument checks of the distillation and gated feed-forward entry points: none of these calls launches anything."""
from cacti_b200 import capi

P = 0x1000          # non-null and aligned, never dereferenced: every call below is refused first


def _topk(values=P, indices=P, lse=P, logits=P, rows=4, vocab=100, k=10, temperature=1.0, dtype=capi.R_16F):
    return capi.lib().cacti_b200_logits_topk(values, indices, lse, logits, rows, vocab, k, temperature, dtype, None)


def _distill(loss_sum=P, loss_rows=P, dlogits=P, logits=P, tv=P, td=capi.R_16F, ti=P, idt=capi.R_32I, lse=0, k=4, temperature=1.0,
             w=0, rows=4, vocab=100, dtype=capi.R_16F, beta=0, status=0, ws=0, wsb=0):
    return capi.lib().cacti_b200_distill_topk_fwd_bwd(loss_sum, loss_rows, dlogits, logits, tv, td, ti, idt, lse, k, temperature, w,
                                                      1.0, rows, vocab, dtype, beta, status, ws, wsb, None)


def _fwd(h=P, gate=0, up=0, x=P, wg=P, wu=P, t=4, d=16, f=24, dtype=capi.R_16F, ws=0, wsb=0):
    return capi.lib().cacti_b200_gated_ffn_fwd(h, gate, up, x, wg, wu, t, d, f, dtype, ws, wsb, None)


def _bwd(dx=P, dwg=P, dwu=P, dh=P, x=P, wg=P, wu=P, gate=P, up=P, t=4, d=16, f=24, dtype=capi.R_16F, bx=0, bw=0, ws=0x1000, wsb=1 << 30):
    return capi.lib().cacti_b200_gated_ffn_bwd(dx, dwg, dwu, dh, x, wg, wu, gate, up, t, d, f, dtype, bx, bw, ws, wsb, None)


def test_topk_refusals():
    assert _topk(rows=-1) == _topk(vocab=-5) == _topk(k=-1) == capi.ERR_INVALID_VALUE
    assert _topk(values=0) == _topk(indices=0) == _topk(logits=0) == capi.ERR_INVALID_VALUE
    assert _topk(values=P + 1) == _topk(logits=P + 1) == _topk(indices=P + 2) == _topk(lse=P + 2) == capi.ERR_INVALID_VALUE
    assert _topk(logits=P + 2, dtype=capi.R_32F) == capi.ERR_INVALID_VALUE
    for t in (0.0, -1.0, float("nan"), float("inf"), 1e-5, 1e5):
        assert _topk(temperature=t) == capi.ERR_INVALID_VALUE
    assert _topk(dtype=capi.R_32I) == capi.ERR_DTYPE
    assert _topk(k=0) == _topk(k=101) == _topk(vocab=1000, k=257) == _topk(vocab=262145) == _topk(vocab=0) == capi.ERR_SHAPE
    assert _topk(rows=0) == capi.OK


def test_distill_refusals():
    assert _distill(rows=-1) == _distill(vocab=-1) == _distill(beta=2) == capi.ERR_INVALID_VALUE
    assert _distill(logits=0) == _distill(tv=0) == _distill(ti=0) == capi.ERR_INVALID_VALUE
    for name in ("loss_sum", "loss_rows", "lse", "w", "status"):
        assert _distill(**{name: P + 2}) == capi.ERR_INVALID_VALUE, name
    assert _distill(logits=P + 1) == _distill(dlogits=P + 1) == _distill(tv=P + 1) == _distill(ti=P + 2) == capi.ERR_INVALID_VALUE
    for t in (0.0, -2.0, float("nan"), float("inf"), 1e-5, 1e5):
        assert _distill(temperature=t) == capi.ERR_INVALID_VALUE
    assert _distill(dtype=capi.R_16U) == _distill(td=capi.R_32I) == _distill(idt=capi.R_32F) == capi.ERR_DTYPE
    assert _distill(k=0) == _distill(k=257) == _distill(vocab=262145) == capi.ERR_SHAPE
    assert _distill(loss_rows=0) == _distill(loss_rows=0, ws=P, wsb=8) == _distill(loss_rows=0, ws=P + 1, wsb=4096) == capi.ERR_WORKSPACE
    assert _distill(rows=0) == _distill(vocab=0) == capi.OK
    assert capi.lib().cacti_b200_distill_topk_workspace_bytes(8192) >= 8192 * 4


def test_gated_ffn_refusals():
    assert _fwd(t=-1) == _fwd(d=-1) == _fwd(f=-1) == capi.ERR_INVALID_VALUE
    assert _fwd(h=0) == _fwd(x=0) == _fwd(wg=0) == _fwd(wu=0) == capi.ERR_INVALID_VALUE
    assert _fwd(gate=P) == _fwd(up=P) == _fwd(x=P + 1) == capi.ERR_INVALID_VALUE
    assert _fwd(dtype=capi.R_32F) == capi.ERR_DTYPE
    assert _fwd(d=0) == _fwd(f=0) == _fwd(t=1 << 31) == capi.ERR_SHAPE
    assert _fwd(t=0) == capi.OK
    assert _bwd(t=-1) == _bwd(bx=2) == _bwd(bw=-1) == capi.ERR_INVALID_VALUE
    for name in ("dx", "dwg", "dwu", "dh", "x", "wg", "wu", "gate", "up"):
        assert _bwd(**{name: 0}) == capi.ERR_INVALID_VALUE, name
        assert _bwd(**{name: P + 1}) == capi.ERR_INVALID_VALUE, name
    assert _bwd(dtype=capi.R_32F) == capi.ERR_DTYPE
    assert _bwd(d=0) == _bwd(f=0) == capi.ERR_SHAPE
    assert _bwd(ws=0) == _bwd(ws=0x1010) == _bwd(wsb=100) == capi.ERR_WORKSPACE
    L = capi.lib()
    for t, d, f in ((1, 8, 8), (77, 1003, 277), (2048, 3200, 8640)):
        assert L.cacti_b200_gated_ffn_bwd_workspace_bytes(t, d, f, 0) >= L.cacti_b200_gated_ffn_bwd_workspace_bytes(t, d, f, 1) >= 4 * t * f
        assert L.cacti_b200_gated_ffn_fwd_workspace_bytes(t, d, f, 0) >= L.cacti_b200_gated_ffn_fwd_workspace_bytes(t, d, f, 1)


def test_gated_ffn_refuses_copies_that_cannot_be_numbered():
    """Operands whose repacked vectors together pass 32 bits; the counts wrapped to a small number, most rows were never copied and
    the call answered OK.  Sizes one step below are refused for their workspace only."""
    big, f = 1 << 62, 1 << 24
    for d, off in ((1017, 0), (1023, 0), (1016, 2)):                    # odd sizes; aligned rows at an odd address
        assert _fwd(t=2, d=d, f=f, x=P + off, wg=P + off, wu=P + off, ws=0x1000, wsb=big) == capi.ERR_SHAPE
        assert _bwd(t=2, d=d, f=f, x=P + off, wg=P + off, wu=P + off, wsb=big) == capi.ERR_SHAPE
    assert _fwd(t=2, d=1025, f=16700000, ws=0x1000, wsb=big) == _bwd(t=2, d=1025, f=16700000, wsb=big) == capi.ERR_SHAPE
    far = 1 << 50                                                       # the forward's output apart from its inputs
    assert _fwd(h=far, t=2, d=1017, f=f // 2, ws=0, wsb=0) == _bwd(t=2, d=1017, f=f // 2, ws=0, wsb=0) == capi.ERR_WORKSPACE
    assert _fwd(h=far, t=2, d=1016, f=f, x=P + 2, ws=0, wsb=0) == _bwd(t=2, d=1016, f=f, x=P + 2, ws=0, wsb=0) == capi.ERR_WORKSPACE   # x alone


def test_outputs_that_share_bytes_with_inputs_are_refused():
    """Also by one element, at either end; buffers that touch are apart (those calls are not made here: they would launch)."""
    A = [(i + 1) << 40 for i in range(9)]                               # addresses of buffers far apart
    n = 4 * 100 * 2                                                     # logits of 4 x 100, 16 bit
    for at in (A[0], A[0] + 2, A[0] - 2, A[0] + n - 2, A[0] - n + 2):
        assert _distill(logits=A[0], dlogits=at, loss_sum=A[1], loss_rows=A[2], tv=A[3], ti=A[4]) == capi.ERR_INVALID_VALUE
    k = 10
    for at in (A[0], A[0] + n - 2, A[0] - 4 * k * 2 + 2):
        assert _topk(logits=A[0], values=at, indices=A[1], lse=A[2]) == capi.ERR_INVALID_VALUE
    for at in (A[0], A[0] + n - 4, A[0] - 4 * k * 4 + 4):
        assert _topk(logits=A[0], values=A[1], indices=at, lse=A[2]) == capi.ERR_INVALID_VALUE
    assert _topk(logits=A[0], values=A[1], indices=A[2], lse=A[0] + 4) == _topk(logits=A[0], values=A[1], indices=A[2], lse=A[0] - 12) == capi.ERR_INVALID_VALUE
    t, d, f = 4, 16, 24
    fwd = dict(h=A[0], gate=A[1], up=A[2], x=A[3], wg=A[4], wu=A[5])
    size = dict(h=t * f, gate=t * f, up=t * f, x=t * d, wg=f * d, wu=f * d)
    for o in ("h", "gate", "up"):
        for other in fwd:
            if other != o:
                for at in (fwd[other], fwd[other] + 2 * size[other] - 2, fwd[other] - 2 * size[o] + 2):
                    assert _fwd(**{**fwd, o: at}, t=t, d=d, f=f) == capi.ERR_INVALID_VALUE, (o, other)
    bwd = dict(dx=A[0], dwg=A[1], dwu=A[2], dh=A[3], x=A[4], wg=A[5], wu=A[6], gate=A[7], up=A[8])
    size = dict(dx=t * d, dwg=f * d, dwu=f * d, dh=t * f, x=t * d, wg=f * d, wu=f * d, gate=t * f, up=t * f)
    for o in ("dx", "dwg", "dwu"):
        for other in bwd:
            if other != o:
                for at in (bwd[other], bwd[other] + 2 * size[other] - 2, bwd[other] - 2 * size[o] + 2):
                    assert _bwd(**{**bwd, o: at}, t=t, d=d, f=f) == capi.ERR_INVALID_VALUE, (o, other)
