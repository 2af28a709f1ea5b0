"""The teacher's listed logits (logits_topk) and the distillation loss with its gradient, against torch in 64 bits.

Tolerances, with u = eps / 2 of the storage type (one rounding) and 2^-24 = one f32 rounding:
  an exponential 2^((x - m) c): the approximate ex2 is good to 2^-22, its argument A = (x - m) c log2(e) carries three
  roundings, so its relative error is at most 2^-22 + 3 ln2 A 2^-24 < 2^-22 (1 + A);
  a sum of V positive terms over 256 or more threads: each thread adds at most V / 256 + 8 of them, the tree 16 more:
  S = (V / 256 + 24) 2^-24;
  a gradient entry is a sum of at most three terms built from one exponential and two sums: its f32 error is at most
  (2 S + 2^-22 (4 + A)) times the sum of the terms' sizes, then one rounding to the type (two when it is added);
  the loss holds log E of such sums (absolute error: their relative one; the weighted A of a softmax is at most
  log2 V <= 18) and is rounded once to f32.
"""
import math

import pytest
import torch

from cacti_b200 import capi, ops

pytestmark = pytest.mark.gpu

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}


def _u(dt):
    return torch.finfo(dt).eps / 2


def _logits(rows, vocab, dt, seed, std=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=g) * std
    j = torch.randint(0, vocab, (rows, 3), device="cuda", generator=g)
    return x.scatter_add_(1, j, torch.full((rows, 3), 6.0, device="cuda")).to(dt)


def _at_offset(t, off):
    """A contiguous copy whose first element lies `off` elements behind a 256-byte boundary, with room around it."""
    buf = torch.full((t.numel() + off + 64,), 7.0 if t.is_floating_point() else 7, dtype=t.dtype, device=t.device)
    v = buf[off:off + t.numel()].view(t.shape)
    v.copy_(t)
    return v, buf


def _ref(x, z, idx, lse, tau, w):
    """(loss per row, gradient, size of the gradient's terms, A, P, r, rest's A) in 64 bits; invalid slots already -1."""
    x, z, idx = x.double(), z.double() / tau, idx.long()
    rows, V = x.shape
    used = idx >= 0
    z = torch.where(used, z, torch.full_like(z, -math.inf))
    col = torch.where(used, idx, V)
    listed = torch.zeros(rows, V + 1, dtype=torch.bool, device=x.device).scatter_(1, col, True)[:, :V]
    some = used.any(1)
    if lse is None:
        lt = torch.logsumexp(z, 1, keepdim=True)
        logp = torch.where(torch.isneginf(lt), torch.full_like(z, -math.inf), z - torch.where(torch.isneginf(lt), torch.zeros_like(lt), lt))
    else:
        logp = z - lse.double()[:, None]
    p = torch.exp(logp)
    r = (1 - p.sum(1)).clamp(min=0) * some * (~listed).any(1) if lse is not None else torch.zeros(rows, dtype=torch.float64, device=x.device)
    logq = torch.log_softmax(x / tau, 1)
    lrest = torch.logsumexp(torch.where(listed, torch.full_like(logq, -math.inf), logq), 1)
    loss = torch.where(p > 0, p * (logp - torch.gather(logq, 1, idx.clamp(min=0))), torch.zeros_like(p)).sum(1)
    loss = loss + torch.where(r > 0, torch.xlogy(r, r) - r * lrest, torch.zeros_like(r))
    P = p.sum(1) + r
    q = torch.exp(logq)
    share = torch.where(listed | (r[:, None] == 0), torch.zeros_like(q), r[:, None] * torch.exp(logq - lrest[:, None]))
    pd = torch.zeros(rows, V + 1, dtype=torch.float64, device=x.device).scatter_add_(1, col, p)[:, :V]
    sc = w.double()[:, None] / tau
    grad = sc * (P[:, None] * q - pd - share)
    mag = sc.abs() * (P[:, None] * q + pd + share)
    live = w != 0
    dead = ~live[:, None]
    return (loss.masked_fill(~live, 0.0), grad.masked_fill(dead, 0.0), mag.masked_fill(dead, 0.0),
            (x.max(1, keepdim=True).values - x) / tau * 1.4427, P, r)


def _check(got, ref, dt, V, old=None, what=""):
    loss_sum, loss_rows, grad = got
    rl, rg, mag, A, P, r = ref
    S = (V / 256 + 24) * 2.0 ** -24
    if loss_rows is not None:
        Amax = A.amax(1)
        tol = 2.0 ** -23 * rl.abs() + P * (2 * S + 2.0 ** -22 * 20) + r * (2 * S + 2.0 ** -22 * (2 + Amax)) + 1e-12
        bad = (loss_rows.double() - rl).abs() > tol
        assert not bad.any(), (what, "loss", (loss_rows.double() - rl)[bad][:4], tol[bad][:4])
    if grad is not None:
        tol = _u(dt) * rg.abs() + mag * (2 * S + 2.0 ** -22 * (4 + A)) * (1 + _u(dt)) + TINY[dt]
        tgt = rg
        if old is not None:
            tgt = rg + old.double()
            tol = tol + _u(dt) * tgt.abs() + TINY[dt]
        err = (grad.double() - tgt).abs()
        bad = err > tol
        assert not bad.any(), (what, "gradient", int(bad.sum()), grad[bad][:4], tgt[bad][:4], tol[bad][:4])


# ---- the teacher's side -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 7), (5, 100, 1), (4, 257, 256), (2, 1000, 33), (7, 4099, 64),
                                          (300, 2048, 17), (3, 32000, 128), (2, 50001, 256), (1, 131072, 100),
                                          (1, 262144, 5)])
def test_topk_values_indices_lse(cuda, dtype, rows, vocab, k):
    x = _logits(rows, vocab, DT[dtype], rows + vocab)
    for tau, off in ((1.0, 0), (2.5, 1)):
        xv, _ = _at_offset(x, off)
        v, i, lse = ops.logits_topk(xv, k, temperature=tau)
        sv, si = torch.sort(x.float(), dim=1, descending=True, stable=True)
        assert torch.equal(i.long(), si[:, :k])
        assert torch.equal(v.float(), sv[:, :k])
        ref = torch.logsumexp(x.double() / tau, 1)
        tol = 2.0 ** -23 * ref.abs() + (vocab / 256 + 24) * 2.0 ** -24 + 2.0 ** -22 * 20
        assert ((lse.double() - ref).abs() <= tol).all()
    v2, i2, none = ops.logits_topk(x, k, want_lse=False)
    assert none is None and torch.equal(i2.long(), si[:, :k]) and torch.equal(v2.float(), sv[:, :k])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("vocab", [40, 1000, 9001, 40000])
def test_topk_ties_infinities_zeros_nan(cuda, dtype, vocab):
    dt, k = DT[dtype], 32
    inf = math.inf
    g = torch.Generator(device="cuda").manual_seed(vocab)
    rows = [torch.zeros(vocab, device="cuda"),                                              # one value everywhere
            torch.full((vocab,), -inf, device="cuda"),                                      # nothing left by the mask
            torch.full((vocab,), torch.finfo(dt).min, device="cuda"),                       # the type's lowest value
            torch.randint(0, 3, (vocab,), device="cuda", generator=g).float(),              # many ties
            torch.where(torch.arange(vocab, device="cuda") % 97 == 5, 1.0, -inf),           # few left, equal
            torch.where(torch.rand(vocab, device="cuda", generator=g) < 0.5, 0.0, -0.0),    # both zeros are one value
            torch.arange(vocab, device="cuda").float() / vocab,                             # rising: ties after rounding
            torch.arange(vocab, 0, -1, device="cuda").float() / vocab,                      # falling
            torch.where(torch.arange(vocab, device="cuda") == vocab - 1, inf, 1.0),         # +inf
            torch.where(torch.arange(vocab, device="cuda") % 256 < 1, 5.0, 0.0)]            # large values in few columns
    x = torch.stack(rows).to(dt)
    v, i, lse = ops.logits_topk(x, k)
    sv, si = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True)               # -0 + 0 = +0
    assert torch.equal(i.long(), si[:, :k])
    assert torch.equal(v.float() + 0.0, sv[:, :k])
    ref = torch.logsumexp(x.double(), 1)
    fin = torch.isfinite(ref)
    assert torch.equal(lse[~fin].double(), ref[~fin])
    assert ((lse.double() - ref)[fin].abs() <= 2.0 ** -23 * ref[fin].abs() + (vocab / 256 + 24) * 2.0 ** -24 + 2.0 ** -22 * 20).all()
    # NaN is above everything, in index order
    x = _logits(2, vocab, dt, 3)
    x[0, 7], x[0, 3], x[1, 11] = math.nan, math.nan, inf
    v, i, lse = ops.logits_topk(x, k)
    assert i[0, :2].tolist() == [3, 7] and v[0, :2].isnan().all() and lse[0].isnan()
    rest = x[0].float().clone()
    rest[[3, 7]] = -inf
    assert torch.equal(i[0, 2:].long(), torch.sort(rest, descending=True, stable=True).indices[:k - 2])
    assert i[1, 0] == 11 and lse[1] == inf


def test_topk_runs_twice_alike_and_writes_nothing_else(cuda):
    x = _logits(50, 3001, torch.float16, 9)
    L = capi.lib()
    k = 20
    vb, ib, lb = (torch.full((n + 16,), 9, dtype=d, device="cuda") for n, d in ((50 * k, torch.float16), (50 * k, torch.int32), (50, torch.float32)))
    for _ in range(2):
        assert L.cacti_b200_logits_topk(vb[8:].data_ptr(), ib[8:].data_ptr(), lb[8:].data_ptr(), x.data_ptr(), 50, 3001, k, 1.0,
                                        capi.R_16F, torch.cuda.current_stream().cuda_stream) == capi.OK
    v, i, lse = ops.logits_topk(x, k)
    for b, t in ((vb, v), (ib, i), (lb, lse)):
        assert torch.equal(b[8:-8].view(t.shape), t) and (b[:8] == 9).all() and (b[-8:] == 9).all()


# ---- the student's side ---------------------------------------------------------------------------------------------
CASES = [(1, 2, 1), (3, 9, 9), (5, 100, 3), (4, 256, 256), (33, 1000, 17), (6, 4099, 64), (300, 2048, 8), (4, 32000, 64),
         (3, 50001, 256), (2, 131072, 128), (1, 262144, 7)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,k", CASES)
def test_loss_and_gradient(cuda, dtype, tail, rows, vocab, k):
    dt, tau = DT[dtype], 1.5
    x, z = _logits(rows, vocab, dt, 1), _logits(rows, vocab, torch.float32, 2)
    tv, ti, lse = ops.logits_topk(z, k, temperature=tau)
    lse = lse if tail else None
    w = torch.linspace(0.5, 3.0, rows, device="cuda") * (64.0 if dt == torch.float16 else 1.0)
    w[rows // 2:rows // 2 + rows // 4] = 0.0
    ref = _ref(x, tv, ti, lse, tau, w)
    for off in (0, 3):
        xv, _ = _at_offset(x, off)
        loss, per_row, grad, status = ops.distill_topk_fwd_bwd(xv, tv, ti, lse, tau, w)
        _check((loss, per_row, grad), ref, dt, vocab, what=f"offset {off}")
        assert int(status) == 0
        want = (w.double() * per_row.double()).sum()
        assert abs(float(loss) - float(want)) <= 2.0 ** -23 * abs(float(want)) + 1e-12
        # added to what is there, through a view of another alignment, nothing around it touched
        old = _logits(rows, vocab, dt, 5, std=1.0)
        acc, buf = _at_offset(old, (off + 1) % 4)
        out = ops.distill_topk_fwd_bwd(xv, tv, ti, lse, tau, w, dlogits=acc, beta=1)[2]
        _check((None, None, out), ref, dt, vocab, old=old, what=f"beta 1, offset {off}")
        n0 = (off + 1) % 4
        assert (buf[:n0] == 7).all() and (buf[n0 + old.numel():] == 7).all()
        assert torch.equal(acc[w == 0], old[w == 0])
    # forward only, and a scalar weight
    l2, r2, none, _ = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w_scalar=0.25, want_grad=False)
    assert none is None
    _check((l2, r2, None), _ref(x, tv, ti, lse, tau, torch.full_like(w, 0.25)), dt, vocab, what="forward only")
    l3, none, _, _ = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w_scalar=0.25, want_grad=False, want_rows=False)
    assert none is None and torch.equal(l3, l2)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("idx_dtype", [torch.int32, torch.uint16])
def test_unused_slots_and_types_of_the_list(cuda, dtype, tail, idx_dtype):
    dt, rows, vocab, k, tau = DT[dtype], 9, 3001, 24, 2.0
    x, z = _logits(rows, vocab, dt, 1), _logits(rows, vocab, torch.float32, 2)
    tv, ti, lse = ops.logits_topk(z, k, temperature=tau)
    ti[0, :] = -1                                                       # no slot
    ti[1, 1:] = -1                                                      # one slot
    ti[2, ::2] = -1                                                     # holes
    ti[3, :5] = -1
    tv[4, 3] = -math.inf                                                # a listed word the teacher excludes
    tv[5, :] = -math.inf                                                # nothing left of the list
    for tdt in DT.values():
        t = tv.to(tdt)
        idx = ti if idx_dtype == torch.int32 else (ti & 0xffff).to(torch.int32).to(torch.int16).view(torch.uint16)
        w = torch.full((rows,), 100.0, device="cuda")
        ls = lse if tail else None
        loss, per_row, grad, status = ops.distill_topk_fwd_bwd(x, t, idx, ls, tau, w)
        ref = _ref(x, t, ti, ls, tau, w)
        _check((loss, per_row, grad), ref, dt, vocab)
        assert int(status) == 0 and per_row[0] == 0 and not grad[0].any()
        if not tail:
            assert per_row[5] == 0 and not grad[5].any()


@pytest.mark.parametrize("dtype", list(DT))
def test_bad_and_repeated_indices_are_reported_and_left_out(cuda, dtype):
    dt, rows, vocab, k = DT[dtype], 6, 5003, 20
    x, z = _logits(rows, vocab, dt, 1), _logits(rows, vocab, torch.float32, 2)
    tv, ti, lse = ops.logits_topk(z, k)
    w = torch.full((rows,), 10.0, device="cuda")
    clean = ops.distill_topk_fwd_bwd(x, tv, ti, lse, w=w)
    bad = ti.clone()
    bad[1, 4], bad[2, 0], bad[3, 19], bad[4, 7] = vocab, -2, -2 ** 31, ti[4, 2]        # the last: listed twice
    loss, per_row, grad, status = ops.distill_topk_fwd_bwd(x, tv, bad, lse, w=w)
    assert int(status) == capi.ERR_INDEX_RANGE
    assert per_row.isnan().tolist() == [False, True, True, True, True, False] and loss.isnan()
    assert torch.equal(per_row[[0, 5]], clean[1][[0, 5]]) and torch.equal(grad[[0, 5]], clean[2][[0, 5]])
    left = bad.clone()
    left[1, 4] = left[2, 0] = left[3, 19] = left[4, 7] = -1                            # left out: as if unused
    ref = _ref(x, tv, left, lse, 1.0, w)
    _check((None, None, grad), ref, dt, vocab)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("vocab", [64, 5000, 40000])
def test_masked_and_extreme_rows(cuda, dtype, tail, vocab):
    dt, k = DT[dtype], 16
    inf, low = math.inf, torch.finfo(dt).min
    x = _logits(8, vocab, dt, 1)
    z = _logits(8, vocab, torch.float32, 2)
    ar = torch.arange(vocab, device="cuda")
    x[0] = torch.where(ar % 3 == 0, x[0].float(), -inf).to(dt)          # masked words of the student
    z[0] = torch.where(ar % 3 == 0, z[0], -inf)
    x[1] = low                                                          # a row of the type's lowest value: uniform
    x[2] = torch.where(ar < vocab // 2, x[2], torch.full_like(x[2], low))
    x[3] = 0.0
    x[4, :] = -inf                                                      # nothing left: NaN, as the row softmax
    x[5, 1] = inf                                                       # NaN likewise
    x[6] = torch.where(ar == 7, 60.0, 0.0).to(dt)                       # one word holds everything
    tv, ti, lse = ops.logits_topk(z, k)
    tail_lse = lse if tail else None
    w = torch.full((8,), 2.0, device="cuda")
    w[7] = 0.0
    x[7] = math.nan                                                     # a padded row is not read
    loss, per_row, grad, status = ops.distill_topk_fwd_bwd(x, tv, ti, tail_lse, w=w)
    ref = _ref(x, tv, ti, tail_lse, 1.0, w)
    ok = [0, 1, 2, 3, 6]
    assert int(status) == 0 and per_row[7] == 0 and not grad[7].any()
    assert grad[4].isnan().all() and grad[5].isnan().any() and per_row[4:6].isnan().all()
    fin = ref[0].isfinite()
    for i in ok:
        part = tuple(t[i:i + 1] for t in ref)
        if fin[i]:
            _check((None, per_row[i:i + 1], grad[i:i + 1]), part, dt, vocab, what=f"row {i}")
        else:                                                           # teacher mass where the student has none
            assert per_row[i] == ref[0][i]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("vocab", [64, 5003, 50001, 200000])
def test_rows_without_a_list_are_zero_whatever_their_logits(cuda, dtype, vocab):
    """No used slot, or used slots that all hold -inf: loss 0, gradient 0, also where the student's logits are no numbers."""
    dt, k, rows = DT[dtype], 12, 9
    x = _logits(rows, vocab, dt, 1)
    x[1], x[2, 3], x[3, vocab - 1], x[4], x[5, ::2] = math.nan, math.inf, math.nan, -math.inf, math.inf
    tv, ti, lse = ops.logits_topk(_logits(rows, vocab, torch.float32, 2), k)
    ti[:5] = -1
    tv[5:7] = -math.inf
    ti[7, 1:], ti[7, 0] = -1, vocab                                     # the only slot used is outside the vocabulary
    empty, w = list(range(7)), torch.linspace(1, 3, rows, device="cuda")
    keep = _logits(rows, vocab, dt, 3)
    for ls, zero in ((None, empty), (lse, empty[:5])):                  # with the teacher's sum rows 5, 6 put everything on the rest
        loss, per_row, grad, status = ops.distill_topk_fwd_bwd(x, tv, ti, ls, w=w)
        assert not per_row[zero].any() and not grad[zero].any()
        assert per_row[7].isnan() and not grad[7].any() and int(status) == capi.ERR_INDEX_RANGE and loss.isnan()
        alone = ops.distill_topk_fwd_bwd(x[8:].contiguous(), tv[8:].contiguous(), ti[8:].contiguous(), None if ls is None else ls[8:], w=w[8:].contiguous())
        assert per_row[8] > 0 and torch.equal(per_row[8:], alone[1])
        acc = ops.distill_topk_fwd_bwd(x, tv, ti, ls, w=w, dlogits=keep.clone(), beta=1)[2]
        assert torch.equal(acc[zero + [7]], keep[zero + [7]]) and not torch.equal(acc[8], keep[8])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("vocab", [40, 5003, 50001])
def test_a_list_without_mass_leaves_it_all_beside_the_list(cuda, dtype, vocab):
    """Used slots that all hold -inf: nothing to learn when the list is renormalised, the loss -log Q with the teacher's sum."""
    dt, k = DT[dtype], 9
    x = _logits(4, vocab, dt, 1)
    _, ti, lse = ops.logits_topk(_logits(4, vocab, torch.float32, 2), k)
    tv = torch.full((4, k), -math.inf, device="cuda")
    w = torch.ones(4, device="cuda")
    total, per_row, grad, _ = ops.distill_topk_fwd_bwd(x, tv, ti, None, w=w)
    assert not per_row.any() and not grad.any() and float(total) == 0.0
    got = ops.distill_topk_fwd_bwd(x, tv, ti, lse, w=w)
    ref = _ref(x, tv, ti, lse, 1.0, w)
    logq = torch.log_softmax(x.double(), 1)
    rest = torch.logsumexp(logq.scatter(1, ti.long(), -math.inf), 1)
    assert torch.allclose(ref[0], -rest, rtol=1e-12, atol=1e-12)
    _check(got[:3], ref, dt, vocab)


def test_exponentials_and_logarithms_of_the_list(cuda):
    """Two words, both listed: the loss is then made of the list's own exponentials and logarithms alone.  The exponentials are good to
    3e-10 (the series' next term over its smallest value), a logarithm passes that on: two sums and their two logarithms, 1.2e-9; the
    probabilities' 3e-10 multiplies log p - log q; c is rounded to f32, 2^-24 of the student's exponents, which acts on the
    difference of the distributions; one rounding to f32."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n = 4000
    a = (torch.rand(n, device="cuda", generator=g) * 12 - 5).exp()                           # 0.007 to 1100
    b = a * (1 + torch.randn(n, device="cuda", generator=g) * torch.logspace(-6, -0.5, n, device="cuda"))
    shift = torch.randn(n, 1, device="cuda", generator=g) * 30
    x = torch.stack([torch.zeros_like(a), -a], 1) + shift
    z = torch.stack([torch.zeros_like(b), -b], 1)
    ti = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda").repeat(n, 1)
    w = torch.ones(n, device="cuda")
    _, rows, _, status = ops.distill_topk_fwd_bwd(x, z, ti, w=w)
    loss = _ref(x, z, ti, None, 1.0, w)[0]
    lp, lq = torch.log_softmax(z.double(), 1), torch.log_softmax(x.double(), 1)
    p, q = lp.exp(), lq.exp()
    A = (x.double() - x.double().amax(1, keepdim=True)).abs().amax(1)
    tol = 1.2e-9 + 3e-10 * (p * (lp - lq).abs()).sum(1) + 2.0 ** -24 * A * (p - q).abs().sum(1) + 2.0 ** -24 * loss + 2.0 ** -149
    err = (rows.double() - loss).abs()
    assert int(status) == 0 and (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("tau,vocab,k,noise", [(1.5, 50001, 17, 0.05), (4.0, 32000, 64, 0.05), (1.0, 8000, 128, 0.2), (2.0, 131072, 100, 0.02)])
def test_a_student_near_its_teacher(cuda, tau, vocab, k, noise):
    """Loss and gradient are then small differences of large terms.  What does not cancel: the error of the sum over the unlisted
    positions, times the difference of its share from the teacher's; the sum is made of f32 sums of at most 128 terms whose roundings
    (2^-24, growing with the square root of the number of terms) average over more than 100 threads: below 2^-25; and
    the temperature's rounding to f32, 2^-24 of the difference of the mean logits.  Single exponentials are good to 2^-22, the listed
    ones to 2^-24."""
    z = _logits(64, vocab, torch.float32, 11, std=1.5)
    g = torch.Generator(device="cuda").manual_seed(12)
    x = z + noise * torch.randn(64, vocab, device="cuda", generator=g)
    tv, ti, _ = ops.logits_topk(z, k, temperature=tau)
    lse = torch.logsumexp(z.double() / tau, 1).float()
    w = torch.ones(64, device="cuda")
    loss, rows, grad, _ = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w)
    rl, rg, mag, A, P, r = _ref(x, tv, ti, lse, tau, w)
    assert (rl < 0.05).all()
    assert ((rows.double() - rl).abs() <= 2.0 ** -22 * rl + noise * 2.0 ** -24 * 8).all(), ((rows.double() - rl).abs() / rl).max()
    assert ((grad.double() - rg).abs() <= 2.0 ** -21 * rg.abs() + 2.0 ** -23 * mag * noise * 8 + 2.0 ** -24 * mag).all()


def test_gradient_against_differences(cuda):
    """Central differences of the loss in 64 bits of torch autograd-free form: the formula's gradient is the loss's."""
    torch.manual_seed(0)
    rows, vocab, k, tau, eps = 2, 50, 7, 1.7, 1e-5
    x, z = torch.randn(rows, vocab, device="cuda") * 2, torch.randn(rows, vocab, device="cuda") * 2
    tv, ti, lse = ops.logits_topk(z, k, temperature=tau)
    w = torch.ones(rows, device="cuda")
    for ls in (None, lse):
        grad = ops.distill_topk_fwd_bwd(x, tv, ti, ls, tau, w)[2]
        for j in (0, 13, int(ti[0, 0]), int(ti[0, k - 1])):
            d = torch.zeros(rows, vocab, device="cuda", dtype=torch.float64)
            d[:, j] = eps
            hi, lo = (_ref(x.double() + s * d, tv, ti, ls, tau, w)[0] for s in (1, -1))
            num = (hi - lo) / (2 * eps)
            # differences: O(eps^2) + 1e-16 / eps; the kernel's entries: f32
            assert ((grad[:, j].double() - num).abs() <= 1e-9 + 2.0 ** -18).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("vocab", [2992, 4099, 50000, 120000])
def test_a_row_of_the_teacher_does_not_depend_on_its_neighbours(cuda, dtype, vocab):
    # rows of large and of small logits in turn before copies of one row, enough rows that each block takes several
    rows = 2000 if vocab < 10000 else 1000
    g = torch.Generator(device="cuda").manual_seed(vocab)
    one = torch.randn(vocab, device="cuda", generator=g) * 3
    x = one.repeat(rows, 1)
    other = torch.rand(rows, device="cuda", generator=g) < 0.5
    x[other] += (torch.rand(int(other.sum()), 1, device="cuda", generator=g) - 0.5) * 200
    v, i, lse = ops.logits_topk(x.to(DT[dtype]), 20)
    same = ~other
    first = int(same.nonzero()[0])
    assert torch.equal(lse[same], lse[first].expand(int(same.sum())))
    assert torch.equal(v[same], v[first].expand(int(same.sum()), 20)) and torch.equal(i[same], i[first].expand(int(same.sum()), 20))
    ref = torch.logsumexp(x.to(DT[dtype]).double(), 1)
    # exponentials at up to 2^60 or re-referenced: 2^-22 (1 + 60) of the sum, one rounding of the result
    assert ((lse.double() - ref).abs() <= 61 * 2.0 ** -22 + (vocab / 256 + 24) * 2.0 ** -24 + ref.abs() * 2.0 ** -24).all()


def test_an_empty_vocabulary_has_zero_losses(cuda):
    x = torch.empty(5, 0, device="cuda", dtype=torch.float16)
    tv = torch.zeros(5, 2, device="cuda", dtype=torch.float16)
    ti = torch.full((5, 2), -1, device="cuda", dtype=torch.int32)
    torch.full((5,), 7.0, device="cuda")                        # what an allocation may find in its memory
    total, loss, d, status = ops.distill_topk_fwd_bwd(x, tv, ti)
    assert loss.tolist() == [0.0] * 5 and total.item() == 0.0 and d.shape == (5, 0) and status.item() == 0


def test_streams_graphs_and_empty_calls(cuda):
    x, z = _logits(40, 4000, torch.bfloat16, 1), _logits(40, 4000, torch.bfloat16, 2)
    want = ops.distill_topk_fwd_bwd(x, *ops.logits_topk(z, 30), want_rows=False)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.distill_topk_fwd_bwd(x, *ops.logits_topk(z, 30), want_rows=False)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    xs, zs = x.clone(), z.clone()
    graphs = []
    for _ in range(2):                                                  # two graphs of the same calls, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.distill_topk_fwd_bwd(xs, *ops.logits_topk(zs, 30), want_rows=False)
        graphs.append((g, out))
    xs.copy_(x.flip(0)), zs.copy_(z.flip(0))
    for g, _ in graphs:
        g.replay()
    for _, out in graphs:
        assert torch.equal(out[2].flip(0), want[2])
    e = ops.distill_topk_fwd_bwd(x[:0], *ops.logits_topk(z[:0], 30))
    assert e[0].item() == 0 and e[1].numel() == 0 and e[2].numel() == 0
    err = capi.C.c_uint(0)
    assert capi.lib().cacti_b200_device_error(capi.C.byref(err)) == capi.OK and err.value == 0


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("rows,vocab,k", [(4, 1030, 100), (4, 1500, 128), (148, 1999, 128), (2, 2050, 256), (4, 3000, 256), (3, 4090, 256)])
def test_topk_of_few_rows_with_fewer_groups_than_k(cuda, dtype, rows, vocab, k):
    """Few rows of 16-bit logits are read by 1024 threads; below 16 k words fewer than k of the groups that bound the k-th largest hold
    any, and the exact search decides."""
    x = _logits(rows, vocab, DT[dtype], vocab)
    x[0, ::3] = -math.inf
    for off in (0, 1):
        xv, _ = _at_offset(x, off)
        v, i, lse = ops.logits_topk(xv, k)
        sv, si = torch.sort(x.float(), dim=1, descending=True, stable=True)
        assert torch.equal(i.long(), si[:, :k]) and torch.equal(v.float(), sv[:, :k])
        ref = torch.logsumexp(x.double(), 1)
        assert ((lse.double() - ref).abs() <= 2.0 ** -23 * ref.abs() + (vocab / 256 + 24) * 2.0 ** -24 + 2.0 ** -22 * 20).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab", [(70, 150001), (41, 200000)])
def test_long_f32_rows_one_after_another_in_a_cluster(cuda, tail, rows, vocab):
    """f32 rows above about 135000 words: parts that are not held in registers and have one slot, several rows to a cluster (a device
    runs at most 18 clusters of eight blocks)."""
    k, tau = 33, 1.3
    x, z = _logits(rows, vocab, torch.float32, 1), _logits(rows, vocab, torch.float32, 2)
    tv, ti, lse = ops.logits_topk(z, k, temperature=tau)
    ti[::4, 5:] = -1
    ti[1] = -1
    lse = lse if tail else None
    w = torch.linspace(0.5, 3.0, rows, device="cuda")
    w[3::5] = 0.0
    ref = _ref(x, tv, ti, lse, tau, w)
    got = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w)
    _check(got[:3], ref, torch.float32, vocab)
    old = _logits(rows, vocab, torch.float32, 5, std=1.0)
    acc = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w, dlogits=old.clone(), beta=1)[2]
    _check((None, None, acc), ref, torch.float32, vocab, old=old, what="beta 1")
    fwd = ops.distill_topk_fwd_bwd(x, tv, ti, lse, tau, w, want_grad=False)
    assert torch.equal(fwd[1], got[1]) and int(got[3]) == 0


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("part", [256, 700])
def test_shorter_parts_of_a_row(cuda, dtype, part):
    """The tuning knob: rows shared by more blocks than they need, same results within the same bounds."""
    dt, rows, vocab, k = DT[dtype], 40, 9001, 20
    x, z = _logits(rows, vocab, dt, 1), _logits(rows, vocab, torch.float32, 2)
    tv, ti, lse = ops.logits_topk(z, k)
    w = torch.ones(rows, device="cuda")
    L = capi.lib()
    try:
        assert L.cacti_b200_tune(b"distill_part", part) == capi.OK
        got = ops.distill_topk_fwd_bwd(x, tv, ti, lse, w=w)
    finally:
        assert L.cacti_b200_tune(b"distill_part", 4096) == capi.OK
    _check(got[:3], _ref(x, tv, ti, lse, 1.0, w), dt, vocab)


def test_more_lengths_of_rows_than_a_launch_cache_keeps(cuda):
    """Two hundred sizes of shared memory for one kernel, and for its cluster form, then the first ones again."""
    x, z = (_logits(1, 42000 + 16 * 200, torch.float16, s) for s in (1, 2))
    first = {}
    for n in list(range(200)) + [0, 1, 70, 135, 199]:
        for base in (20000, 42000):
            v = base + 16 * n                                           # each another number of vectors a row
            xs, zs = x[:, :v].contiguous(), z[:, :v].contiguous()
            k = 1 + 32 * (n % 8)
            got = ops.distill_topk_fwd_bwd(xs, *ops.logits_topk(zs, k))
            if v in first:
                assert torch.equal(got[1], first[v][0]) and torch.equal(got[2], first[v][1])
                continue
            first[v] = got[1:3]
            if n % 40 == 0 or n == 199:
                tv, ti, lse = ops.logits_topk(zs, k)
                _check(got[:3], _ref(xs, tv, ti, lse, 1.0, torch.ones(1, device="cuda")), torch.float16, v, what=f"{v}")


def test_two_host_threads_with_rows_of_two_lengths(cuda):
    """One kernel with two sizes of shared memory: what one thread's call asks for must not take away from the other's."""
    import threading
    cases = {v: (_logits(30, v, torch.float16, v), *ops.logits_topk(_logits(30, v, torch.float16, v + 1), 64)) for v in (32000, 20000)}
    torch.cuda.synchronize()
    got, errors = {}, []
    turns = [threading.Semaphore(1), threading.Semaphore(0)]

    def work(me, order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n, v in enumerate(order):
                    turns[me].acquire()
                    got[me, n, v] = [t.clone() for t in ops.distill_topk_fwd_bwd(*cases[v])[:3]]
                    torch.cuda.current_stream().synchronize()
                    turns[1 - me].release()
        except Exception as e:                                          # (the other thread goes on without this one)
            errors.append(e)
            for _ in order:
                turns[1 - me].release()

    # a: the longer row; b: the shorter one, its thread's first; a: the longer row again
    threads = [threading.Thread(target=work, args=a) for a in ((0, (32000, 32000, 20000)), (1, (20000, 32000, 20000)))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not errors, errors
    want = {v: ops.distill_topk_fwd_bwd(*cases[v])[:3] for v in cases}
    assert len(got) == 6
    for (_, _, v), out in got.items():
        assert all(torch.equal(a, b) for a, b in zip(out, want[v]))


def test_more_elements_than_32_bits_count(cuda):
    """70000 x 32768 f16: the last rows' results are those of a call on them alone."""
    rows, vocab, n = 70000, 32768, 9
    x = torch.empty(rows, vocab, dtype=torch.float16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    for i in range(0, rows, 10000):
        x[i:i + 10000].normal_(generator=g)
    top = ops.logits_topk(x, 16)
    assert all(torch.equal(a[-n:], b) for a, b in zip(top[:2], ops.logits_topk(x[-n:], 16)))
    # (few rows are read by more threads, whose sums have another order: the sum is held to 64 bits, at this file's tolerance)
    ref = torch.logsumexp(x[-n:].double(), 1)
    assert ((top[2][-n:].double() - ref).abs() <= 2.0 ** -23 * ref.abs() + (vocab / 256 + 24) * 2.0 ** -24 + 2.0 ** -22 * 20).all()
    top = [t.roll(1, 0) for t in top]                                   # each row against its neighbour's list
    _, loss, grad, _ = ops.distill_topk_fwd_bwd(x, *top, w_scalar=100.0)
    alone = ops.distill_topk_fwd_bwd(x[-n:], *(t[-n:] for t in top), w_scalar=100.0)
    assert torch.equal(loss[-n:], alone[1]) and torch.equal(grad[-n:], alone[2]) and alone[2].any(1).all()


def test_refusals(cuda):
    x = _logits(4, 100, torch.float16, 1)
    tv, ti, lse = ops.logits_topk(x, 10)
    for bad in (lambda: ops.logits_topk(x, 0), lambda: ops.logits_topk(x, 101), lambda: ops.logits_topk(x, 10, temperature=0.0),
                lambda: ops.logits_topk(_logits(2, 600, torch.float16, 1), 257),
                lambda: ops.distill_topk_fwd_bwd(x, tv, ti, temperature=math.nan),
                lambda: ops.distill_topk_fwd_bwd(x, tv[:, :0].contiguous(), ti[:, :0].contiguous())):
        with pytest.raises(capi.CactiB200Error):
            bad()
    for bad in (lambda: ops.logits_topk(x.t(), 5), lambda: ops.logits_topk(x.double(), 5), lambda: ops.logits_topk(x.cpu(), 5),
                lambda: ops.logits_topk(x[0], 5),
                lambda: ops.distill_topk_fwd_bwd(x, tv[:2], ti), lambda: ops.distill_topk_fwd_bwd(x, tv, ti.long()),
                lambda: ops.distill_topk_fwd_bwd(x, tv, ti, lse.half()), lambda: ops.distill_topk_fwd_bwd(x, tv, ti, w=lse[:2]),
                lambda: ops.distill_topk_fwd_bwd(x, tv, ti, beta=1), lambda: ops.distill_topk_fwd_bwd(x, tv.cpu(), ti),
                lambda: ops.distill_topk_fwd_bwd(x, tv, ti, dlogits=torch.empty(4, 100, device="cuda"))):
        with pytest.raises((ValueError, KeyError)):
            bad()
