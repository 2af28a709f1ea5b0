"""The gated feed-forward block in both directions against torch in 64 bits.

Tolerances, u = eps / 2 of the type: a product summed over n terms in f32, in whatever order, is off by at most
(n + 32) 2^-24 times the sum of the terms' sizes; silu and its derivative are evaluated in f32 with the fast exponential
(2^-20 covers them for |g| < 30) and have slopes below 1.1; one rounding to the type.  dg and du are rounded to the type before
they are multiplied: independent errors of at most u relative (u / sqrt(3) in the mean), so 7 of their standard deviations,
sqrt(sum of squared terms) u / sqrt(3), on each sum.
"""
import pytest
import torch

from cacti_b200 import capi, ops

pytestmark = pytest.mark.gpu

DT = {"float16": torch.float16, "bfloat16": torch.bfloat16}
SHAPES = [(1, 8, 8), (1, 3200, 640), (2, 64, 128), (3, 100, 72), (7, 33, 50), (8, 1, 1), (17, 256, 1000), (64, 72, 136),
          (77, 1003, 277), (129, 264, 200), (128, 512, 512), (200, 1160, 520), (300, 128, 1000), (513, 192, 264)]


def _u(dt):
    return torch.finfo(dt).eps / 2


def _inputs(t, d, f, dt, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, sc=1.0: (torch.randn(*s, device="cuda", generator=g) * sc).to(dt)
    return r(t, d), r(f, d, sc=d ** -0.5), r(f, d, sc=d ** -0.5), r(t, f)


def _at_offset(t, off):
    buf = torch.full((t.numel() + off + 64,), 7.0, dtype=t.dtype, device=t.device)
    v = buf[off:off + t.numel()].view(t.shape)
    v.copy_(t)
    return v, buf


def _within(got, ref, tol, what):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], ref[bad][:4], tol[bad][:4])


def _check_fwd(out, x, wg, wu, what=""):
    h, gate, up = out
    dt, n = x.dtype, x.shape[1]
    xd, g64, u64 = x.double(), wg.double(), wu.double()
    g, u = xd @ g64.t(), xd @ u64.t()
    eg, eu = ((n + 32) * 2.0 ** -24 * (xd.abs() @ w.abs().t()) for w in (g64, u64))
    tiny = 2.0 ** -25
    if gate is not None:
        _within(gate, g, _u(dt) * g.abs() + eg * (1 + _u(dt)) + tiny, what + " gate")
        _within(up, u, _u(dt) * u.abs() + eu * (1 + _u(dt)) + tiny, what + " up")
    sg = g * torch.sigmoid(g)
    _within(h, sg * u, (_u(dt) + 2.0 ** -20) * (sg * u).abs() + (1.1 * eg * (u.abs() + eu) + sg.abs() * eu) * (1 + _u(dt)) + tiny, what + " h")


def _check_bwd(out, dh, x, wg, wu, gate, up, old=(None, None, None), what=""):
    dt = x.dtype
    xd, wgd, wud, g, u, d = (t.double() for t in (x, wg, wu, gate, up, dh))
    s = torch.sigmoid(g)
    dg, du = d * u * s * (1 + g * (1 - s)), d * g * s
    ur = _u(dt) + 2.0 ** -20

    def tol(terms, n, ref, o):
        mag = sum(a.abs() @ b.abs() for a, b in terms)
        sq = sum((a * a) @ (b * b) for a, b in terms).sqrt()
        base = 7 * ur / 3 ** 0.5 * sq + (n + 32) * 2.0 ** -24 * mag + 2.0 ** -25
        # few terms: the errors do not average, but each is at most ur
        base = torch.maximum(base, (ur + (n + 32) * 2.0 ** -24) * mag) if n < 64 else base
        total = ref if o is None else ref + o.double()
        return total, _u(dt) * total.abs() + base * (1 + _u(dt)) + (0 if o is None else 2.0 ** -22 * o.double().abs())

    f, t = wg.shape[0], x.shape[0]
    for name, got, terms, n, o in (("dx", out[0], [(dg, wgd), (du, wud)], 2 * f, old[0]),
                                   ("dw_gate", out[1], [(dg.t(), xd)], t, old[1]), ("dw_up", out[2], [(du.t(), xd)], t, old[2])):
        ref = sum(a @ b for a, b in terms)
        total, tl = tol(terms, n, ref, o)
        _within(got, total, tl, f"{what} {name}")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,d,f", SHAPES)
def test_forward(cuda, dtype, t, d, f):
    x, wg, wu, _ = _inputs(t, d, f, DT[dtype])
    out = ops.gated_ffn_fwd(x, wg, wu, save=True)
    _check_fwd(out, x, wg, wu)
    h, gate, up = ops.gated_ffn_fwd(x, wg, wu)
    assert gate is None and up is None and torch.equal(h, out[0])
    # operands and outputs at odd addresses: same values within the same bounds, nothing around the outputs touched
    (xv, _), (gv, _), (uv, _) = _at_offset(x, 3), _at_offset(wg, 1), _at_offset(wu, 5)
    bufs = [_at_offset(torch.zeros(t, f, dtype=x.dtype, device="cuda"), o) for o in (1, 2, 3)]
    _check_fwd(ops.gated_ffn_fwd(xv, gv, uv, h=bufs[0][0], gate=bufs[1][0], up=bufs[2][0]), x, wg, wu, "views")
    for (v, b), o in zip(bufs, (1, 2, 3)):
        assert (b[:o] == 7).all() and (b[o + t * f:] == 7).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,d,f", SHAPES)
def test_backward(cuda, dtype, t, d, f):
    x, wg, wu, dh = _inputs(t, d, f, DT[dtype], 1)
    _, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    out = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    _check_bwd(out, dh, x, wg, wu, gate, up)
    again = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    assert all(torch.equal(a, b) for a, b in zip(out, again))
    # Accumulate mode and odd addresses; nothing around the outputs touched
    g = torch.Generator(device="cuda").manual_seed(5)
    old = [torch.randn(o.shape, device="cuda", generator=g).to(x.dtype) for o in out]
    (xv, _), (gv, _), (uv, _), (dv, _) = _at_offset(x, 1), _at_offset(wg, 3), _at_offset(wu, 2), _at_offset(dh, 5)
    bufs = [_at_offset(o, n) for o, n in zip(old, (1, 2, 7))]
    acc = ops.gated_ffn_bwd(dv, xv, gv, uv, gate, up, *(v for v, _ in bufs), beta_dx=1, beta_dw=1)
    _check_bwd(acc, dh, x, wg, wu, gate, up, old, "added")
    for (v, b), o, n in zip(bufs, old, (1, 2, 7)):
        assert (b[:n] == 7).all() and (b[n + o.numel():] == 7).all()
    acc = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dw_gate=old[1].clone(), dw_up=old[2].clone(), beta_dw=1)
    _check_bwd(acc, dh, x, wg, wu, gate, up, (None, old[1], old[2]), "weights added")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,d,f", [(2048, 3200, 1000), (300, 640, 8640), (16, 3200, 8640), (4, 3200, 8640), (1100, 520, 2056)])
def test_both_directions_at_larger_sizes(cuda, dtype, t, d, f):
    x, wg, wu, dh = _inputs(t, d, f, DT[dtype], 2)
    out = ops.gated_ffn_fwd(x, wg, wu, save=True)
    _check_fwd(out, x, wg, wu)
    _check_bwd(ops.gated_ffn_bwd(dh, x, wg, wu, out[1], out[2]), dh, x, wg, wu, out[1], out[2])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,d,f", [(256, 256, 128), (513, 264, 184), (2048, 2560, 2048)])
def test_everything_added_through_the_tma_epilogue(cuda, dtype, t, d, f):
    """Aligned results and a contraction of dx that is not cut: old values of all three arrive by TMA."""
    x, wg, wu, dh = _inputs(t, d, f, DT[dtype], 8)
    _, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    want = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    zeros = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, *(torch.zeros_like(o) for o in want), beta_dx=1, beta_dw=1)
    assert all(torch.equal(a, b) for a, b in zip(zeros, want))
    g = torch.Generator(device="cuda").manual_seed(9)
    old = [torch.randn(o.shape, device="cuda", generator=g).to(x.dtype) for o in want]
    acc = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, *(o.clone() for o in old), beta_dx=1, beta_dw=1)
    _check_bwd(acc, dh, x, wg, wu, gate, up, old, "added")
    only = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dx=old[0].clone(), beta_dx=1)
    assert torch.equal(only[0], acc[0]) and torch.equal(only[1], want[1]) and torch.equal(only[2], want[2])


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("t,d,f,dx_off", [(16, 3200, 8640, 0), (77, 1024, 2048, 0), (300, 640, 8640, 1)])
def test_partial_sums_and_accumulating_tiles_in_one_staging(cuda, dtype, t, d, f, dx_off):
    """Few tokens cut dx's contraction (and a dx at an odd address cannot leave by TMA): its tiles leave the staging by ordinary
    accesses, and the same warps then load old weight gradients into it by TMA.  More items than workers, so that one warp does both.
    Added to zeros the weight gradients are those of Apply mode, bit for bit; added to ones, one rounding of the f32 sum away."""
    x, wg, wu, dh = _inputs(t, d, f, DT[dtype], 6)
    _, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    want = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    for _ in range(3):
        dx, _ = _at_offset(torch.zeros_like(x), dx_off)
        zeros = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dx=dx, dw_gate=torch.zeros_like(wg), dw_up=torch.zeros_like(wu), beta_dw=1)
        assert all(torch.equal(a, b) for a, b in zip(zeros, want))
        old = (None, torch.ones_like(wg), torch.full_like(wu, -2.0))
        dx, _ = _at_offset(torch.zeros_like(x), dx_off)
        out = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dx=dx, dw_gate=old[1].clone(), dw_up=old[2].clone(), beta_dw=1)
        assert torch.equal(out[0], want[0])
        _check_bwd(out, dh, x, wg, wu, gate, up, old, "added")


def test_gradient_against_differences(cuda):
    """The backward's formulas are the forward's derivative: central differences of sum(dh * h) in 64 bits."""
    t, d, f, eps = 3, 16, 24, 1e-5
    x, wg, wu, dh = _inputs(t, d, f, torch.float16, 3)
    gate, up = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    dx, dwg, dwu = ops.gated_ffn_bwd(dh, x, wg, wu, gate.half(), up.half())

    def value(xd, g, u):
        a, b = xd @ g.t(), xd @ u.t()
        return (dh.double() * (a * torch.sigmoid(a) * b)).sum()

    args = [t_.double() for t_ in (x, wg, wu)]
    for which, grad in ((0, dx), (1, dwg), (2, dwu)):
        for i in (0, 5, 17):
            e = torch.zeros_like(args[which]).view(-1)
            e[i] = eps
            e = e.view(args[which].shape)
            hi, lo = (value(*[a + s * e if j == which else a for j, a in enumerate(args)]) for s in (1, -1))
            num = float((hi - lo) / (2 * eps))
            # gate and up are saved with 2^-11 relative error, dg and du rounded likewise; sums of at most 48 terms of size ~1
            assert abs(float(grad.view(-1)[i]) - num) <= 48 * 4 * 2.0 ** -11


def test_no_tokens(cuda):
    x, wg, wu, dh = _inputs(0, 64, 72, torch.bfloat16)
    h, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    assert h.shape == (0, 72)
    dx, dwg, dwu = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    assert dx.shape == (0, 64) and not dwg.any() and not dwu.any()
    a, b = torch.ones_like(wg), torch.ones_like(wu)
    ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dw_gate=a, dw_up=b, beta_dw=1)
    assert (a == 1).all() and (b == 1).all()


def test_values_that_overflow_or_vanish(cuda):
    """Large and small gates: silu saturates, h overflows the type like a rounded product, no NaN comes from finite inputs."""
    for dt in DT.values():
        x = torch.tensor([[1.0] * 8, [-1.0] * 8], device="cuda").to(dt)
        wg = torch.tensor([0.0, 1.0, 12.0, 100.0, 1000.0], device="cuda")[:, None].expand(5, 8).contiguous().to(dt)
        wu = torch.full((5, 8), 8.0, device="cuda").to(dt)
        h, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
        g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
        ref = (g * torch.sigmoid(g) * u).to(dt)
        assert torch.allclose(h.double(), ref.double(), rtol=4 * _u(dt), atol=1e-6)
        out = ops.gated_ffn_bwd(torch.ones_like(h), x, wg, wu, gate, up)
        assert not any(t.isnan().any() for t in out)


def test_streams_and_graphs(cuda):
    x, wg, wu, dh = _inputs(96, 264, 400, torch.float16, 4)
    out = ops.gated_ffn_fwd(x, wg, wu, save=True)
    want = out + ops.gated_ffn_bwd(dh, x, wg, wu, out[1], out[2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:                                                   # two calls at once
        with torch.cuda.stream(s):
            o = ops.gated_ffn_fwd(x, wg, wu, save=True)
            got.append(o + ops.gated_ffn_bwd(dh, x, wg, wu, o[1], o[2]))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    xs = x.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = ops.gated_ffn_fwd(xs, wg, wu, save=True)
            o = o + ops.gated_ffn_bwd(dh, xs, wg, wu, o[1], o[2])
        graphs.append((g, o))
    xs.copy_(-x)
    o = ops.gated_ffn_fwd(-x, wg, wu, save=True)
    want = o + ops.gated_ffn_bwd(dh, -x, wg, wu, o[1], o[2])
    torch.cuda.synchronize()
    for s, (g, _) in zip(streams, graphs):                              # both replayed at the same time
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for _, o in graphs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))
    err = capi.C.c_uint(0)
    assert capi.lib().cacti_b200_device_error(capi.C.byref(err)) == capi.OK and err.value == 0


def test_refusals(cuda):
    x, wg, wu, dh = _inputs(4, 16, 24, torch.float16)
    _, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    for bad in (lambda: ops.gated_ffn_fwd(x.float(), wg, wu), lambda: ops.gated_ffn_fwd(x, wg, wu.bfloat16()),
                lambda: ops.gated_ffn_fwd(x, wg[:8], wu), lambda: ops.gated_ffn_fwd(x, wg.t(), wu.t()),
                lambda: ops.gated_ffn_fwd(x.cpu(), wg, wu), lambda: ops.gated_ffn_fwd(x[:, ::2], wg[:, :8].contiguous(), wu[:, :8].contiguous()),
                lambda: ops.gated_ffn_bwd(dh, x, wg, wu, gate, up[:2]), lambda: ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, beta_dx=1),
                lambda: ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, dw_gate=torch.empty_like(wg), beta_dw=1)):
        with pytest.raises(ValueError):
            bad()
    small = torch.empty(256, dtype=torch.uint8, device="cuda")
    with pytest.raises(capi.CactiB200Error):
        ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, workspace=small)


def test_workspaces_of_another_place_or_type_are_refused(cuda):
    """A workspace in host memory has an address like any other: the wrapper has to see it before a kernel does."""
    x, wg, wu, dh = _inputs(4, 17, 24, torch.float16)
    _, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    n = 1 << 20
    for ws in (torch.empty(n, dtype=torch.uint8), torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2],
               torch.empty(n, dtype=torch.float32, device="cuda")):
        with pytest.raises(ValueError, match="workspace"):
            ops.gated_ffn_fwd(x, wg, wu, workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, workspace=ws)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    assert torch.equal(ops.gated_ffn_fwd(x, wg, wu, workspace=ws)[0], ops.gated_ffn_fwd(x, wg, wu)[0])
    for a, b in zip(ops.gated_ffn_bwd(dh, x, wg, wu, gate, up, workspace=ws), ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)):
        assert torch.equal(a, b)


def test_more_elements_than_32_bits_count(cuda):
    """270000 tokens x 8192: the last tokens' results are those of a call on them alone; the weight gradients see them."""
    t, d, f, n = 270000, 64, 8192, 300
    x, wg, wu, _ = _inputs(1, d, f, torch.float16, 10)
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(t, d, device="cuda", generator=g).half()
    h, gate, up = ops.gated_ffn_fwd(x, wg, wu, save=True)
    few = ops.gated_ffn_fwd(x[-n:], wg, wu, save=True)
    assert all(torch.equal(a[-n:], b) for a, b in zip((h, gate, up), few))
    dh = h.zero_()                                                      # only the last tokens have a gradient
    dh[-n:] = torch.randn(n, f, device="cuda", generator=g).half()
    dx, dwg, dwu = ops.gated_ffn_bwd(dh, x, wg, wu, gate, up)
    assert not dx[:-n].any()
    _check_bwd((dx[-n:], dwg, dwu), dh[-n:], x[-n:], wg, wu, few[1], few[2])
