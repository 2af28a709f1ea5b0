"""What is measured of the training operators: the teacher's top logits, the distillation loss with its gradient, and the
gated feed-forward block in both directions.  `run` computes them in plain torch operations, or, with `own` set, through
cacti_b200.ops."""
import math

import torch

own = False

F16, BF16, F32 = "float16", "bfloat16", "float32"
_SIZE = {F16: 2, BF16: 2, F32: 4}


def listed():
    return [
        # one prompt token's logits of a 32000-word teacher: a call where launch latency is what counts
        {"name": "topk 1x32000 f16", "op": "topk", "rows": 1, "vocab": 32000, "k": 32, "tau": 1.0, "dtype": F16},
        # a teacher's batch at the loss benchmark's shape: the ordinary case
        {"name": "topk 8192x32000 f16", "op": "topk", "rows": 8192, "vocab": 32000, "k": 64, "tau": 2.0, "dtype": F16},
        # f32 logits, a vocabulary that is no multiple of a vector: rows start at odd addresses
        {"name": "topk 1001x50001 f32", "op": "topk", "rows": 1001, "vocab": 50001, "k": 100, "tau": 1.0, "dtype": F32},
        # the student's loss at the loss benchmark's shape; teacher mass outside the list in one bucket; padded tokens
        {"name": "distill 8192x32000 f16 tail", "op": "distill", "rows": 8192, "vocab": 32000, "k": 64, "tau": 2.0,
         "tail": True, "ragged": False, "pad": 512, "dtype": F16, "teacher": F16},
        # a large vocabulary, bf16, the teacher's distribution renormalised over what it listed, lists of unequal length
        {"name": "distill 2048x131072 bf16", "op": "distill", "rows": 2048, "vocab": 131072, "k": 128, "tau": 1.0,
         "tail": False, "ragged": True, "pad": 0, "dtype": BF16, "teacher": F32},
        # few rows, f32, odd vocabulary
        {"name": "distill 37x50001 f32 tail", "op": "distill", "rows": 37, "vocab": 50001, "k": 17, "tau": 1.5,
         "tail": True, "ragged": True, "pad": 3, "dtype": F32, "teacher": F32},
        # a single token through the 3B shape's block: weight bandwidth and latency
        {"name": "ffn fwd 1x3200x8640 f16", "op": "ffn_fwd", "tokens": 1, "d": 3200, "f": 8640, "save": False, "dtype": F16},
        # an odd number of tokens and sizes that are multiples of 8 but of no tile
        {"name": "ffn fwd 333x1160x3080 bf16", "op": "ffn_fwd", "tokens": 333, "d": 1160, "f": 3080, "save": True, "dtype": BF16},
        # eight sequences of 2048 at the 3B shape, gate and up kept for the backward pass: the training step's forward
        {"name": "ffn fwd 16384x3200x8640 f16", "op": "ffn_fwd", "tokens": 16384, "d": 3200, "f": 8640, "save": True, "dtype": F16},
        # sizes that are no multiple of a 16-byte vector: every row starts at another alignment
        {"name": "ffn bwd 77x1003x2777 bf16", "op": "ffn_bwd", "tokens": 77, "d": 1003, "f": 2777, "dtype": BF16},
        # one sequence of 2048 at the 3B shape: the backward of one GPU of eight
        {"name": "ffn bwd 2048x3200x8640 f16", "op": "ffn_bwd", "tokens": 2048, "d": 3200, "f": 8640, "dtype": F16},
        # eight sequences of 2048: the training step's backward
        {"name": "ffn bwd 16384x3200x8640 bf16", "op": "ffn_bwd", "tokens": 16384, "d": 3200, "f": 8640, "dtype": BF16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["topk", "distill", "distill", "ffn_fwd", "ffn_bwd"])
    if op in ("topk", "distill"):
        vocab = _log_int(rng, 1000, 131072)
        if rng.random() < 0.5:
            vocab = (vocab + 7) // 8 * 8
        rows = _log_int(rng, 1, min(8192, 2048 * 131072 // vocab))
        c = {"op": op, "rows": rows, "vocab": vocab, "k": _log_int(rng, 1, 128), "tau": rng.choice([1.0, 1.5, 2.0, 4.0]),
             "dtype": rng.choice([F16, BF16, F32])}
        if op == "distill":
            c.update(tail=rng.random() < 0.5, ragged=rng.random() < 0.5, pad=rng.randint(0, rows // 8),
                     teacher=rng.choice([c["dtype"], F32]))
        return c
    d, f = _log_int(rng, 64, 4096), _log_int(rng, 128, 11008)
    if rng.random() < 0.7:
        d, f = (d + 7) // 8 * 8, (f + 7) // 8 * 8
    tokens = _log_int(rng, 1, min(16384, 16384 * 3200 * 8640 // (d * f)))
    c = {"op": op, "tokens": tokens, "d": d, "f": f, "dtype": rng.choice([F16, BF16])}
    if op == "ffn_fwd":
        c["save"] = rng.random() < 0.5
    return c


def _logits(rows, vocab, gen):
    """Rows of logits as a language model gives them: a broad bulk and a few words that stand out."""
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * 1.5
    peaks = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
    return x.scatter_add_(1, peaks, 2.0 + 6.0 * torch.rand(rows, 8, device="cuda", generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = getattr(torch, case["dtype"])
    s = dict(case)
    if case["op"] == "topk":
        s["logits"] = _logits(case["rows"], case["vocab"], gen).to(dt)
        return s
    if case["op"] == "distill":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        z = _logits(rows, vocab, gen)
        x = z + 0.7 * torch.randn(rows, vocab, device="cuda", generator=gen)
        s["logits"] = x.to(dt)
        tdt = getattr(torch, case["teacher"])
        s["t_lse"] = torch.logsumexp(z / case["tau"], 1) if case["tail"] else None
        v, i = torch.topk(z, k, dim=1)
        s["t_values"], s["t_indices"] = v.to(tdt), i.to(torch.int32)
        if case["ragged"]:
            # lists of unequal length: what follows a list's end is marked unused
            used = torch.randint(0, k + 1, (rows, 1), device="cuda", generator=gen)
            s["t_indices"].masked_fill_(torch.arange(k, device="cuda")[None] >= used, -1)
        # padded tokens have weight 0; the others share the mean, times the loss scale that f16 gradients are kept with
        scale = 65536.0 if case["dtype"] == F16 else 1.0
        w = torch.full((rows,), scale / max(rows - case["pad"], 1), device="cuda")
        w[torch.randperm(rows, device="cuda", generator=gen)[:case["pad"]]] = 0.0
        s["w"] = w
        return s
    t, d, f = case["tokens"], case["d"], case["f"]
    s["x"] = torch.randn(t, d, device="cuda", generator=gen).to(dt)
    s["w_gate"], s["w_up"] = ((torch.randn(f, d, device="cuda", generator=gen) / math.sqrt(d)).to(dt) for _ in range(2))
    if case["op"] == "ffn_bwd":
        s["gate"], s["up"] = s["x"] @ s["w_gate"].t(), s["x"] @ s["w_up"].t()
        s["dh"] = torch.randn(t, f, device="cuda", generator=gen).to(dt)
    return s


def _own(s):
    from cacti_b200 import ops
    if s["op"] == "topk":
        return ops.logits_topk(s["logits"], s["k"], temperature=s["tau"])
    if s["op"] == "distill":
        loss, rows, grad, _ = ops.distill_topk_fwd_bwd(s["logits"], s["t_values"], s["t_indices"], s["t_lse"],
                                                       temperature=s["tau"], w=s["w"])
        return loss, rows, grad
    if s["op"] == "ffn_fwd":
        h, gate, up = ops.gated_ffn_fwd(s["x"], s["w_gate"], s["w_up"], save=s["save"])
        return (h, gate, up) if s["save"] else (h,)
    return ops.gated_ffn_bwd(s["dh"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"])


def _plain_topk(s):
    x = s["logits"].float()
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    v, i = v[:, :s["k"]], i[:, :s["k"]]
    m = v[:, :1]
    lse = torch.log(torch.exp((x - m) * (1.0 / s["tau"])).sum(1)) + m[:, 0] * (1.0 / s["tau"])
    return v.to(s["logits"].dtype), i.to(torch.int32), lse


def _plain_distill(s):
    # what belongs to a row or to a listed entry is kept in 64 bits: the loss is a difference of nearly equal logarithms,
    # and the bucket's mass is what a sum near one leaves
    it = 1.0 / s["tau"]
    x = s["logits"].float()
    idx = s["t_indices"].long()
    used = idx >= 0
    z = torch.where(used, s["t_values"].double() * it, -math.inf)
    idx = idx.clamp(min=0)
    some = used.any(1)
    if s["t_lse"] is not None:
        lse_t = s["t_lse"].double()[:, None]
        r = (1.0 - torch.exp(z - lse_t).sum(1)).clamp(min=0.0) * some
    else:
        zm = z.max(1, keepdim=True).values.clamp(min=-1e30)
        lse_t = torch.log(torch.exp(z - zm).sum(1, keepdim=True).clamp(min=1e-30)) + zm
        r = torch.zeros_like(z[:, 0])
    p = torch.exp(z - lse_t)
    m = x.max(1, keepdim=True).values
    ex = torch.exp((x - m) * it)
    total = ex.sum(1, keepdim=True, dtype=torch.float64)
    top = torch.zeros_like(x).scatter_add_(1, idx, used.float())        # 1 on listed positions
    rest = torch.where(top > 0, 0.0, ex).sum(1, keepdim=True, dtype=torch.float64)
    r = torch.where((top > 0).all(1), 0.0, r)
    log_q = (torch.gather(x, 1, idx).double() - m) * it - torch.log(total)
    loss = torch.where(p > 0, p * (z - lse_t - log_q), 0.0).sum(1)
    q_rest = rest[:, 0] / total[:, 0]
    loss = loss + torch.where(r > 0, r * (torch.log(torch.where(r > 0, r, 1.0)) - torch.log(torch.where(r > 0, q_rest, 1.0))), 0.0)
    mass = (p.sum(1) + r)[:, None]
    on_top, on_rest = mass / total, mass / total - torch.where(rest > 0, r[:, None] / rest, 0.0)
    grad = ex * torch.where(top > 0, on_top.float(), on_rest.float())
    grad = grad.scatter_add_(1, idx, -p.float())
    w = s["w"][:, None]
    grad = torch.where(w != 0, grad * (w * it), 0.0)
    loss = torch.where(s["w"] != 0, loss, 0.0)
    return (s["w"] * loss).sum().float().reshape(1), loss.float(), grad.to(s["logits"].dtype)


def _plain_ffn_fwd(s):
    x = s["x"].float()
    g, u = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
    h = g / (1.0 + torch.exp(-g)) * u
    dt = s["x"].dtype
    return (h.to(dt), g.to(dt), u.to(dt)) if s["save"] else (h.to(dt),)


def _plain_ffn_bwd(s):
    x, wg, wu, g, u, dh = (s[n].float() for n in ("x", "w_gate", "w_up", "gate", "up", "dh"))
    sg = 1.0 / (1.0 + torch.exp(-g))
    dg, du = dh * u * (sg * (1.0 + g * (1.0 - sg))), dh * (g * sg)
    dt = s["x"].dtype
    return (dg @ wg + du @ wu).to(dt), (dg.t() @ x).to(dt), (du.t() @ x).to(dt)


def run(state):
    if own:
        return _own(state)
    return {"topk": _plain_topk, "distill": _plain_distill, "ffn_fwd": _plain_ffn_fwd, "ffn_bwd": _plain_ffn_bwd}[state["op"]](state)


def work(case):
    if case["op"] == "topk":
        n, e = case["rows"] * case["vocab"], _SIZE[case["dtype"]]
        return {"bytes": n * e + case["rows"] * (case["k"] * (e + 4) + 4), "flops": 4 * n}
    if case["op"] == "distill":
        n, e = case["vocab"], _SIZE[case["dtype"]]
        live = case["rows"] - case["pad"]
        return {"bytes": (live + case["rows"]) * n * e + live * case["k"] * (_SIZE[case["teacher"]] + 4) +
                case["rows"] * (12 if case["tail"] else 8), "flops": 8 * live * n}
    t, d, f = case["tokens"], case["d"], case["f"]
    if case["op"] == "ffn_fwd":
        return {"bytes": 2 * (t * d + 2 * f * d + (3 if case["save"] else 1) * t * f), "flops": 4 * t * d * f}
    return {"bytes": 2 * (3 * t * f + 2 * t * d + 4 * f * d), "flops": 8 * t * d * f}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "topk":
        # a value's place is the number of entries before it in the order (value downwards, index upwards)
        x = s["logits"].double()
        order = torch.argsort(-x, dim=1, stable=True)[:, :case["k"]]
        return torch.gather(x, 1, order), order.to(torch.int32), torch.logsumexp(x / case["tau"], 1)
    if case["op"] == "distill":
        return _exact_distill(s)
    x, wg, wu = s["x"].double(), s["w_gate"].double(), s["w_up"].double()
    if case["op"] == "ffn_fwd":
        g, u = x @ wg.t(), x @ wu.t()
        h = g * torch.sigmoid(g) * u
        return (h, g, u) if case["save"] else (h,)
    g, u, dh = s["gate"].double(), s["up"].double(), s["dh"].double()
    sg = torch.sigmoid(g)
    dg, du = dh * u * (sg + g * sg * (1 - sg)), dh * g * sg
    return torch.addmm(du @ wu, dg, wg), dg.t() @ x, du.t() @ x


def _exact_distill(s):
    """Row blocks, from log-probabilities: the unlisted positions' log of their sum directly, never as a difference."""
    rows = s["rows"]
    loss, grad = torch.zeros(rows, dtype=torch.float64, device="cuda"), []
    step = max(1, 2 ** 25 // s["vocab"])
    for a in range(0, rows, step):
        b = min(rows, a + step)
        x = s["logits"][a:b].double() / s["tau"]
        idx, w = s["t_indices"][a:b].long(), s["w"][a:b].double()
        used = idx >= 0
        z = s["t_values"][a:b].double() / s["tau"]
        z = torch.where(used, z, torch.full_like(z, -math.inf))
        if s["t_lse"] is not None:
            logp = z - s["t_lse"][a:b, None].double()
        else:
            logp = z - torch.logsumexp(z, 1, keepdim=True)
        logp = torch.where(used, logp, torch.full_like(logp, -math.inf))
        p = torch.exp(logp)
        logq = torch.log_softmax(x, 1)
        j = torch.where(used, idx, s["vocab"])                               # unused slots go to a column behind the last
        unlisted = torch.ones(b - a, s["vocab"] + 1, dtype=torch.bool, device="cuda").scatter_(1, j, False)[:, :-1]
        log_rest = torch.logsumexp(torch.where(unlisted, logq, torch.full_like(logq, -math.inf)), 1)
        r = (1 - p.sum(1)).clamp(min=0) if s["t_lse"] is not None else torch.zeros(b - a, dtype=torch.float64, device="cuda")
        r = r * used.any(1) * unlisted.any(1)
        lk = torch.where(p > 0, p * (logp - torch.gather(logq, 1, idx.clamp(min=0))), torch.zeros_like(p)).sum(1)
        lk = lk + torch.where(r > 0, torch.xlogy(r, r) - r * log_rest, torch.zeros_like(r))
        g = torch.exp(logq) * (p.sum(1) + r)[:, None]
        g = g - unlisted * r[:, None] * torch.exp(logq - log_rest[:, None])
        full = torch.cat([g, torch.zeros(b - a, 1, dtype=torch.float64, device="cuda")], 1).scatter_add_(1, j, -p)
        live = w != 0
        loss[a:b] = torch.where(live, lk, torch.zeros_like(lk))
        grad.append(torch.where(live[:, None], full[:, :-1] * (w / s["tau"])[:, None], torch.zeros_like(g)))
    return (s["w"].double() * loss).sum().reshape(1), loss, torch.cat(grad)
