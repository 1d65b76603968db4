"""The two ends of a training step on the rule weights, as timed cases.

* ``logprob``: log probabilities of given channels (or tails) in rows of logits, with each row's
  entropy and its top alternatives; ``train`` adds the gradient of the logits.
* ``adamw``: one AdamW step over many tensors at once, moments held in 32 or in 8 bits.

``own`` chooses between the plain form (elementary torch operations) and the framework's calls.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256  # moments in 8 bits: values that share a scale; every tensor starts on a new block
LARGEST = 64 * 4594485  # logits of the largest case


def listed():
    lp = dict(op="logprob", tau=1.0, masked=False, train=False, targets=1)
    aw = dict(op="adamw", rules=0, tensors=0, numel=0, shape_seed=0, step=100, weight_decay=0.01)
    return [
        # the rules of one query on the 12-relation graph, read out: 3 hops x 3 rules over 25 channels
        dict(lp, name="lp one query", rows=9, width=25, topk=3, dtype="f32"),
        # a training batch on the 51-relation graph: 256 queries x 3 hops x 3 rules over 103 channels
        dict(lp, name="lp rules train", rows=2304, width=103, topk=5, dtype="f32", train=True),
        # a training batch on the 822-relation graph: 256 queries x 2 hops x 4 rules
        dict(lp, name="lp wide rules train", rows=2048, width=1645, topk=8, dtype="f32", train=True, tau=0.7),
        # the 14,824-relation graph, 128 queries: four given channels a row, some channels shut, no alternatives
        dict(lp, name="lp web rules train", rows=1024, width=29649, topk=0, dtype="bf16", train=True, targets=4, masked=True),
        # answers among the 17,050 entities, known ones masked out
        dict(lp, name="lp entities", rows=256, width=17050, topk=10, dtype="f32", targets=8, masked=True),
        # one served query against all 4,594,485 entities
        dict(lp, name="lp one row", rows=1, width=4594485, topk=20, dtype="f16"),
        # a training batch against all 4,594,485 entities
        dict(lp, name="lp all entities train", rows=64, width=4594485, topk=8, dtype="f32", train=True),
        # the rule producer's parameters, 3 rules of size 64 and 103 channels: 27 small tensors
        dict(aw, name="aw producer", rules=3, hidden=64, channels=103, bits=32, dtype="f32", grad="f32"),
        # 16 rules and 1,645 channels: 131 tensors, moments in 8 bits
        dict(aw, name="aw wide producer 8 bit", rules=16, hidden=64, channels=1645, bits=8, dtype="f32", grad="f32"),
        # one score for each of the 20,624,575 facts
        dict(aw, name="aw facts", tensors=1, numel=20624575, bits=32, dtype="f32", grad="f32"),
        # the same held in 16 bits, with moments in 8
        dict(aw, name="aw facts 8 bit", tensors=1, numel=20624575, bits=8, dtype="bf16", grad="bf16"),
        # 150 tensors of odd sizes, 16-bit weights with 32-bit gradients
        dict(aw, name="aw ragged", tensors=150, numel=60000000, shape_seed=3, bits=32, dtype="bf16", grad="f32"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.5:
        width = _log_uniform(rng, 2, 4594485)
        rows = _log_uniform(rng, 1, max(1, min(65536, LARGEST // width)))
        return dict(op="logprob", rows=rows, width=width, targets=rng.choice((1, 1, 2, 3, 7, 16)),
                    topk=rng.choice((0, 1, 5, 8, 13, 20, 32)), dtype=rng.choice(sorted(DTYPES)),
                    masked=rng.random() < 0.4, train=rng.random() < 0.5, tau=rng.choice((0.5, 1.0, 1.3)))
    dtype = rng.choice(sorted(DTYPES))
    numel = _log_uniform(rng, 100, 60000000)
    return dict(op="adamw", rules=0, tensors=min(_log_uniform(rng, 1, 300), numel), numel=numel,
                shape_seed=rng.randrange(1 << 20), bits=rng.choice((8, 32)), dtype=dtype,
                grad=rng.choice((dtype, "f32")), step=rng.choice((0, 1, 10, 5000)),
                weight_decay=rng.choice((0.0, 0.01, 0.1)))


def _shapes(case):
    """The tensors' shapes: the producer's parameters, or `tensors` odd ones that hold `numel` values."""
    if case["rules"]:
        h, n = case["hidden"], case["channels"]
        lstm = [(4 * h, h), (4 * h, h), (4 * h,), (4 * h,)] * 2
        return [(n, h)] + lstm * case["rules"] + [(n, 2 * h), (n,)]
    k, total = case["tensors"], case["numel"]
    share = np.random.default_rng(case["shape_seed"]).exponential(1.0, k) ** 2 if k > 1 else np.ones(1)
    sizes = np.maximum(1, np.floor(share / share.sum() * (total - k)).astype(np.int64))
    sizes[-1] += max(0, total - int(sizes.sum()))
    return [(int(s),) for s in sizes]


def _spans(case):
    """(offset, shape, numel) of each tensor in the flat buffers, and the buffers' length."""
    out, at = [], 0
    for shape in _shapes(case):
        n = math.prod(shape)
        out.append((at, shape, n))
        at += -(-n // BLOCK) * BLOCK
    return out, at


LR, BETA1, BETA2, EPS = 1e-3, 0.9, 0.999, 1e-8


def _inputs(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "logprob":
        rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        s = {"case": case, "logits": normal(rows, width).mul_(3.0).to(dtype), "mask": None}
        s["targets"] = torch.randint(0, width, (rows, case["targets"]), generator=gen, device=dev)
        if case["targets"] > 1:
            s["targets"][::3, -1] = -1  # rows with fewer given ones are padded
        if case["masked"]:
            s["mask"] = torch.rand((rows, width), generator=gen, device=dev) < 0.9
            if rows > 3:
                s["mask"][1] = False  # a row that is left with nothing
        if case["train"]:
            s["grads"] = [normal(rows, case["targets"]), normal(rows).mul_(0.1), normal(rows, case["topk"]).mul_(0.1)]
        return s
    spans, total = _spans(case)
    s = {"case": case, "step": case["step"], "param": torch.zeros(total, device=dev, dtype=DTYPES[case["dtype"]]),
         "grad": torch.zeros(total, device=dev, dtype=DTYPES[case["grad"]]), "m": torch.zeros(total, device=dev),
         "v": torch.zeros(total, device=dev)}
    inside = torch.zeros(total, dtype=torch.bool, device=dev)
    for at, _, n in spans:
        inside[at:at + n] = True
    size = torch.exp(normal(total // BLOCK).mul_(2.0)).repeat_interleave(BLOCK).mul_(1e-3)  # gradients differ from layer to layer
    s["param"].copy_(normal(total).mul_(0.1) * inside)
    s["grad"].copy_(normal(total).mul_(size) * inside * (torch.rand(total, generator=gen, device=dev) < 0.9))
    if case["step"]:
        s["m"].copy_(normal(total).mul_(size).mul_(0.3) * inside)
        s["v"].copy_(normal(total).square_().add_(0.1).mul_(size.square_()).mul_(0.5) * inside)
        if case["bits"] == 8:
            s["m"], s["v"] = _held_m(s["m"].double()).float(), _held_v(s["v"].double()).float()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["op"] == "adamw":  # the optimizer that a training program keeps
        from minikg_dev_b200 import optim
        spans, _ = _spans(case)
        params = [torch.nn.Parameter(s["param"][at:at + n].view(shape)) for at, shape, n in spans]
        opt = optim.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=case["weight_decay"],
                          state_bits=case["bits"])
        if case["step"]:
            opt.load_state_dict({"param_groups": opt.state_dict()["param_groups"], "state": {
                i: {"step": case["step"], "exp_avg": s["m"][at:at + n].view(shape),
                    "exp_avg_sq": s["v"][at:at + n].view(shape)} for i, (at, shape, n) in enumerate(spans)}})
        for p, (at, shape, n) in zip(params, spans):
            p.grad = s["grad"][at:at + n].view(shape)
        s["opt"] = opt
        s["m"] = s["v"] = None
    return s


def run(state):
    if state["case"]["op"] == "logprob":
        return _logprob_own(state) if own else _logprob_plain(state)
    return _adamw_own(state) if own else _adamw_plain(state)


def _logprob_own(s):
    from minikg_dev_b200 import logprobs
    c = s["case"]
    logits = s["logits"].detach().requires_grad_(c["train"])
    out = logprobs.target_logprobs(logits, s["targets"], tau=c["tau"], mask=s["mask"], topk=c["topk"])
    got = {"logprobs": out.logprobs, "entropy": out.entropy, "top_ids": out.top_ids, "top_logprobs": out.top_logprobs}
    if c["train"]:
        got["grad"], = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], logits, s["grads"])
        got = {k: v.detach() for k, v in got.items()}
    return got


def _adamw_own(s):
    s["opt"].step()
    m, v = s["opt"].moments()
    return {"param": s["param"], "exp_avg": m, "exp_avg_sq": v}


# ------------------------------------------------------------------ the plain forms
def _top(x, k):
    """The k largest of each row, ties to the lowest index; -1 where a row has no more candidates."""
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()
    order = order * (1 << 32) + ((1 << 32) - 1 - torch.arange(x.shape[1], device=x.device))
    ids = torch.topk(order, min(k, x.shape[1]), dim=1).indices
    ids = torch.where(torch.gather(x, 1, ids) == -math.inf, -1, ids)
    return torch.nn.functional.pad(ids, (0, k - ids.shape[1]), value=-1)


def _logprob_plain(s):
    c, tau = s["case"], s["case"]["tau"]
    raw = s["logits"].float()
    if s["mask"] is not None:
        raw = torch.where(s["mask"], raw, -math.inf)
    top_ids = _top(raw, c["topk"])
    x = raw / tau
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    y = x - m
    e = torch.exp(y)
    total = e.sum(1, keepdim=True)
    ey = e * torch.where(e > 0, y, 0.0)
    log_total = torch.log(total)
    entropy = torch.where(total > 0, log_total - ey.sum(1, keepdim=True) / total, 0.0)

    def of(ids):
        at = torch.gather(y, 1, ids.clamp_min(0)) - torch.where(total > 0, log_total, 0.0)
        return at

    lp = torch.where(s["targets"] < 0, 0.0, of(s["targets"]))
    top_lp = torch.where(top_ids < 0, -math.inf, of(top_ids))
    got = {"logprobs": lp, "entropy": entropy[:, 0], "top_ids": top_ids, "top_logprobs": top_lp}
    if c["train"]:
        g_lp, g_h, g_top = s["grads"]
        ids = torch.cat([s["targets"], top_ids], 1)
        g = torch.where(ids < 0, 0.0, torch.cat([g_lp, g_top], 1))
        p = e / torch.where(total > 0, total, 1.0)
        logp = torch.where(e > 0, y - log_total, 0.0)
        grad = -p * (g.sum(1, keepdim=True) + g_h[:, None] * (logp + entropy))
        grad.scatter_add_(1, ids.clamp_min(0), g)
        grad = grad / tau
        if s["mask"] is not None:
            grad = torch.where(s["mask"], grad, 0.0)
        got["grad"] = grad.to(s["logits"].dtype)
    return got


def _pow2(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def _scale(most, top, low):
    """The smallest power of two with most <= top * it, 2**low at least."""
    mant, e = torch.frexp(most / top)
    return _pow2(torch.where(mant == 0.5, e - 1, e).clamp_min(low))


def _held_m(m):
    """What is held of first moments in 8 bits (sign, 4 exponent bits, 3 of mantissa, a power of two for each block)."""
    x = m.view(-1, BLOCK)
    s = _scale(x.abs().amax(1, keepdim=True), 448.0, -120)
    y = x / s
    step = _pow2((torch.frexp(y)[1] - 1).clamp_min(-6) - 3)
    return (torch.round(y / step) * step * s).view(-1)


def _held_v(v):
    """What is held of second moments in 8 bits (5 exponent bits, 3 of mantissa, a power of two for each block); none becomes zero."""
    x = v.view(-1, BLOCK)
    s = _scale(x.amax(1, keepdim=True), 1.75, -90)
    y = x / s
    step = _pow2((torch.frexp(y)[1] - 1).clamp_min(-30) - 3)
    q = torch.round(y / step) * step
    return (torch.where(y > 0, q.clamp_min(2.0 ** -33), q) * s).view(-1)


def _adamw_plain(s):
    c = s["case"]
    s["step"] += 1
    t = s["step"]
    g = s["grad"].double() if c["bits"] == 8 else s["grad"].float()
    m = s["m"].to(g.dtype) * BETA1 + g * (1 - BETA1)
    v = s["v"].to(g.dtype) * BETA2 + g * g * (1 - BETA2)
    p = s["param"].to(g.dtype) * (1 - LR * c["weight_decay"])
    p = p - (LR / (1 - BETA1 ** t)) * m / (v.sqrt() / math.sqrt(1 - BETA2 ** t) + EPS)
    s["param"].copy_(p)
    s["m"].copy_(_held_m(m) if c["bits"] == 8 else m)
    s["v"].copy_(_held_v(v) if c["bits"] == 8 else v)
    return {"param": s["param"], "exp_avg": s["m"], "exp_avg_sq": s["v"]}


# ------------------------------------------------------------------ the work, and the definitions in 64 bits
def work(case):
    if case["op"] == "logprob":
        n, w, size = case["rows"], case["rows"] * case["width"], BYTES[case["dtype"]]
        k, t = case["topk"], case["targets"]
        moved = w * (size + case["masked"]) + n * (t * 12 + 4 + k * 12)
        if case["train"]:
            moved += w * size + n * (t + 1 + k) * 4
        return {"bytes": moved, "flops": w * (12 if case["train"] else 6)}
    numel = sum(n for _, _, n in _spans(case)[0])
    held = 8 if case["bits"] == 32 else 2 + 2 * 4 / BLOCK
    told = 0 if case["bits"] == 32 else 8  # moments in 8 bits come back as the values they stand for
    return {"bytes": numel * (2 * BYTES[case["dtype"]] + BYTES[case["grad"]] + 2 * held + told), "flops": numel * 16}


def exact(case, seed):
    s = _inputs(case, seed)
    return _logprob_exact(s) if case["op"] == "logprob" else _adamw_exact(s)


def _logprob_exact(s):
    c = s["case"]
    rows, width = s["logits"].shape
    parts, chunk = [], max(1, (1 << 25) // width)
    for a in range(0, rows, chunk):
        b = min(rows, a + chunk)
        z = s["logits"][a:b].double() / c["tau"]
        allowed = torch.ones_like(z, dtype=torch.bool) if s["mask"] is None else s["mask"][a:b]
        z = z.masked_fill(~allowed, -math.inf)
        lse = torch.logsumexp(z, 1, keepdim=True)
        none = lse == -math.inf
        logp = torch.where(none, -math.inf, z - lse)
        p = torch.exp(logp)
        h = torch.special.entr(p).sum(1)
        t = s["targets"][a:b]
        lp = torch.where(t < 0, 0.0, logp.gather(1, t.clamp_min(0)))
        # the alternatives by the logits themselves: a stable sort keeps the lowest index first
        order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :c["topk"]] if c["topk"] else t[:, :0]
        top = logp.gather(1, order)
        pad = (0, c["topk"] - top.shape[1])
        order = torch.nn.functional.pad(torch.where(top == -math.inf, -1, order), pad, value=-1)
        top = torch.nn.functional.pad(top, pad, value=-math.inf)
        out = {"logprobs": lp, "entropy": h, "top_logprobs": top}
        if c["train"]:
            g_lp, g_h, g_top = (x[a:b].double() for x in s["grads"])
            up = torch.zeros_like(z)  # the gradient that arrives at log p
            for ids, g in ((t, g_lp), (order, g_top)):
                up.scatter_add_(1, ids.clamp_min(0), torch.where(ids < 0, 0.0, g))
            up_all = up.sum(1, keepdim=True)
            through_h = -p * (torch.where(p > 0, logp, 0.0) + h[:, None]) * g_h[:, None]
            out["grad"] = torch.where(allowed, (up - p * up_all + through_h) / c["tau"], 0.0)
        parts.append(out)
    out = {k: torch.cat([x[k] for x in parts]) for k in parts[0]}
    return dict(out, top_ids=None)


def _near(table, y):
    """The nearest value of an ascending table, ties to the even place."""
    hi = torch.searchsorted(table, y).clamp_max(len(table) - 1)
    lo = (hi - 1).clamp_min(0)
    up, down = table[hi] - y, y - table[lo]
    take = (up < down) | ((up == down) & (hi % 2 == 0)) | (y >= table[hi])
    return torch.where(take, table[hi], table[lo])


def _adamw_exact(s):
    c, t = s["case"], s["case"]["step"] + 1
    dev = s["grad"].device
    g, m, v, p = (s[k].double() for k in ("grad", "m", "v", "param"))
    # in the definition's own order: 8-bit moments and 16-bit gradients often sum to the middle of two held values
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g.square()
    m_hat, v_hat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = p - LR * (c["weight_decay"] * p + m_hat / (v_hat.sqrt() + EPS))
    if c["bits"] == 8:
        codes = torch.arange(127, device=dev).double()  # 0..126: the non-negative values of the sign-4-3 form
        e4 = torch.where(codes < 8, codes / 8 * 2.0 ** -6, (1 + codes % 8 / 8) * 2.0 ** (codes // 8 - 7))
        codes = torch.arange(255, device=dev).double()
        e5 = torch.where(codes < 8, codes / 8 * 2.0 ** -30, (1 + codes % 8 / 8) * 2.0 ** (codes // 8 - 31))

        def held(x, table, low):
            x = x.view(-1, BLOCK)
            most = x.abs().amax(1, keepdim=True)
            scale = torch.exp2(torch.ceil(torch.log2(most / table[-1])).clamp_min(low))
            return x.sign(), (x.abs() / scale).clamp_max(table[-1]), scale

        sign, y, scale = held(m, e4, -120)
        m = (sign * _near(e4, y) * scale).view(-1)
        sign, y, scale = held(v, e5, -90)
        v = (torch.where(y > 0, _near(e5, y).clamp_min(e5[1]), 0.0) * scale).view(-1)
    return {"param": p, "exp_avg": m, "exp_avg_sq": v}
