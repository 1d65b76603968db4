"""optim.AdamW against its definition in float64, what 8 bits hold against a table of the held values,
the bookkeeping around a step, and its refusals.

Tolerances, from the arithmetic, with u = 2^-24 (fp32 rounds by u relative):
* m = fma(b1, m, a1 g): b1, a1 and the product are rounded, then the sum: 3 u (|b1 m| + |a1 g|);
  v likewise with one more product: 5 u v (all terms positive);
* the update s m / (sqrt(v) r + eps): s, r, the root, the fma, the division and the product: 8 u on
  top of what m and v carry (m's 3 u is of |b1 m| + |a1 g|), then the sum with p (1 - lr wd): 2 u |p|
  and the rounding to the parameter's type, half a step: eps / 2.
Moments in 8 bits are sums in fp64 rounded once: they have to be the nearest held value exactly.
"""
from __future__ import annotations

import copy
import math

import pytest
import torch

from minikg_dev_b200 import _native as N
from minikg_dev_b200.optim import AdamW

gpu = pytest.mark.gpu
U = 2.0 ** -24
BLOCK = 256
DTYPES = (torch.float32, torch.bfloat16, torch.float16)


# ------------------------------------------------------------------ what 8 bits hold, by table
def first_table():
    c = torch.arange(127, dtype=torch.float64)
    return torch.where(c < 8, c * 2.0 ** -9, (1 + c % 8 / 8) * 2.0 ** (torch.div(c, 8, rounding_mode="floor") - 7))


def second_table():
    c = torch.arange(255, dtype=torch.float64)
    return torch.where(c < 8, c * 2.0 ** -33, (1 + c % 8 / 8) * 2.0 ** (torch.div(c, 8, rounding_mode="floor") - 31))


def nearest(table, y):
    """Codes of the nearest table values to y >= 0 (largest at most), ties to the even code."""
    hi = torch.searchsorted(table, y).clamp_max(len(table) - 1)
    lo = (hi - 1).clamp_min(0)
    up, down = table[hi] - y, y - table[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def hold(x, table, low):
    """(values, codes, scales) that 8 bits hold of one tensor's x >= 0, block by block."""
    n = x.numel()
    pad = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64)
    pad[:n] = x.reshape(-1).cpu()
    b = pad.view(-1, BLOCK)
    scales = []
    for a in b.amax(1).tolist():
        e = low
        while a > float(table[-1]) * 2.0 ** e:
            e += 1
        scales.append(2.0 ** e)
    s = torch.tensor(scales, dtype=torch.float64)[:, None]
    codes = nearest(table, b / s)
    return (table[codes] * s).view(-1)[:n], codes.view(-1)[:n], s[:, 0]


def held(m, v):
    mm, _, _ = hold(m.abs(), first_table(), -120)
    vv, codes, s = hold(v, second_table(), -90)
    least = second_table()[1] * s.repeat_interleave(BLOCK)[:vv.numel()]
    vv = torch.where((codes == 0) & (v.reshape(-1).cpu() > 0), least, vv)
    return (torch.sign(m.reshape(-1).cpu()) * mm).view(m.shape), vv.view(v.shape)


def definition(p, g, m, v, t, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, wd=0.01):
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    b1, b2 = betas
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    step = lr / (1 - b1 ** t)
    below = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    return p * (1 - lr * wd) - step * m / below, m, v, (size, step / below)


def close(got, want, tol, what):
    off = (got.double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"{what}: {float((off / tol.clamp_min(1e-300)).max())} times the tolerance"


def make(sizes, dtype, grad_dtype, seed=0, shift=0):
    """Parameters (views `shift` elements into their storage) with gradients."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for n in sizes:
        n = n if isinstance(n, tuple) else (n,)
        k = math.prod(n)
        flat = torch.randn(k + shift, generator=gen, device="cuda").to(dtype)
        p = torch.nn.Parameter(flat[shift:].view(n))
        size = 10.0 ** float(torch.rand((), generator=gen, device="cuda") * 6 - 5)
        g = (torch.randn(k + shift, generator=gen, device="cuda") * size)
        g[torch.rand(k + shift, generator=gen, device="cuda") < 0.1] = 0
        g = g.to(grad_dtype)[shift:].view(n)
        p.grad = g if grad_dtype == dtype else None
        out.append((p, g))
    return out


def set_grads(pairs):
    """Gradients of another type than the parameter's, as a program that accumulates in fp32 has them."""
    for p, g in pairs:
        if p.grad is None:
            if hasattr(p, "grad_dtype"):
                p.grad_dtype = g.dtype
            p.grad = g


SIZES = (1, 3, 4, 255, 256, 257, 2047, 2048, 2049, (33, 65), 10000, (1, 1), 0)


@gpu
@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("shift", (0, 1, 2))
@pytest.mark.parametrize("dtype, grad_dtype", [(a, b) for a in DTYPES for b in (a, torch.float32)][1:])
def test_steps(dtype, grad_dtype, shift, bits):
    pairs = make(SIZES, dtype, grad_dtype, seed=shift, shift=shift)
    set_grads(pairs)
    params = [p for p, _ in pairs]
    opt = AdamW(params, lr=1e-2, weight_decay=0.1, state_bits=bits)
    sizes = [p.numel() for p in params]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + -(-n // BLOCK) * BLOCK)
    for t in (1, 2, 3):
        before = [p.detach().clone() for p in params]
        fm, fv = (x.clone() for x in opt.moments())
        opt.step()
        gm, gv = opt.moments()
        for i, (p, g) in enumerate(pairs):
            n, at = sizes[i], starts[i]
            m0, v0 = fm[at:at + n].view(p.shape), fv[at:at + n].view(p.shape)
            want, m, v, (size, rate) = definition(before[i], g, m0, v0, t, lr=1e-2, wd=0.1)
            m_tol, v_tol = 3 * U * size + 1e-45, 5 * U * v + 1e-45
            eps = torch.finfo(dtype).eps
            tiny = torch.finfo(dtype).smallest_normal * eps  # a subnormal's step
            tol = rate * (3 * U * size + 8 * U * (m.abs() + size)) + 4 * U * want.abs() + 4 * U * before[i].double().cpu().abs()
            # v's share: its root is off by half its relative error (and by what an fp32 subnormal v loses)
            tol += rate * m.abs() * 3 * U
            close(p, want, tol + eps / 2 * (want.abs() + tol) + tiny, f"step {t} parameter {i}")
            if bits == 32:
                close(gm[at:at + n].view(p.shape), m, m_tol, f"step {t} m {i}")
                close(gv[at:at + n].view(p.shape), v, v_tol, f"step {t} v {i}")
            elif n:
                hm, hv = held(m, v)
                assert torch.equal(gm[at:at + n].view(p.shape).double().cpu(), hm), f"step {t} held m {i}"
                assert torch.equal(gv[at:at + n].view(p.shape).double().cpu(), hv), f"step {t} held v {i}"
            # what is left of the last block stays 0
            assert not gm[at + n:starts[i + 1]].any() and not gv[at + n:starts[i + 1]].any()
            assert int(opt.state[p]["step"]) == (t if n else 0)


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_many_tensors_take_several_launches(bits):
    sizes = [1 + (i * 37) % 301 for i in range(1700)]
    pairs = make(sizes, torch.float32, torch.float32, seed=4)
    before = [p.detach().clone() for p, _ in pairs]
    opt = AdamW([p for p, _ in pairs], state_bits=bits)
    opt.step()
    for i in range(0, 1700, 7):
        p, g = pairs[i]
        zero = torch.zeros_like(g)
        want, m, v, (size, rate) = definition(before[i], g, zero, zero, 1)
        close(p, want, 16 * U * (rate * size + want.abs() + before[i].double().cpu().abs()), f"tensor {i}")
        assert int(opt.state[p]["step"]) == 1
    assert int(opt._buffers["ticket"]) == 0


@gpu
def test_against_torch():
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(37, 51), torch.nn.LSTM(51, 16, bidirectional=True)).cuda()
    twin = copy.deepcopy(model)
    a = AdamW(model.parameters(), lr=3e-3, weight_decay=0.05)
    b = torch.optim.AdamW(twin.parameters(), lr=3e-3, weight_decay=0.05)
    sched = [torch.optim.lr_scheduler.ExponentialLR(o, 0.9) for o in (a, b)]
    for i in range(20):
        x = torch.randn(5, 37, device="cuda")
        for net, opt, s in ((model, a, sched[0]), (twin, b, sched[1])):
            opt.zero_grad()
            net[1](net[0](x))[0].square().sum().backward()
            if net is twin:  # the same gradients for both: only the update is compared
                for p, q in zip(model.parameters(), twin.parameters()):
                    q.grad.copy_(keep[p])
            else:
                keep = {p: p.grad.clone() for p in model.parameters()}
            opt.step()
            s.step()
    for p, q in zip(model.parameters(), twin.parameters()):
        # 20 steps of at most lr each, 16 u off a step, and the parameter's own roundings
        assert float((p - q).abs().max()) <= 20 * (16 * U * 3e-3 * 4 + 2 * U * float(q.abs().max()))


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_groups_missing_gradients_and_rates(bits):
    pairs = make((300, 40, 500, 7), torch.float32, torch.float32)
    (p0, g0), (p1, _), (p2, g2), (p3, g3) = pairs
    p1.grad = None
    opt = AdamW([{"params": [p0, p1]}, {"params": [p2], "lr": 0.5, "betas": (0.5, 0.6), "weight_decay": 0.0}],
                lr=0.1, eps=1e-3, state_bits=bits)
    opt.step()
    opt.add_param_group({"params": [p3], "lr": 0.25})
    before = [p.detach().clone() for p, _ in pairs]
    m0, v0 = (x.clone() for x in opt.moments())
    opt.step()
    assert torch.equal(p1, before[1]) and [int(opt.state[p]["step"]) for p, _ in pairs] == [2, 0, 2, 1]
    for i, p, g, at, t, kw in ((0, p0, g0, 0, 2, dict(lr=0.1)), (2, p2, g2, 768, 2, dict(lr=0.5, betas=(0.5, 0.6), wd=0.0)),
                               (3, p3, g3, 1280, 1, dict(lr=0.25))):
        want, *_, (size, rate) = definition(before[i], g, m0[at:at + p.numel()], v0[at:at + p.numel()], t, eps=1e-3, **kw)
        close(p, want, 16 * U * (rate * size + want.abs() + before[i].double().cpu().abs()), f"parameter {i}")


@gpu
def test_mixed_types_in_one_group():
    pairs = make((100, 300), torch.float32, torch.float32) + make((200, 50), torch.bfloat16, torch.bfloat16)
    opt = AdamW([p for p, _ in pairs])
    before = [p.detach().clone() for p, _ in pairs]
    opt.step()
    for (p, g), b in zip(pairs, before):
        zero = torch.zeros_like(g)
        want, *_ = definition(b, g, zero, zero, 1)
        close(p, want, (torch.finfo(p.dtype).eps / 2 + 32 * U) * (want.abs() + 2e-3), str(p.dtype))


@gpu
def test_gradients_of_other_layouts_and_shared_ones():
    p = torch.nn.Parameter(torch.randn(30, 50, device="cuda"))
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn(50, 30, device="cuda")
    p.grad, q.grad = g.t(), g.t().contiguous()
    AdamW([p]).step()
    AdamW([q]).step()
    assert torch.equal(p, q)
    a, b = (torch.nn.Parameter(torch.ones(5, device="cuda")) for _ in range(2))
    a.grad = b.grad = torch.arange(5.0, device="cuda")
    AdamW([a, b]).step()
    assert torch.equal(a, b)


@gpu
def test_not_finite_gradients():
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(600, device="cuda"))
        p.grad = torch.full((600,), 0.5, device="cuda")
        p.grad[3], p.grad[300] = math.nan, math.inf
        opt = AdamW([p], state_bits=bits)
        opt.step()
        bad = torch.zeros(600, dtype=torch.bool, device="cuda")
        bad[3] = bad[300] = True
        assert torch.equal(torch.isnan(p), bad)
        m, v = opt.moments()
        assert not torch.isfinite(m[:600])[bad].any() and not torch.isfinite(v[:600])[bad].any()
        assert torch.isfinite(m[:600])[~bad].all() and torch.isfinite(v[:600])[~bad].all()


@gpu
def test_extremes_in_8_bits():
    """Second moments down to the smallest stay above 0; those too large to square stay finite."""
    p = torch.nn.Parameter(torch.zeros(1024, device="cuda"))
    g = torch.zeros(1024, device="cuda")
    g[:256] = 2.0 ** -torch.arange(256, device="cuda").float().clamp_max(140)
    g[256:512] = 1e-30
    g[512] = 1e38
    g[513:768] = 1.0
    p.grad = g
    opt = AdamW([p], lr=0.0, state_bits=8)
    opt.step()
    m, v = opt.moments()
    gd = g.double().cpu()
    hm, _ = held((1 - 0.9) * gd, torch.zeros(1024, dtype=torch.float64))
    assert torch.equal(m.double().cpu(), hm)
    nonzero = gd != 0
    assert bool((v.cpu()[nonzero] > 0).all()) and not v.cpu()[~nonzero].any() and torch.isfinite(v).all()


@gpu
@pytest.mark.parametrize("start", (torch.float32, "codes", "torch"))
@pytest.mark.parametrize("bits", (32, 8))
def test_state_dicts(start, bits):
    pairs = make((700, (3, 5), 1000), torch.float32, torch.float32, seed=2)
    params = [p for p, _ in pairs]
    if start == "torch":
        src = torch.optim.AdamW(params, lr=0.02)
    else:
        src = AdamW(params, lr=0.02, state_bits=8 if start == "codes" else 32)
    for _ in range(3):
        src.step()
    saved = copy.deepcopy(src.state_dict())
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for q, (_, g) in zip(twins, pairs):
        q.grad = g.clone()
    dst = AdamW(twins, lr=0.7, state_bits=bits)
    before = dst._buffers["exp_avg"].data_ptr()
    dst.load_state_dict(saved)
    assert dst._buffers["exp_avg"].data_ptr() == before  # in place: captured steps stay valid
    assert dst.param_groups[0]["lr"] == 0.02 and [int(dst.state[q]["step"]) for q in twins] == [3, 3, 3]
    m, v = (x.clone() for x in dst.moments())
    at = 0
    for p, q in zip(params, twins):
        n = p.numel()
        if start == "codes":
            sm, sv = (x[at:at + n] for x in src.moments())
        else:
            sm, sv = src.state[p]["exp_avg"].reshape(-1), src.state[p]["exp_avg_sq"].reshape(-1)
        if bits == 8 and start != "codes":
            sm, sv = (x.float().cuda() for x in held(sm, sv))
        assert torch.equal(m[at:at + n], sm) and torch.equal(v[at:at + n], sv)
        at += -(-n // BLOCK) * BLOCK
    if start == "codes" and bits == 8 or start is torch.float32 and bits == 32:
        src.step()
        dst.step()
        for p, q in zip(params, twins):
            assert torch.equal(p, q)
        again = copy.deepcopy(dst.state_dict())  # there and back
        dst.load_state_dict(again)
        for key, a in again["state"].items():
            for name, x in a.items():
                assert torch.equal(x, dst.state_dict()["state"][key][name]), name
    copied = copy.deepcopy(dst)
    copied.param_groups[0]["params"][0].grad = twins[0].grad.clone()
    copied.step()
    assert int(copied.state[copied.param_groups[0]["params"][0]]["step"]) == int(dst.state[twins[0]]["step"]) + 1
    import pickle
    again = pickle.loads(pickle.dumps(dst))
    for q, r in zip(twins, again.param_groups[0]["params"]):
        r.grad = q.grad.clone()
    dst.step()
    again.step()
    for q, r in zip(twins, again.param_groups[0]["params"]):
        assert torch.equal(q, r)
    with pytest.raises(ValueError, match="groups"):
        AdamW(twins[:2]).load_state_dict(saved)
    for change in (dict(amsgrad=True), dict(maximize=True), dict(decoupled_weight_decay=False)):
        with pytest.raises(ValueError, match="amsgrad"):
            dst.load_state_dict({**saved, "param_groups": [{**saved["param_groups"][0], **change}]})
    key = next(iter(saved["state"]))
    if "exp_avg_sq" in saved["state"][key]:
        saved["state"][key]["exp_avg_sq"] = -saved["state"][key]["exp_avg_sq"]
        with pytest.raises(ValueError, match="negative"):
            dst.load_state_dict(saved)


@gpu
@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("where, dtype", (("cpu", torch.float32), ("cuda", torch.float64), ("cuda", torch.bfloat16)))
def test_state_from_elsewhere(bits, where, dtype):
    """Moments on the host, of other types, not contiguous, beside empty parameters and missing entries."""
    params = [torch.nn.Parameter(torch.randn(s, device="cuda")) for s in ((0,), (30, 9), (256,), (1, 1), (4, 0))]
    opt = AdamW(params, state_bits=bits)
    wide = [torch.randn(9, 30, device=where).to(dtype).t(), torch.ones(1, 1, device=where, dtype=dtype)]
    saved = opt.state_dict()
    saved["state"] = {k: {"step": 7.0, "exp_avg": x, "exp_avg_sq": x.abs()} for k, x in zip((1, 3), wide)}
    saved["state"][4] = {"step": torch.tensor(2), "exp_avg": params[4].data, "exp_avg_sq": params[4].data}
    opt.load_state_dict(saved)
    m, v = opt.moments()
    for at, x in ((0, wide[0]), (768, wide[1]), (512, torch.zeros(256))):
        x = x.float().cpu().reshape(-1)
        want = (x, x.abs()) if bits == 32 else held(x, x.abs())
        got = m[at:at + x.numel()].cpu(), v[at:at + x.numel()].cpu()
        for a, b in zip(got, want):
            assert torch.equal(a, b.float())
    assert [int(opt.state[p]["step"]) for p in params] == [0, 7, 0, 7, 2]
    assert all(t.shape == p.shape for p in params for k, t in opt.state[p].items() if k in ("exp_avg", "exp_avg_codes"))


@gpu
def test_torch_takes_the_state():
    """A state dict with moments in 32 bits continues in torch.optim.AdamW."""
    pairs = make((700, (3, 5)), torch.float32, torch.float32, seed=9)
    a = AdamW([p for p, _ in pairs], lr=0.02)
    for _ in range(3):
        a.step()
    twins = [torch.nn.Parameter(p.detach().clone()) for p, _ in pairs]
    b = torch.optim.AdamW(twins, lr=0.5)
    b.load_state_dict(copy.deepcopy(a.state_dict()))
    for q, (_, g) in zip(twins, pairs):
        q.grad = g.clone()
    a.step()
    b.step()
    for (p, _), q in zip(pairs, twins):
        assert float((p - q).abs().max()) <= 16 * U * 0.02 * 4 + 4 * U * float(q.abs().max())


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_captured_steps(bits):
    """A captured step replayed is the step itself, with the rate read from its tensor."""
    lr = torch.tensor(0.01, device="cuda")
    pairs = make((5000, 3, 257), torch.float32, torch.float32, seed=6)
    twins = [torch.nn.Parameter(p.detach().clone()) for p, _ in pairs]
    for q, (_, g) in zip(twins, pairs):
        q.grad = g.clone()
    a, b = AdamW([p for p, _ in pairs], lr=lr, state_bits=bits), AdamW(twins, lr=0.01, state_bits=bits)
    a.load_kernels()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        a.step()
    for i in range(4):
        rate = float(torch.tensor(0.01 * (i + 1), dtype=torch.float32))
        lr.fill_(rate)
        b.param_groups[0]["lr"] = rate
        for (p, g), q in zip(pairs, twins):
            g.mul_(-0.5)
            q.grad.copy_(g)
        graph.replay()
        b.step()
    torch.cuda.synchronize()
    for (p, _), q in zip(pairs, twins):
        assert torch.equal(p, q) and int(a.state[p]["step"]) == 4
    for x, y in zip(a.moments(), b.moments()):
        assert torch.equal(x, y)


@gpu
def test_the_version_counter_moves():
    p = torch.nn.Parameter(torch.randn(10, device="cuda"))
    loss = (p * p).sum()
    p.grad = torch.ones(10, device="cuda")
    AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@gpu
def test_closures_and_scalers():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    opt = AdamW([p], lr=0.1)

    def closure():
        opt.zero_grad()
        loss = p.square().sum()
        loss.backward()
        return loss

    assert float(opt.step(closure)) == 4.0 and float(p.detach().max()) < 1.0
    scaler = torch.amp.GradScaler("cuda", init_scale=4.0)
    opt.zero_grad()
    scaler.scale((p * math.inf).sum()).backward()
    before = p.detach().clone()
    scaler.step(opt)  # gradients that are not finite: no step
    scaler.update()
    assert torch.equal(p, before) and int(opt.state[p]["step"]) == 1


@gpu
def test_offsets_past_32_bits():
    n = (1 << 31) + 777
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    small = torch.nn.Parameter(torch.zeros(777, dtype=torch.bfloat16, device="cuda"))
    with torch.no_grad():
        for part in (slice(0, 777), slice(n - 777, n)):
            p.grad[part] = torch.linspace(-1, 1, 777, device="cuda").to(torch.bfloat16)
    small.grad = p.grad[:777].clone()
    for bits in (8,):
        opt, other = AdamW([p], lr=0.5, state_bits=bits), AdamW([small], lr=0.5, state_bits=bits)
        opt.step()
        other.step()
        assert torch.equal(p[:777], small) and torch.equal(p[n - 777:], small)
        assert not p[777:n - 777].any()
        assert torch.equal(opt.state[p]["exp_avg_codes"][:777], other.state[small]["exp_avg_codes"])


# ------------------------------------------------------------------------------ refusals
def test_refusals_on_the_cpu():
    p = torch.nn.Parameter(torch.ones(5))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        AdamW([p])
    for kw in (dict(lr=-1.0), dict(lr=math.nan), dict(lr=math.inf), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
               dict(eps=-1.0), dict(eps=math.nan), dict(weight_decay=-0.1), dict(state_bits=16),
               dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        AdamW([torch.nn.Parameter(torch.ones(5, dtype=torch.float64))])
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([torch.nn.Parameter(torch.ones(5, 6).t())])


def test_gathering_on_the_cpu():
    """The list of tensors that a step reads: what it refuses, and which entry it is of."""
    import ctypes

    from minikg_dev_b200.build import build
    build()

    def gather(params, numel=None, device=0):
        n = len(numel or params)
        table = ctypes.c_int64 * n
        sizes = table(*(numel or [p.numel() for p in params]))
        p_at, g_at, kinds, at = table(), table(), (ctypes.c_int32 * n)(), (ctypes.c_int64 * 2)()
        status = N.gather_gradients()(params, n, device, sizes, p_at, g_at, kinds, at)
        return status, at[0], at[1], list(kinds)

    def parameter(grad=True, shape=(3, 4), dtype=torch.float32):
        p = torch.nn.Parameter(torch.ones(shape, dtype=dtype))
        if grad:
            p.grad = torch.ones_like(p)
        return p

    assert gather([parameter(False), parameter(False)]) == (0, 1, 1, [-1, -1])
    assert gather([]) == (0, 0, 1, [])
    assert gather([parameter(False), parameter()])[:2] == (4, 1)  # on the host
    assert gather([parameter(False), None], [12, 12])[:2] == (1, 1)
    assert gather([parameter(), parameter()], [12])[0] == 1  # another length
    assert gather((parameter(),))[0] == 1  # not a list
    assert gather([parameter(False), parameter(), parameter()], [12, 13, 12])[:2] == (3, 1)
    assert gather([parameter(False), parameter(dtype=torch.float64)])[:2] == (5, 1)
    sparse, turned = parameter(), parameter()
    sparse.grad = torch.ones(3, 4).to_sparse()
    turned.data = torch.ones(4, 3).t()
    assert gather([parameter(False), sparse])[:2] == (2, 1)
    assert gather([turned])[:2] == (3, 0)


@gpu
def test_gradients_of_every_kind():
    """Missing, transposed, broadcast and lazily negated gradients and two types in one group."""
    g = torch.Generator(device="cuda").manual_seed(5)
    shapes = ((6, 5), (300, 4), (7,), (4, 4), (2, 3), (1,), (9, 2))
    params = [torch.nn.Parameter(torch.randn(s, generator=g, device="cuda")) for s in shapes]
    params.append(torch.nn.Parameter(torch.randn(40, generator=g, device="cuda").bfloat16()))
    params[0].grad = torch.randn(5, 6, generator=g, device="cuda").t()
    params[1].grad = torch.randn(4, generator=g, device="cuda").expand(300, 4)
    params[2].grad = torch._neg_view(torch.randn(7, generator=g, device="cuda"))
    params[4].grad = torch.randn(2, 3, generator=g, device="cuda")
    params[7].grad = torch.randn(40, generator=g, device="cuda").bfloat16()
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, twins):
        if p.grad is not None:
            q.grad = p.grad.resolve_neg().contiguous().clone()
    versions = [p._version for p in params]
    a, b = AdamW(params, lr=0.1), [AdamW([q], lr=0.1) for q in twins if q.grad is not None]
    for _ in range(2):
        a.step()
        for o in b:
            o.step()
    for i, (p, q) in enumerate(zip(params, twins)):
        assert torch.equal(p, q), i
        assert int(a.state[p]["step"]) == (0 if p.grad is None else 2)
        assert (p._version > versions[i]) == (p.grad is not None)


@gpu
def test_refusals():
    flat = torch.ones(100, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        AdamW([torch.nn.Parameter(flat[:60]), torch.nn.Parameter(flat[50:])])
    p, q = (torch.nn.Parameter(torch.ones(8, 4, device="cuda")) for _ in range(2))
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [p]})
    with pytest.raises(ValueError, match="lr"):
        opt.add_param_group({"params": [q], "lr": -1.0})
    assert len(opt.param_groups) == 1 and q not in opt.state
    p.grad = torch.ones(8, 4, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        opt.step()
    p.grad = torch.ones(8, 4, device="cuda")
    p.data = torch.ones(9, 4, device="cuda")
    with pytest.raises(RuntimeError, match="size"):
        opt.step()
    p.data = torch.ones(4, 8, device="cuda").t()
    with pytest.raises(RuntimeError, match="layout"):
        opt.step()
    p.data = torch.ones(8, 4, device="cuda")
    opt.param_groups[0]["lr"] = -0.5
    with pytest.raises(ValueError, match="lr"):
        opt.step()
    opt.param_groups[0]["lr"] = 0.5
    opt.param_groups[0]["params"].append(q)
    with pytest.raises(RuntimeError, match="changed"):
        opt.step()


def test_c_entries_refuse_bad_parameters():
    import numpy as np

    from minikg_dev_b200.build import build
    build()
    lib = N.load()
    fake = 4096  # never dereferenced: the host checks come first
    good_p = dict(lr=0.1, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, lr_device=None, param_dtype=0, grad_dtype=0,
                  state_bits=8, reserved=0)
    good_s = dict(exp_avg=fake, exp_avg_sq=fake, exp_avg_scale=fake, exp_avg_sq_scale=fake, steps=fake, ticket=fake,
                  total=512, tensors=2)

    def step(p=(), s=(), params=fake, grads=fake, numel=256, offset=256, index=1):
        rows = [np.array([x], dtype=np.int64) for x in (params, grads, numel, offset, index)]
        return lib.mkg_adamw_step(N.AdamwParams(**(good_p | dict(p))), N.AdamwState(**(good_s | dict(s))), 1,
                                  *(r.ctypes.data for r in rows), None)

    for bad in (dict(p=dict(beta1=1.0)), dict(p=dict(beta2=-0.1)), dict(p=dict(eps=-1.0)), dict(p=dict(weight_decay=-1.0)),
                dict(p=dict(lr=-1.0)), dict(p=dict(lr=math.nan)), dict(p=dict(param_dtype=3)), dict(p=dict(grad_dtype=-1)),
                dict(p=dict(state_bits=4)), dict(s=dict(exp_avg=None)), dict(s=dict(exp_avg_scale=None)),
                dict(s=dict(steps=None)), dict(s=dict(ticket=None)), dict(s=dict(total=500)), dict(s=dict(exp_avg=fake + 4)),
                dict(params=0), dict(grads=0), dict(numel=257), dict(numel=-1), dict(offset=128), dict(offset=-256),
                dict(offset=512), dict(index=2), dict(index=-1), dict(params=fake + 2), dict(grads=fake + 1)):
        assert step(**bad) == 1, bad
        assert "adamw" in N.last_error()
    assert lib.mkg_adamw_step(N.AdamwParams(**good_p), N.AdamwState(**good_s), 1, None, None, None, None, None, None) == 1
    assert lib.mkg_adamw_step(N.AdamwParams(**good_p), N.AdamwState(**good_s), 0, None, None, None, None, None, None) == 0
    for f in (lib.mkg_adamw_pack, lib.mkg_adamw_unpack):
        assert f(N.AdamwState(**good_s), None, fake, None) == 1
        assert f(N.AdamwState(**good_s), fake, fake + 4, None) == 1


def test_struct_layouts(tmp_path):
    import ctypes
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    for name, cls in (("mkg_adamw_params", N.AdamwParams), ("mkg_adamw_state", N.AdamwState)):
        fields = [f for f, _ in cls._fields_]
        src = tmp_path / "layout.c"
        src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "minikg_b200.h"\nint main(void) {\n'
                       + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                       + f'printf("%zu\\n", sizeof({name})); return 0; }}\n')
        subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
        got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                              check=True).stdout.split()]
        assert got == [getattr(cls, f).offset for f in fields] + [ctypes.sizeof(cls)]


@gpu
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_sixteen_bit_parameters_take_gradients_in_32_bits(dtype):
    """A gradient in 32 bits can be given to them as it is, after copying and unpickling too; a type that
    the program has chosen stays, and so does the type of a gradient that autograd brings."""
    import pickle
    gen = torch.Generator(device="cuda").manual_seed(3)
    p = torch.nn.Parameter(torch.randn(300, generator=gen, device="cuda").to(dtype))
    g = torch.randn(300, generator=gen, device="cuda")
    opt = AdamW([p])
    p.grad = g
    before, zero = p.detach().clone(), torch.zeros_like(g)
    opt.step()
    want, *_ = definition(before, g, zero, zero, 1)
    close(p, want, (torch.finfo(dtype).eps / 2 + 32 * U) * (want.abs() + 2e-3), "32-bit gradient")
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        q = again.param_groups[0]["params"][0]
        q.grad = g
        again.step()
    opt.step()
    assert torch.equal(p, q)
    p.grad = None
    (p * 2).sum().backward()
    assert p.grad.dtype == dtype
    chosen, wide = (torch.nn.Parameter(torch.ones(4, device="cuda", dtype=t)) for t in (dtype, torch.float32))
    chosen.grad_dtype = torch.float32
    AdamW([chosen, wide])
    assert chosen.grad_dtype is torch.float32 and wide.grad_dtype is torch.float32


@gpu
def test_large_second_moments_in_8_bits():
    """Squares past the largest held value (1.75 * 2^120, about 2.3e36) are held as that, and later steps stay
    finite: the sums are below fp32's largest value for all of these gradients."""
    big = (4.7e19, 4.8e19, 4.823e19, 4.83e19, 5e19, 5.2e19, 1e20, 3e20, 5e20)
    g = torch.full((len(big), BLOCK), 1e10, device="cuda")
    g[:, 0] = torch.tensor(big)
    g[:, 1] = -g[:, 0]
    g[:, 2] = 0.0
    g[:, 3] = 1.0
    p = torch.nn.Parameter(torch.zeros_like(g))
    p.grad = g
    opt = AdamW([p], lr=0.1, state_bits=8)
    table, most = second_table(), 1.75 * 2.0 ** 120
    for _ in range(3):
        v0 = opt.moments()[1].double().cpu()
        opt.step()
        v = opt.moments()[1].double().cpu()
        want = 0.999 * v0 + (1 - 0.999) * g.reshape(-1).double().cpu().square()
        _, _, s = hold(want.clamp_max(most), table, -90)
        s = s.repeat_interleave(BLOCK)
        least = torch.where(want > 0, table[1], 0.0)
        want = torch.maximum(table[nearest(table, (want / s).clamp_max(1.75))], least) * s
        assert torch.equal(v, want)
        assert torch.isfinite(p).all()


@gpu
@pytest.mark.parametrize("bits", (32, 8))
@pytest.mark.parametrize("eps", (0.0, 2.0 ** -62, 2.0 ** -60, 1e-18, 1e-17, 1e-16, 1e-13, 1e-11, 1e-9, 1e-8))
@pytest.mark.parametrize("beta2", (0.5, 0.999, 0.999999))
def test_small_eps(eps, bits, beta2):
    """Second moments around fp32's smallest normal number beside an eps of their root's size.  What a
    subnormal v is rounded by (its sum and two products: 3 * 2^-149) counts with half its share of v."""
    n = 4 * BLOCK
    g = torch.logspace(-19, -14, n, device="cuda")
    g[1::2] *= -1
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    p.grad = g
    opt = AdamW([p], lr=1e-3, betas=(0.9, beta2), eps=eps, weight_decay=0.0, state_bits=bits)
    for t in (1, 2):
        before, (m0, v0) = p.detach().clone(), (x.clone() for x in opt.moments())
        opt.step()
        want, m, v, (size, rate) = definition(before, g, m0, v0, t, betas=(0.9, beta2), eps=eps, wd=0.0)
        lost = 3 * 2.0 ** -149 / v
        seen = v > 64 * 2.0 ** -149  # below that the root itself is lost
        tol = rate * (3 * U * size + (8 * U + 3 * U + lost) * (m.abs() + size)) + 4 * U * (want.abs() + before.double().cpu().abs())
        close(p.detach().cpu()[seen], want[seen], tol[seen], f"step {t}")
        assert int(seen.sum()) > n // 2


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_an_unpickled_optimizer_checkpoints_its_own_moments(bits):
    """After a step of the unpickled one, its state and state dict are the original's."""
    import pickle
    pairs = make((700, (3, 5), 1000), torch.float32, torch.float32, seed=12)
    opt = AdamW([p for p, _ in pairs], lr=0.02, state_bits=bits)
    opt.step()
    for again in (pickle.loads(pickle.dumps(opt)), copy.deepcopy(opt)):
        twins = again.param_groups[0]["params"]
        for q, (p, g) in zip(twins, pairs):
            q.grad = g.clone()
        again.step()
        moved = copy.deepcopy(opt)
        for q, (_, g) in zip(moved.param_groups[0]["params"], pairs):
            q.grad = g.clone()
        moved.step()
        want = moved.state_dict()["state"]
        for key, entry in again.state_dict()["state"].items():
            assert float(entry["step"]) == 2.0
            for name, x in entry.items():
                assert torch.equal(x, want[key][name]), name
        at = 0
        for q in twins:
            assert int(again.state[q]["step"]) == 2
            name = "exp_avg" if bits == 32 else "exp_avg_codes"
            flat = again._buffers["exp_avg"][at:at + q.numel()]
            assert torch.equal(again.state[q][name].reshape(-1), flat) and bool(flat.any())
            at += -(-q.numel() // BLOCK) * BLOCK


@gpu
def test_load_kernels_of_many_tensors(monkeypatch):
    """What is loaded is what a step of so many tensors launches, for each pair of types."""
    few, many = make((5,) * 40, torch.bfloat16, torch.bfloat16, seed=1), make((5,) * 131, torch.float32, torch.float32, seed=2)
    opt = AdamW([p for p, _ in few + many])
    asked = []
    call = opt._call

    def record(group, p_dtype, g_dtype, p_at, *rest):
        asked.append((p_dtype, g_dtype, len(p_at)))
        call(group, p_dtype, g_dtype, p_at, *rest)
    monkeypatch.setattr(opt, "_call", record)
    opt.load_kernels()
    loaded, asked[:] = sorted(asked, key=str), []
    assert all(int(opt.state[p]["step"]) == 0 for p, _ in few + many)
    opt.step()
    assert loaded == sorted(asked, key=str) and len(loaded) == 2


FIRST_CAPTURE = """
import sys
import torch
from minikg_dev_b200.optim import AdamW
bits = int(sys.argv[1])
params = [torch.nn.Parameter(torch.full((3 + i,), 1.0, device="cuda")) for i in range(131)]
twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
for p in params + twins:
    p.grad = torch.linspace(-1, 1, p.numel(), device="cuda")
a, b = AdamW(params, state_bits=bits), AdamW(twins, state_bits=bits)
a.load_kernels()
graph = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(graph):
    a.step()
for _ in range(2):
    graph.replay()
    b.step()
torch.cuda.synchronize()
assert all(torch.equal(p, q) and int(a.state[p]["step"]) == 2 for p, q in zip(params, twins))
print("same")
"""


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_the_first_step_of_many_tensors_is_captured(bits):
    """In a process of its own, in which nothing has loaded the kernel before."""
    import subprocess
    import sys
    from pathlib import Path
    out = subprocess.run([sys.executable, "-c", FIRST_CAPTURE, str(bits)], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parent.parent)
    assert out.returncode == 0 and out.stdout.strip().endswith("same"), out.stderr[-2000:]


@gpu
def test_a_loaded_group_keeps_what_the_saved_one_had():
    """A scheduler resumes from a loaded optimizer, and other keys of a group come along, as copies."""
    (p, _), = make((40,), torch.float32, torch.float32)
    src = AdamW([{"params": [p], "note": ["facts"]}], lr=0.1)
    sched = torch.optim.lr_scheduler.ExponentialLR(src, 0.5)
    for _ in range(2):
        src.step()
        sched.step()
    saved = src.state_dict()
    q = torch.nn.Parameter(p.detach().clone())
    dst = AdamW([q], lr=0.7)
    dst.load_state_dict(saved)
    group = dst.param_groups[0]
    assert group["initial_lr"] == 0.1 and group["lr"] == 0.025 and group["note"] == ["facts"]
    assert group["params"][0] is q
    src.param_groups[0]["note"].append("changed")
    assert group["note"] == ["facts"]
    again = torch.optim.lr_scheduler.ExponentialLR(dst, 0.5, last_epoch=1)
    q.grad = torch.ones(40, device="cuda")
    dst.step()
    again.step()
    sched.step()
    assert dst.param_groups[0]["lr"] == src.param_groups[0]["lr"]
    torch_side = torch.optim.AdamW([torch.nn.Parameter(p.detach().clone())], lr=0.3)
    torch_side.load_state_dict(dst.state_dict())
    assert torch_side.param_groups[0]["initial_lr"] == 0.1


@gpu
@pytest.mark.parametrize("where", ("cuda", "cpu"))
def test_a_loaded_rate_is_a_copy(where):
    """Two optimizers do not share a rate's tensor after a load; one saved on the host comes to the device."""
    (p, _), (q, _) = make((40, 40), torch.float32, torch.float32)
    src, dst = AdamW([p], lr=torch.tensor(0.25, device="cuda")), AdamW([q], lr=0.7)
    saved = src.state_dict()
    saved["param_groups"][0]["lr"] = saved["param_groups"][0]["lr"].to(where)
    dst.load_state_dict(saved)
    src.param_groups[0]["lr"].fill_(0.5)
    assert float(dst.param_groups[0]["lr"]) == 0.25 and dst.param_groups[0]["lr"].is_cuda
    kept = dst.param_groups[0]["lr"]
    dst.step()
    dst.load_state_dict(src.state_dict())
    assert dst.param_groups[0]["lr"] is kept and float(kept) == 0.5  # in place: captured steps read it


@gpu
def test_hooks_around_loading():
    """Hooks before a load see the dict and may give another; hooks after it see the loaded optimizer."""
    (p, _), (q, _) = make((40, 40), torch.float32, torch.float32)
    src, dst = AdamW([p], lr=0.25), AdamW([q], lr=0.7)
    src.step()
    saved, seen = src.state_dict(), []

    def halve(opt, d):
        seen.append(("pre", opt is dst, d["param_groups"][0]["lr"]))
        return {**d, "param_groups": [{**d["param_groups"][0], "lr": d["param_groups"][0]["lr"] / 2}]}

    handles = [dst.register_load_state_dict_pre_hook(halve),
               dst.register_load_state_dict_pre_hook(lambda opt, d: seen.append("first"), prepend=True),
               dst.register_load_state_dict_post_hook(
                   lambda opt: seen.append(("post", opt.param_groups[0]["lr"], int(opt.state[q]["step"])))),
               dst.register_load_state_dict_post_hook(lambda opt: seen.append("soonest"), prepend=True)]
    dst.load_state_dict(saved)
    assert seen == ["first", ("pre", True, 0.25), "soonest", ("post", 0.125, 1)]
    assert saved["param_groups"][0]["lr"] == 0.25
    for h in handles:
        h.remove()
    dst.load_state_dict(saved)
    assert len(seen) == 4 and dst.param_groups[0]["lr"] == 0.25


@gpu
def test_pickling_beside_schedulers_and_hooks():
    """What others attach to an optimizer (a scheduler wraps its step, hooks may be local functions) stays
    with it: copies and pickles carry groups and moments, as those of torch's optimizers do."""
    import pickle
    pairs = make((300, 40), torch.float32, torch.float32, seed=4)
    opt = AdamW([p for p, _ in pairs], lr=0.1)
    sched = torch.optim.lr_scheduler.ExponentialLR(opt, 0.5)
    calls = []
    opt.register_step_post_hook(lambda *a: calls.append(1))
    opt.register_load_state_dict_post_hook(lambda *a: calls.append(2))
    opt.step()
    sched.step()
    assert calls == [1]
    for again in (pickle.loads(pickle.dumps(opt)), copy.deepcopy(opt)):
        assert again.param_groups[0]["lr"] == 0.05
        for q, (_, g) in zip(again.param_groups[0]["params"], pairs):
            q.grad = g.clone()
        again.step()
        again.register_step_post_hook(lambda *a: calls.append(3))
        again.load_state_dict(again.state_dict())
        assert [int(again.state[q]["step"]) for q in again.param_groups[0]["params"]] == [2, 2]
    assert calls == [1] and int(opt.state[pairs[0][0]]["step"]) == 1


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_a_captured_step_keeps_its_moments(bits):
    """A group that is added after a capture moves the moments; what the graph would write to is not
    handed to others (the graph itself has to be captured again, and is not replayed here)."""
    pairs = make((5000, 300), torch.float32, torch.float32, seed=6)
    (p, _), (q, _) = pairs
    opt = AdamW([p], state_bits=bits)
    opt.load_kernels()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    old = [(b.data_ptr(), b.numel(), b.dtype) for b in opt._buffers.values()]
    opt.add_param_group({"params": [q]})
    now = {b.data_ptr() for b in opt._buffers.values()}
    others = [torch.empty(n, dtype=t, device="cuda") for _, n, t in old for _ in range(20)]
    taken = {x.data_ptr() for x in others} | now
    assert not any(at in taken for at, _, _ in old)


@gpu
def test_optimizers_that_were_never_captured_keep_one_set_of_moments():
    pairs = make((5000, 300), torch.float32, torch.float32, seed=6)
    opt = AdamW([pairs[0][0]])
    opt.step()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(8):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(256, device="cuda"))]})
    assert torch.cuda.memory_allocated() - before < 4 * 2 * 5000 * 4


@gpu
@pytest.mark.parametrize("default", (torch.bfloat16, torch.float64))
@pytest.mark.parametrize("bits", (32, 8))
def test_state_dicts_under_another_default_type(bits, default):
    """torch's default type decides nothing: steps are float32 on the host, scales fp32."""
    (p, g), (q, _) = make((700, 700), torch.float32, torch.float32, seed=8)
    src = AdamW([p], state_bits=8)
    src.step()
    src._buffers["steps"].fill_(1001)  # not a bf16 number
    want = [x.clone() for x in src.moments()]
    q.data.copy_(p.detach())
    q.grad = g.clone()
    torch.set_default_dtype(default)
    try:
        saved = src.state_dict()
        dst = AdamW([q], state_bits=bits)
        dst.load_state_dict(saved)
        entry = saved["state"][0]["step"]
        got = [x.clone() for x in dst.moments()]
        dst.step()
    finally:
        torch.set_default_dtype(torch.float32)
    src.step()
    assert entry.dtype == torch.float32 and float(entry) == 1001.0 and not entry.is_cuda
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert int(dst.state[q]["step"]) == 1002
    if bits == 8:
        assert torch.equal(p, q)
    else:
        close(q, p.detach().double().cpu(), 64 * U * (1e-3 + p.detach().double().cpu().abs()), "step")


def test_every_tensor_names_its_type():
    """A factory call that leaves its type to torch's default is read as something else by a kernel."""
    import ast
    from pathlib import Path
    for module in ("optim", "logprobs"):
        tree = ast.parse((Path(__file__).resolve().parent.parent / "minikg_dev_b200" / f"{module}.py").read_text())
        for call in ast.walk(tree):
            if isinstance(call, ast.Call) and isinstance(call.func, ast.Attribute) and isinstance(call.func.value, ast.Name) \
                    and call.func.value.id == "torch" and call.func.attr in ("zeros", "ones", "empty", "full", "tensor"):
                named = "dtype" in {k.arg for k in call.keywords}
                assert named or ast.unparse(call) == "torch.empty(0)", f"{module}.py:{call.lineno}: {ast.unparse(call)}"


@gpu
@pytest.mark.parametrize("call", (0, 1, 3))
def test_a_group_without_memory_leaves_the_optimizer_as_it_was(call, monkeypatch):
    (p, _), (q, _) = make((300, 40), torch.float32, torch.float32)
    opt = AdamW([p])
    opt.step()
    before = [x.clone() for x in opt.moments()]
    zeros, made = torch.zeros, []

    def full(*args, **kw):
        made.append(1)
        if len(made) > call:
            raise torch.OutOfMemoryError("no memory left")
        return zeros(*args, **kw)
    monkeypatch.setattr(torch, "zeros", full)
    with pytest.raises(torch.OutOfMemoryError):
        opt.add_param_group({"params": [q]})
    monkeypatch.undo()
    assert len(opt.param_groups) == 1 and q not in opt.state
    assert all(torch.equal(a, b) for a, b in zip(opt.moments(), before))
    opt.step()
    assert int(opt.state[p]["step"]) == 2
    opt.add_param_group({"params": [q]})
    opt.step()
    assert int(opt.state[p]["step"]) == 3 and int(opt.state[q]["step"]) == 1
