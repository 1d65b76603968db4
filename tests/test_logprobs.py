"""target_logprobs against its definition in float64: values, alternatives, gradients, the rows and
columns where it can go wrong, and its refusals.

Tolerances, from the arithmetic.  fp32 rounds by u = 2^-24.  With y_j = (x_j - max) / tau in bits:
* the sum s = sum 2^{y_j}: 2^y is good to 2^-22 and y to 3 u |y| (only |y| < 30 contributes:
  30 * 3 u * ln 2 < 2^-18), adding n terms per thread and a tree costs (n + 16) u; so s is good to
  rel(n) = 2^-17 + (n + 16) u, with n <= width / 32 for a warp per row and never above 4096 here.
  rel_typical below uses the far smaller share of terms with large |y|: 2^-20 + (n + 16) u / 4.
* log p = ln 2 (y - log2 s): 4 u |log p| + 4 u |log s| + rel;  entropy = log s - t / s: both terms
  carry rel, each is at most log(width).
* gradient: p from 2^{y - log2 s}: the exponent is off by at most 3 u (|y| + log2 s) + rel, that is
  below 2^-17 where p matters; its terms add up in absolute value, then one rounding to the type
  (half a step: eps / 2).
"""
from __future__ import annotations

import math

import pytest
import torch

from minikg_dev_b200 import _native as N
from minikg_dev_b200.logprobs import target_logprobs

gpu = pytest.mark.gpu
U = 2.0 ** -24


def definition(x, targets, tau, mask, topk, ups=None):
    """Everything in float64, on the logits' device: outputs, and the gradient of x for the
    upstream gradients (logprobs, entropy, lse, top_logprobs)."""
    z = x.double() / tau
    on = torch.ones_like(z, dtype=torch.bool) if mask is None else mask.expand(z.shape)
    z = torch.where(on, z, -math.inf)
    top = z.amax(1, keepdim=True)
    none = top == -math.inf
    top = torch.where(none, 0.0, top)
    y = z - top  # logits of size 1e38 would swallow the log of the sum
    log_sum = torch.logsumexp(y, 1, keepdim=True)
    lse = (top + log_sum)[:, 0]
    logp = torch.where(none, -math.inf, y - log_sum)
    p = logp.exp()
    ent = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
    lp = torch.where(targets < 0, 0.0, logp.gather(1, targets.clamp_min(0)))
    k = min(topk, x.shape[1])
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :k]
    top = logp.gather(1, order)
    ids = torch.where(top == -math.inf, -1, order)
    pad = (0, topk - k)
    ids, top = torch.nn.functional.pad(ids, pad, value=-1), torch.nn.functional.pad(top, pad, value=-math.inf)
    out = dict(logprobs=lp, entropy=ent, lse=lse, top_ids=ids, top_logprobs=top)
    if ups is not None:
        g_lp, g_h, g_l, g_top = (u.double() for u in ups)
        up, size = torch.zeros_like(z), torch.zeros_like(z)
        for i, g in ((targets, g_lp), (ids, g_top)):
            g = torch.where(i < 0, 0.0, g)
            up.scatter_add_(1, i.clamp_min(0), g)
            size.scatter_add_(1, i.clamp_min(0), g.abs())
        lg = torch.where(p > 0, logp, 0.0)
        grad = up + p * (g_l[:, None] - up.sum(1, keepdim=True) - g_h[:, None] * (lg + ent[:, None]))
        share = p * (g_l[:, None].abs() + size.sum(1, keepdim=True) + g_h[:, None].abs() * (lg.abs() + ent[:, None]))
        big = size + share
        out["grad"] = torch.where(on & ~none, grad / tau, 0.0)
        out["size"] = torch.where(on & ~none, big / tau, 0.0)
        out["flushed"] = torch.where(on & ~none & (p < 2.0 ** -125), share / tau, 0.0)
    return out


def check(got, want, width, err=""):
    n = max(width / 32 if width <= 1024 else 4096 * 2, 1)
    rel = 2.0 ** -20 + (min(n, 4096) + 16) * U / 4
    log_w = math.log(max(width, 2))
    assert torch.equal(got.top_ids, want["top_ids"]), err
    for name in ("logprobs", "top_logprobs", "lse"):
        torch.testing.assert_close(getattr(got, name).double().reshape(want[name].shape), want[name], rtol=8 * U,
                                   atol=rel + 8 * U * log_w, equal_nan=True, msg=lambda m, n=name: f"{err} {n}: {m}")
    torch.testing.assert_close(got.entropy.double(), want["entropy"], rtol=0, atol=2 * log_w * rel, equal_nan=True)


def check_grad(got, want):
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal
    off = (got.double() - want["grad"]).abs()
    tol = 2.0 ** -17 * want["size"] + eps / 2 * (want["grad"].abs() + 2.0 ** -17 * want["size"]) + tiny
    tol += want["flushed"]  # p below 2^-126 is 0 in fp32 without subnormals: its whole share is missing
    assert bool((off <= tol).all()), f"worst {float((off / tol).max())} times the tolerance"


def case(rows, width, s, dtype, mask, seed, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, width, generator=g, device="cuda") * scale).to(dtype)
    t = torch.randint(0, width, (rows, s), generator=g, device="cuda")
    if s > 1:
        t[:, -1] = t[:, 0]      # the same column twice
        t[0, -1] = -1
    m = None
    if mask:
        m = torch.rand(rows, width, generator=g, device="cuda") < 0.7
        if rows > 2:
            m[rows // 2] = False
    return x, t, m


def run(x, t, m, tau, topk, seed=1):
    """Outputs and gradient of one call with gradients through every output, and what they should be."""
    g = torch.Generator(device=x.device).manual_seed(seed)
    rows = x.shape[0]
    ups = [torch.randn(sh, generator=g, device=x.device) for sh in ((rows, t.shape[1]), (rows,), (rows,), (rows, topk))]
    leaf = x.detach().requires_grad_(True)
    out = target_logprobs(leaf, t, tau, m, topk)
    grad, = torch.autograd.grad([out.logprobs, out.entropy, out.lse, out.top_logprobs], leaf, ups)
    return out, grad, definition(x, t, tau, m, topk, ups)


WIDTHS = (1, 2, 25, 31, 32, 33, 64, 103, 255, 1000, 1024, 1025, 2051, 8191, 29649, 100003)


@gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16, torch.float16))
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(width, dtype):
    for rows, s, topk, mask, tau in ((1, 1, 1, False, 1.0), (5, 3, 8, True, 0.7), (37, 1, 32, False, 1.3)):
        x, t, m = case(rows, width, s, dtype, mask, seed=width + rows)
        out, grad, want = run(x, t, m, tau, topk)
        check(out, want, width, f"{rows} x {width}")
        check_grad(grad, want)


@gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
def test_few_long_rows(dtype):
    x, t, m = case(3, 1000003, 4, dtype, True, seed=5)
    out, grad, want = run(x, t, m, 1.0, 20)
    check(out, want, x.shape[1])
    check_grad(grad, want)


@gpu
def test_many_rows():
    x, t, m = case(5000, 75, 2, torch.float32, True, seed=6)
    out, grad, want = run(x, t, m, 1.0, 5)
    check(out, want, 75)
    check_grad(grad, want)


@gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.float16))
@pytest.mark.parametrize("rows, width, topk, mask", ((8192, 103, 5, False), (8197, 25, 8, True), (9001, 122, 1, True),
                                                     (8200, 7, 8, False), (8193, 1, 3, True), (8192, 123, 9, False)))
def test_many_narrow_rows(rows, width, topk, mask, dtype):
    """Enough short rows that several share a warp; the last warps are part full."""
    x, t, m = case(rows, width, 2, dtype, mask, seed=rows)
    x[5] = 0.0                      # ties all along
    x[6, :] = torch.arange(width, device="cuda").to(dtype)
    out, grad, want = run(x, t, m, 0.9, topk)
    check(out, want, width)
    check_grad(grad, want)


@gpu
@pytest.mark.parametrize("width", (40, 1024, 5000, 70001))
@pytest.mark.parametrize("kind", ("equal", "ascending", "descending", "one thread", "zeros of both signs"))
def test_ties_and_orders(width, kind):
    """Alternatives in value order with ties to the lowest column, wherever the large values sit."""
    j = torch.arange(width, device="cuda", dtype=torch.float32)
    x = {"equal": torch.zeros(width, device="cuda"), "ascending": j / width, "descending": -j / width,
         "one thread": torch.where(j % 1024 < 4, 5.0 + (j // 1024) % 3, j % 2),
         "zeros of both signs": torch.where(j % 2 == 0, -0.0, 0.0)}[kind].repeat(2, 1)
    t = torch.zeros((2, 1), dtype=torch.int64, device="cuda")
    for topk in (1, 7, 32):
        out, grad, want = run(x, t, None, 1.0, topk)
        check(out, want, width, f"{kind} top {topk}")
        check_grad(grad, want)
    if width == 40:  # the same where several rows share a warp
        out = target_logprobs(x[:1].expand(8192, width), t[:1].expand(8192, 1), topk=7)
        assert torch.equal(out.top_ids, definition(x[:1], t[:1], 1.0, None, 7)["top_ids"].expand(8192, 7))


@gpu
@pytest.mark.parametrize("width", (33, 1500, 40000))
def test_strides_and_masks(width):
    g = torch.Generator(device="cuda").manual_seed(3)
    big = torch.randn(6, width + 13, generator=g, device="cuda")
    t = torch.randint(0, width, (6, 2), generator=g, device="cuda")
    row_mask = torch.rand(width, generator=g, device="cuda") < 0.5
    wide_mask = torch.rand(6, width + 5, generator=g, device="cuda") < 0.5
    for x in (big[:, 3:3 + width], big[:, 1:1 + width], big[::2, :width], big[:1, 5:5 + width].expand(6, width),
              torch.randn(width, 6, generator=g, device="cuda").t()):
        across = torch.zeros(width, x.shape[0], dtype=torch.bool, device="cuda")
        across[::3] = True
        for m in (None, row_mask, wide_mask[:x.shape[0], 2:2 + width], row_mask[None].expand(x.shape[0], width),
                  across.t()):
            out, grad, want = run(x, t[:x.shape[0]], m, 1.0, 6)
            check(out, want, width)
            check_grad(grad, want)


@gpu
def test_leading_dimensions():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(2, 3, 4, 57, generator=g, device="cuda")
    t = torch.randint(0, 57, (2, 3, 4), generator=g, device="cuda", dtype=torch.int32)
    flat = target_logprobs(x.view(24, 57), t.view(24, 1).long(), topk=4)
    out = target_logprobs(x, t, topk=4)
    assert out.logprobs.shape == t.shape and out.entropy.shape == (2, 3, 4) and out.top_ids.shape == (2, 3, 4, 4)
    assert torch.equal(out.logprobs.reshape(-1), flat.logprobs.reshape(-1))
    swapped = target_logprobs(x.transpose(0, 1), t.transpose(0, 1), topk=4)
    assert torch.equal(swapped.logprobs, out.logprobs.transpose(0, 1))
    one = target_logprobs(x[0, 0, 0], t[0, 0, 0])
    assert one.logprobs.shape == () and one.logprobs == out.logprobs[0, 0, 0] and one.top_ids.shape == (0,)
    none = target_logprobs(x[:0], t[:0], topk=3)
    assert none.logprobs.shape == (0, 3, 4) and none.top_ids.shape == (0, 3, 4, 3)
    assert target_logprobs(x, x.new_empty((2, 3, 4, 0), dtype=torch.int64)).logprobs.shape == (2, 3, 4, 0)


@gpu
@pytest.mark.parametrize("width", (20, 3001, 50000))
def test_rows_without_candidates_and_masked_values(width):
    x = torch.randn(5, width, device="cuda")
    m = torch.ones(5, width, dtype=torch.bool, device="cuda")
    m[1] = False                        # nothing left
    x[2] = -math.inf                    # nothing above -inf
    m[3, 4:], x[3, 4:] = False, math.nan  # NaN and infinities off the candidates
    x[3, 5] = math.inf
    x[4, :] = torch.finfo(torch.float32).min  # the type's lowest value is a candidate like another
    t = torch.tensor([[0, 1], [0, 1], [0, 1], [0, 5], [3, -1]], device="cuda")
    out, grad, _ = run(x, t, m, 1.0, 6)
    clean = torch.where(m, x, torch.zeros_like(x))
    ups_seed = 1
    g = torch.Generator(device="cuda").manual_seed(ups_seed)
    ups = [torch.randn(sh, generator=g, device="cuda") for sh in ((5, 2), (5,), (5,), (5, 6))]
    want = definition(clean, t, 1.0, m, 6, ups)
    check(out, want, width)
    check_grad(grad, want)
    assert out.lse[1] == -math.inf and out.entropy[1] == 0 and not grad[1:3].any()
    assert out.logprobs[3, 1] == -math.inf and (out.top_ids[1:3] == -1).all()


@gpu
@pytest.mark.parametrize("width", (20, 3001, 50000))
@pytest.mark.parametrize("bad", (math.nan, math.inf))
def test_not_finite_candidates_make_the_row_nan(width, bad):
    x = torch.randn(3, width, device="cuda")
    clean = x.clone()
    x[1, width // 2] = bad
    t = torch.zeros((3, 1), dtype=torch.int64, device="cuda")
    out, grad, _ = run(x, t, None, 1.0, 4)
    for v in (out.logprobs[1], out.entropy[1], out.lse[1], out.top_logprobs[1], grad[1]):
        assert torch.isnan(v).all()
    assert (out.top_ids[1] == -1).all()
    other, other_grad, _ = run(clean, t, None, 1.0, 4)
    for i in (0, 2):
        assert torch.equal(out.logprobs[i], other.logprobs[i]) and torch.equal(grad[i], other_grad[i])
        assert torch.equal(out.top_ids[i], other.top_ids[i])


@gpu
def test_peaked_and_far_rows():
    """Logits far from zero keep the digits of their differences; a peaked row has entropy near 0."""
    x = torch.randn(4, 2000, device="cuda", dtype=torch.float64).float()
    x[0] += 30000.0
    x[1] -= 30000.0
    x[2, 7] = 200.0
    x[3] *= 40.0
    t = torch.full((4, 1), 7, device="cuda")
    out, grad, want = run(x, t, None, 1.0, 3)
    rel = 2.0 ** -20
    torch.testing.assert_close(out.logprobs.double(), want["logprobs"], rtol=8 * U, atol=4 * rel)
    torch.testing.assert_close(out.entropy.double(), want["entropy"], rtol=0, atol=16 * rel)
    torch.testing.assert_close(out.lse.double(), want["lse"], rtol=4 * U, atol=4 * rel)
    check_grad(grad, want)


@gpu
def test_offsets_past_32_bits():
    stride = (1 << 30) + 24
    flat = torch.empty(2 * stride + 4100, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((3, 4099), (stride, 1))
    x.copy_(torch.randn(3, 4099, device="cuda"))
    t = torch.tensor([[5], [4098], [0]], device="cuda")
    out, grad, want = run(x, t, None, 1.0, 8)
    check(out, want, 4099)
    check_grad(grad, want)


@gpu
def test_gradient_against_differences():
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(2, 2100, generator=g, device="cuda")
    t = torch.tensor([[3, 3, 900], [-1, 2000, 0]], device="cuda")
    w = torch.randn(2, 3, generator=g, device="cuda")
    d = torch.randn(2, 2100, generator=g, device="cuda")

    def loss(v):
        o = target_logprobs(v, t, 0.8)
        return (o.logprobs * w).double().sum() + 0.3 * o.entropy.double().sum() - 0.2 * o.lse.double().sum()

    leaf = x.clone().requires_grad_(True)
    loss(leaf).backward()
    h = 2.0 ** -7
    diff = (loss(x + h * d) - loss(x - h * d)) / (2 * h)
    along = (leaf.grad.double() * d).sum()
    # third derivatives of the loss along d are below 100, and the loss's rounding is below 2^-18
    assert abs(float(diff - along)) < 100 * h * h / 6 + 2 * 2.0 ** -18 / h


@gpu
def test_only_the_asked_gradients():
    x, t, m = case(4, 3000, 2, torch.float32, False, seed=8)
    leaf = x.clone().requires_grad_(True)
    out = target_logprobs(leaf, t, topk=3)
    assert not out.top_ids.requires_grad
    a, = torch.autograd.grad(out.entropy.sum(), leaf, retain_graph=True)
    zeros = [torch.zeros(s, device="cuda") for s in ((4, 2), (4,), (4, 3))]
    want = definition(x, t, 1.0, None, 3, (zeros[0], torch.ones(4, device="cuda"), zeros[1], zeros[2]))
    check_grad(a, want)
    b, = torch.autograd.grad(out.logprobs.sum(), leaf)
    want = definition(x, t, 1.0, None, 3, (torch.ones(4, 2, device="cuda"), zeros[1], zeros[1], zeros[2]))
    check_grad(b, want)


@gpu
def test_the_same_bits_every_time():
    x, t, m = case(7, 30011, 3, torch.bfloat16, True, seed=2)
    a, ga, _ = run(x, t, m, 1.0, 9)
    b, gb, _ = run(x, t, m, 1.0, 9)
    for u, v in zip((*a, ga), (*b, gb)):
        assert torch.equal(u, v)


@gpu
def test_bad_targets_are_flagged_not_read():
    x = torch.randn(2, 50, device="cuda")
    for bad in (50, -2, 1 << 40):
        leaf = x.clone().requires_grad_(True)
        out = target_logprobs(leaf, torch.tensor([[3, bad], [1, 2]], device="cuda"))
        out.logprobs[:, 0].sum().backward()
        assert torch.isnan(out.logprobs[0, 1]) and torch.isfinite(out.logprobs[1]).all()
        with pytest.raises(RuntimeError, match="target"):
            N.raise_device_errors(x.device)
        assert torch.isfinite(leaf.grad).all()


@gpu
def test_streams_and_graphs():
    x, t, m = case(6, 20011, 2, torch.float32, True, seed=12)
    want = target_logprobs(x, t, 1.0, m, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = target_logprobs(x, t, 1.0, m, 5)
        leaf = x.clone().requires_grad_(True)
        static = torch.randn(6, 2, device="cuda")

        def step():
            out = target_logprobs(leaf, t, 1.0, m, 5)
            return out, torch.autograd.grad(out.logprobs, leaf, static)[0]

        step()
    torch.cuda.synchronize()
    assert torch.equal(got.logprobs, want.logprobs) and torch.equal(got.top_ids, want.top_ids)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, grad = step()
    y, _, _ = case(6, 20011, 2, torch.float32, True, seed=13)
    with torch.no_grad():
        leaf.copy_(y)
    graph.replay()
    torch.cuda.synchronize()
    fresh = y.clone().requires_grad_(True)
    o = target_logprobs(fresh, t, 1.0, m, 5)
    want_grad, = torch.autograd.grad(o.logprobs, fresh, static)
    assert torch.equal(out.logprobs, o.logprobs) and torch.equal(out.top_ids, o.top_ids)
    assert torch.equal(grad, want_grad)


@gpu
@pytest.mark.parametrize("rows, width", ((3, 40), (4, 2500), (2, 70001), (4100, 600)))
def test_many_targets(rows, width):
    """More targets than lanes, threads or columns: each column collects all that is named there."""
    s = 1024 if rows < 100 else 70
    x, t, m = case(rows, width, s, torch.float32, True, seed=width)
    t[1, 5:] = t[1, 5]  # one column, over and over
    t[2 % rows, ::2] = -1
    out, grad, want = run(x, t, m, 1.1, 3)
    check(out, want, width)
    check_grad(grad, want)


@gpu
@pytest.mark.parametrize("dtype", (torch.float32, torch.bfloat16))
@pytest.mark.parametrize("rows, width, topk, mask", ((4096, 300, 0, False), (4099, 513, 5, True), (4101, 1201, 20, False),
                                                     (4097, 2600, 8, True), (4096, 5003, 0, True), (4100, 130, 0, True),
                                                     (4098, 1500, 32, True)))
def test_many_streamed_rows(rows, width, topk, mask, dtype):
    """Enough rows of middling length that a warp, or eight lanes, stream each."""
    x, t, m = case(rows, width, 2, dtype, mask, seed=rows + width)
    x[5] = 0.0                      # ties all along
    x[6, :] = torch.arange(width, device="cuda").to(dtype)
    x[7, :] = torch.where(torch.arange(width, device="cuda") // 4 % 32 == 3, 9.0, 0.0).to(dtype)  # one lane has them all
    x[8, 1] = math.nan
    if m is not None:
        m[8, 1] = False             # off the candidates: not seen
    else:
        x[8, 1] = 0.0
    out, grad, want = run(x, t, m, 0.9, topk)
    check(out, want, width)
    check_grad(grad, want)
    x[9, width - 1] = math.inf
    if m is not None:
        m[9, width - 1] = True
    bad = target_logprobs(x, t, 0.9, m, topk)
    assert torch.isnan(bad.lse[9]) and (bad.top_ids[9] == -1).all() and torch.equal(bad.top_ids[:9], out.top_ids[:9])


@gpu
def test_two_streams_at_once():
    """Calls in flight together share nothing: each has its own workspace."""
    cases = [case(3, 300007, 2, torch.float32, False, seed=20 + i)[:2] for i in range(4)]
    want = [target_logprobs(x, t, 1.0, None, 12) for x, t in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, (x, t) in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(target_logprobs(x, t, 1.0, None, 12))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, want[i % 4]):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------ refusals (CPU)
@pytest.mark.parametrize("change, error", [
    (dict(logits=torch.zeros(2, 5, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(logits=torch.zeros(())), ValueError),
    (dict(targets=torch.zeros(2, 1)), TypeError),
    (dict(targets=torch.zeros(3, 1, dtype=torch.int64)), ValueError),
    (dict(targets=torch.zeros(2, 1, 1, dtype=torch.int64)), ValueError),
    (dict(targets=torch.zeros(2, 1025, dtype=torch.int64)), ValueError),
    (dict(topk=33), ValueError),
    (dict(topk=-1), ValueError),
    (dict(tau=0.0), ValueError),
    (dict(tau=math.inf), ValueError),
    (dict(tau=math.nan), ValueError),
    (dict(mask=torch.ones(2, 5)), TypeError),
    (dict(mask=torch.ones(2, 4, dtype=torch.bool)), ValueError),
    (dict(), RuntimeError),  # fine, but on the CPU
])
def test_refusals(change, error):
    args = dict(logits=torch.zeros(2, 5), targets=torch.zeros(2, 1, dtype=torch.int64)) | change
    with pytest.raises(error):
        target_logprobs(**args)


def test_c_entries_refuse_bad_parameters():
    from minikg_dev_b200.build import build
    build()
    lib = N.load()
    good = dict(rows=2, width=5, row_stride=5, mask_row_stride=0, targets=1, topk=1, tau=1.0, dtype=0, reserved=0)
    for change in (dict(rows=-1), dict(width=0), dict(width=(1 << 30) + 1), dict(targets=1025), dict(topk=33),
                   dict(tau=0.0), dict(tau=-1.0), dict(dtype=3), dict(row_stride=-1)):
        p = N.LogprobParams(**(good | change))
        assert lib.mkg_logprob_workspace_bytes(p) == 0
        assert lib.mkg_logprob_forward(p, *[None] * 10, 0, None, None) != N.MKG_OK
        assert lib.mkg_logprob_backward(p, *[None] * 12) != N.MKG_OK
        assert "logprob" in N.last_error()
    p = N.LogprobParams(**good)
    assert lib.mkg_logprob_forward(p, *[None] * 10, 0, None, None) != N.MKG_OK  # null pointers
    p = N.LogprobParams(**(good | dict(rows=1, width=1 << 20, row_stride=1 << 20)))
    need = lib.mkg_logprob_workspace_bytes(p)
    assert need > 0  # one long row is cut over several blocks
    fake = 256  # never dereferenced: the workspace is refused first
    assert lib.mkg_logprob_forward(p, *[fake] * 10, need - 1, None, None) == 3


def test_params_layout(tmp_path):
    """The ctypes mirror of mkg_logprob_params has the C layout."""
    import ctypes
    import subprocess
    from pathlib import Path
    root = Path(__file__).resolve().parent.parent
    fields = [f for f, _ in N.LogprobParams._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "minikg_b200.h"\nint main(void) {\n'
                   + "".join(f'printf("%zu\\n", offsetof(mkg_logprob_params, {f}));\n' for f in fields)
                   + 'printf("%zu\\n", sizeof(mkg_logprob_params)); return 0; }\n')
    subprocess.run(["gcc", "-I", str(root / "include"), str(src), "-o", str(tmp_path / "layout")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == [getattr(N.LogprobParams, f).offset for f in fields] + [ctypes.sizeof(N.LogprobParams)]


class Recorder:
    """Stands in for the library on the host: remembers what it was asked to read."""

    def __init__(self):
        self.calls = []

    def mkg_logprob_workspace_bytes(self, p):
        return 0

    def _note(self, p, x, m):
        self.calls.append((p.rows, p.width, p.row_stride, p.mask_row_stride, x, m))
        return 0

    def mkg_logprob_forward(self, p, x, m, *rest):
        return self._note(p, x, m)

    def mkg_logprob_backward(self, p, x, m, *rest):
        return self._note(p, x, m)


def test_the_backward_reads_what_saved_tensor_hooks_hand_back(monkeypatch):
    """Its strides are those of the tensors that arrive: hooks that pack a copy return a slice as a contiguous
    tensor.  Tensors of another type or shape are refused."""
    import contextlib

    from minikg_dev_b200 import logprobs as L
    lib = Recorder()
    monkeypatch.setattr(N, "load", lambda: lib)
    monkeypatch.setattr(N, "on_device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(N, "stream_handle", lambda d=None: 0)
    monkeypatch.setattr(N, "error_word", lambda d: torch.zeros(1, dtype=torch.int32))
    x = torch.randn(6, 128)[:, :100].detach().requires_grad_(True)
    m = (torch.rand(6, 160) < 0.5)[:, 20:120].view(torch.uint8)
    t = torch.zeros(6, 2, dtype=torch.int64)
    arrived = []

    def unpack(v):
        arrived.append(v)
        return v

    def packed(copy):
        lib.calls.clear()
        arrived.clear()
        with torch.autograd.graph.saved_tensors_hooks(copy, unpack):
            out = L._TargetLogprobs.apply(x, t, m, 1.0, 3)
        out[0].sum().backward()
        return lib.calls

    for copy, strides in ((lambda v: v, (128, 160)), (lambda v: v.clone(memory_format=torch.contiguous_format), (100, 100)),
                          (lambda v: v.t().contiguous().t() if v.dim() == 2 else v, (100, 100))):
        first, second = packed(copy)
        assert first[2:4] == (128, 160) and second[2:4] == strides
        assert second[:2] == (6, 100)
        if strides == (128, 160):
            assert second[4:] == first[4:]
    for change in (torch.Tensor.double, lambda v: v[:3], lambda v: v.reshape(-1)):
        with pytest.raises(RuntimeError, match="saved"):
            packed(lambda v: change(v) if v.shape == (6, 100) and v.dtype == torch.float32 else v)
        with pytest.raises(RuntimeError, match="saved"):
            packed(lambda v: change(v) if v.dtype == torch.uint8 else v)
    with pytest.raises(RuntimeError, match="saved"):
        packed(lambda v: v.int() if v.dtype == torch.int64 and v.shape == (6, 2) else v)


@gpu
@pytest.mark.parametrize("rows, width", ((7, 100), (3, 5000), (4099, 700), (2, 70001)))
@pytest.mark.parametrize("masked", (False, True))
def test_gradients_under_saved_tensor_hooks(rows, width, masked):
    """Sliced logits and masks under hooks that copy: the same bits as without hooks."""
    g = torch.Generator(device="cuda").manual_seed(width)
    wide = torch.randn(rows, width + 28, generator=g, device="cuda")
    on = (torch.rand(rows, width + 60, generator=g, device="cuda") < 0.7)[:, 3:3 + width] if masked else None
    t = torch.randint(0, width, (rows, 2), generator=g, device="cuda")
    ups = [torch.randn(sh, generator=g, device="cuda") for sh in ((rows, 2), (rows,), (rows,), (rows, 5))]
    grads = []
    for hooks in (None, (lambda v: v.clone(memory_format=torch.contiguous_format), lambda v: v),
                  (lambda v: (v.device, v.cpu()), lambda v: v[1].to(v[0]))):
        leaf = wide.detach().requires_grad_(True)
        x = leaf[:, 5:5 + width]
        if hooks:
            with torch.autograd.graph.saved_tensors_hooks(*hooks):
                out = target_logprobs(x, t, 0.9, on, 5)
        else:
            out = target_logprobs(x, t, 0.9, on, 5)
        grads.append(torch.autograd.grad([out.logprobs, out.entropy, out.lse, out.top_logprobs], leaf, ups)[0])
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])


def test_forward_mode_tangents_are_refused():
    """There is no forward-mode derivative: a tangent is not dropped in silence."""
    import torch.autograd.forward_ad as forward_ad

    from minikg_dev_b200.decode import tail_logprobs
    x, t = torch.rand(3, 8) + 0.5, torch.zeros(3, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: target_logprobs(dual, t), lambda: tail_logprobs(dual, t)):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward"):
                call()


@gpu
def test_forward_mode_around_other_tensors():
    """Inside a dual level, logits without a tangent are read as ever."""
    import torch.autograd.forward_ad as forward_ad
    x, t = torch.randn(3, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    want = target_logprobs(x, t)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert torch.equal(target_logprobs(x, t).logprobs, want.logprobs)
        with pytest.raises(NotImplementedError, match="forward"):
            target_logprobs(dual, t)


@gpu
def test_outputs_without_gradients_are_tensors_of_their_own():
    """Changing one in place leaves a graph that saved another as it is, and none keeps the others' memory."""
    x, t = torch.randn(5, 300, device="cuda"), torch.zeros(5, 2, dtype=torch.int64, device="cuda")
    w = torch.ones(5, 2, device="cuda", requires_grad=True)
    out = target_logprobs(x, t, topk=4)
    want = out.logprobs.clone()
    loss = (w * out.logprobs).sum()
    for o in (out.entropy, out.lse, out.top_logprobs):
        o.zero_()
    loss.backward()
    assert torch.equal(w.grad, want)
    parts = [out.logprobs, out.entropy, out.lse, out.top_ids, out.top_logprobs]
    assert len({o.untyped_storage().data_ptr() for o in parts}) == 5 and not any(o._is_view() for o in parts)


@gpu
def test_lazily_negated_logits_and_gradients():
    """Tensors that torch negates when they are read (imaginary parts of conjugates): single elements count
    as contiguous and arrive as they are in memory."""
    z = torch.complex(torch.randn(4, device="cuda"), torch.randn(4, device="cuda"))
    t = torch.zeros(4, dtype=torch.int64, device="cuda")
    x = z.conj().imag[:, None]
    assert x.is_neg()
    assert torch.equal(target_logprobs(x, t).lse, -z.imag)
    assert torch.equal(target_logprobs(x[:1], t[:1], topk=1).lse, -z.imag[:1])
    whole = torch._neg_view(torch.randn(3, 50, device="cuda"))
    t = torch.ones(3, dtype=torch.int64, device="cuda")
    want = target_logprobs(whole.resolve_neg(), t, topk=3)
    for a, b in zip(target_logprobs(whole, t, topk=3), want):
        assert torch.equal(a, b)
    leaf = torch.randn(1, 50, device="cuda", requires_grad=True)
    grads = []
    for up in (torch._neg_view(torch.full((1,), 0.5, device="cuda")), torch.full((1,), -0.5, device="cuda")):
        out = target_logprobs(leaf, t[:1], topk=1)
        grads += [torch.autograd.grad(o, leaf, up.view(o.shape), retain_graph=True)[0]
                  for o in (out.logprobs, out.entropy, out.lse, out.top_logprobs)]
    for a, b in zip(grads[:4], grads[4:]):
        assert torch.equal(a, b) and bool(a.any())
    neg = whole.detach().requires_grad_(True)
    pos = whole.detach().resolve_neg().clone().requires_grad_(True)
    ga, gb = (torch.autograd.grad(target_logprobs(v, t).logprobs.sum(), v)[0] for v in (neg, pos))
    assert torch.equal(ga, gb)


@gpu
@pytest.mark.parametrize("rows, width", ((3, 1789), (4100, 1789), (4100, 97), (5, 14013), (4100, 2851), (2, 3000017), (1, 4594485)))
def test_equal_columns_share_the_gradient(rows, width):
    """p is 1 / width for equal logits.  Every power is 1 and the sum a whole number below 2^24, so both are
    exact; the reciprocal, the upstream gradient's product and p itself are rounded once each: 4 u, with one u
    in hand for the scale of tau.  A logarithm of the sum in fp32 in between would cost up to 11 u (half
    a step of log2 s, times ln 2) on every column alike."""
    x = torch.full((rows, width), 1.5, device="cuda", requires_grad=True)
    t = torch.zeros((rows, 1), dtype=torch.int64, device="cuda")
    out = target_logprobs(x, t)
    grad, = torch.autograd.grad(out.lse, x, torch.ones(rows, device="cuda"))
    assert float((grad.double() * width - 1).abs().max()) <= 4 * U
    out = target_logprobs(x, t)
    grad, = torch.autograd.grad(out.logprobs, x, torch.ones(rows, 1, device="cuda"))
    assert float((grad[:, 1:].double() * width + 1).abs().max()) <= 4 * U
    assert float((grad[:, 0].double() - (1 - 1 / width)).abs().max()) <= 4 * U


def test_a_trained_temperature_is_refused():
    """tau is a number: a tensor that asks for its gradient, or has a tangent, would silently get none."""
    import torch.autograd.forward_ad as forward_ad
    x, t = torch.rand(3, 8), torch.zeros(3, dtype=torch.int64)
    tau = torch.tensor(0.7, requires_grad=True)
    with pytest.raises(NotImplementedError, match="tau"):
        target_logprobs(x, t, tau)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="tau"):
        target_logprobs(x, t, forward_ad.make_dual(torch.tensor(0.7), torch.tensor(1.0)))
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA tensor"):  # read as a number: the next check's turn
        target_logprobs(x, t, tau)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        target_logprobs(x, t, tau.detach())
