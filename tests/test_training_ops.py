"""Log probabilities and AdamW where the package uses them: rule bodies read from a producer, tails
ranked by raw scores, an update inside the captured training step, and a training run of all of it."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from minikg_dev_b200 import _native as N
from minikg_dev_b200 import rules
from minikg_dev_b200.decode import tail_logprobs
from minikg_dev_b200.optim import AdamW

gpu = pytest.mark.gpu
U = 2.0 ** -24


class Producer(torch.nn.Module):
    """The producer attributes of the reference's rule model (drum.py:303-330)."""

    def __init__(self, R=7, H=16, K=2, L=3, tau=0.8, device="cuda"):
        super().__init__()
        n = 2 * R + 1
        self.relation_count, self.step, self.rules, self.tau_1 = R, K, L, tau
        self.emb = torch.nn.Parameter(torch.randn(n, H))
        self.lstm = torch.nn.ModuleList(torch.nn.LSTM(H, H, 1, bidirectional=True) for _ in range(L))
        self.linear = torch.nn.Linear(2 * H, n)
        self.to(device)

    def exact(self):
        """The same model in float64 on the CPU."""
        twin = Producer(self.relation_count, self.emb.shape[1], self.step, self.rules, self.tau_1, "cpu").double()
        twin.load_state_dict({k: v.double().cpu() for k, v in self.state_dict().items()})
        return twin

    def logits64(self, rel):
        """drum.py:429-438 with torch's own LSTM: [B, K, L, n]."""
        seq = torch.stack([self.emb[rel]] * self.step + [self.emb[-1].expand(len(rel), -1)])
        out = [self.linear(m(seq)[0][:self.step]) for m in self.lstm]
        return torch.stack(out, 2).transpose(0, 1)


def bodies_of(rel, S, K, n, seed):
    g = torch.Generator().manual_seed(seed)
    b = torch.randint(0, n, (len(rel), S, K), generator=g)
    if S > 1:
        b[0, -1] = -1      # padding
        b[1, 0, 0] = -1    # a hop left out
        b[2, 1] = b[2, 0]  # the same body twice
    return b


def body_logprobs64(logits, bodies, tau):
    lp = torch.log_softmax(logits / tau, -1)                   # [B, K, L, n]
    at = bodies.clamp_min(0).permute(0, 2, 1)[:, :, None, :]   # [B, K, 1, S]
    got = lp.gather(3, at.expand(-1, -1, logits.shape[2], -1))
    got = torch.where(bodies.permute(0, 2, 1)[:, :, None, :] < 0, 0.0, got)
    return got.sum(1).transpose(1, 2), -(lp.exp() * lp).sum(-1), lp


@gpu
@pytest.mark.parametrize("B, S", ((5, 1), (40, 3), (6, 700)))
def test_rule_logprobs(B, S):
    """Values and every parameter's gradient; S = 700 needs several calls for a relation's bodies."""
    torch.manual_seed(B)
    model = Producer()
    twin = model.exact()
    n, K = 2 * model.relation_count + 1, model.step
    rel = torch.randint(0, 4, (B,))
    bodies = bodies_of(rel, S, K, n, seed=S)
    out = rules.rule_logprobs(model, rel.cuda(), bodies.cuda(), topk=4)
    lp, ent, logp = body_logprobs64(twin.logits64(rel), bodies, model.tau_1)
    # the producer's logits carry 1e-5 of themselves (tests of the producer); log p is logits / tau twice over
    tol = dict(rtol=1e-5, atol=4e-5)
    torch.testing.assert_close(out.logprobs.double().cpu(), lp.detach(), **tol)
    torch.testing.assert_close(out.entropy.double().cpu(), ent.detach(), **tol)
    assert out.top_channels.shape == (B, K, model.rules, 4)
    torch.testing.assert_close(out.top_logprobs.double().cpu(), logp.detach().topk(4, -1).values, **tol)
    w = torch.randn(B, S, model.rules, dtype=torch.float64)
    ((out.logprobs * w.float().cuda()).sum() + 0.1 * out.entropy.sum()).backward()
    ((lp * w.float().double()).sum() + 0.1 * ent.sum()).backward()
    N.raise_device_errors(out.logprobs.device)
    for (name, p), (_, q) in zip(model.named_parameters(), twin.named_parameters()):
        scale = float(q.grad.abs().max())
        # backpropagation through K + 1 LSTM steps: the bar of the producer's own tests
        torch.testing.assert_close(p.grad.double().cpu(), q.grad, rtol=1e-4, atol=1e-5 * scale, msg=lambda m: f"{name}: {m}")


@gpu
def test_rule_logprobs_of_other_producers_and_weights():
    """A model with its own logits; the log of what the hop loop's rule weights give a path."""
    model = Producer()
    rel = torch.tensor([1, 2, 1], device="cuda")
    bodies = bodies_of(rel, 2, 2, 15, seed=0).cuda()

    class Own:
        tau_1 = model.tau_1

        def build_rule_logits(self, r):
            return rules.build_rule_logits(model, r)

    a, b = rules.rule_logprobs(model, rel, bodies), rules.rule_logprobs(Own(), rel, bodies)
    torch.testing.assert_close(a.logprobs, b.logprobs, rtol=4 * U, atol=4 * U)
    w = rules.rule_weights(model, rel)  # [K, B, L, n]
    path = w[0, 1, :, bodies[1, 1, 0]] * w[1, 1, :, bodies[1, 1, 1]]
    torch.testing.assert_close(a.logprobs[1, 1].exp(), path, rtol=1e-5, atol=0)


@gpu
def test_rule_logprobs_refusals():
    model, rel = Producer(), torch.tensor([1, 2], device="cuda")
    for bad, error in ((torch.zeros(2, 2, dtype=torch.int64), ValueError), (torch.zeros(3, 1, 2, dtype=torch.int64), ValueError),
                       (torch.zeros(2, 1, 3, dtype=torch.int64), ValueError), (torch.zeros(2, 1, 2), TypeError)):
        with pytest.raises(error):
            rules.rule_logprobs(model, rel, bad.cuda())
    rules.rule_logprobs(model, rel, torch.full((2, 1, 2), 15, device="cuda"))  # one past the last channel
    with pytest.raises(RuntimeError, match="target"):
        N.raise_device_errors(rel.device)


@gpu
@pytest.mark.parametrize("sparse", (False, True))
def test_tail_logprobs(sparse):
    g = torch.Generator(device="cuda").manual_seed(1)
    raw = torch.rand(6, 5000, generator=g, device="cuda") * (torch.rand(6, 5000, generator=g, device="cuda") < 0.2)
    raw[3] = 0  # a query without an answer
    tails = torch.randint(0, 5000, (6, 4), generator=g, device="cuda")
    tails[:, 0] = raw.argmax(1)
    tails[0, 3] = -1
    mask = torch.rand(6, 5000, generator=g, device="cuda") < 0.8
    mask[torch.arange(6), tails[:, 0]] = True
    leaf = (raw.to_sparse_coo() if sparse else raw.clone()).requires_grad_(True)
    out = tail_logprobs(leaf, tails, mask, topk=5)
    d = (raw * mask).double().requires_grad_(True)
    total = d.sum(1, keepdim=True)
    p = torch.where(total > 0, d / torch.where(total > 0, total, 1.0), 0.0)
    want = torch.where(tails < 0, 0.0, p.gather(1, tails.clamp_min(0)).log())
    # log of the scores, of their sum, and what exp of the first gives back: 2^-20 of log p's size of 10
    torch.testing.assert_close(out.logprobs.double(), want.detach(), rtol=2.0 ** -19, atol=2.0 ** -18)
    best = torch.sort(p.detach(), dim=1, descending=True, stable=True)
    assert torch.equal(out.top_ids[0], best.indices[0, :5]) and (out.top_ids[3] == -1).all()
    assert (out.logprobs[3] == -math.inf).all() and out.entropy[3] == 0
    keep = [0, 1, 2, 4, 5]
    out.logprobs[keep, 0].sum().backward()
    # autograd of the gathered logs would multiply 0 by the infinite slope of log 0 at the other tails
    (d.gather(1, tails[:, :1])[keep].log() - total[keep].log()).sum().backward()
    got = leaf.grad.to_dense() if sparse else leaf.grad
    where = (raw > 0) & mask
    assert torch.isfinite(got).all() and not got[~where].any()
    torch.testing.assert_close(got.double()[where], d.grad[where], rtol=2.0 ** -16, atol=0)


def test_tail_logprobs_refusals():
    raw, tails = torch.ones(2, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError):
        tail_logprobs(raw[0], tails)
    with pytest.raises(TypeError):
        tail_logprobs(raw, tails, torch.ones(2, 4))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        tail_logprobs(raw, tails)


@gpu
def test_tail_logprobs_keep_a_nan_in_sight():
    raw = torch.rand(2, 300, device="cuda")
    raw[0, 7] = math.nan
    out = tail_logprobs(raw, torch.tensor([1, 1], device="cuda"))
    assert torch.isnan(out.logprobs[0]) and torch.isfinite(out.logprobs[1])


def small_graph():
    from minikg_dev_b200.graph import DeviceGraph
    from minikg_dev_b200.synth import sample_graph
    kg = sample_graph(300, 5, 3000, (("rel", ("zipf", 1.0)), ("head", (1.2, 3.0)), ("tail", (1.0, 2.0))), seed=3)
    up = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    return kg, DeviceGraph.from_triples(up(kg.head), up(kg.rel), up(kg.tail), kg.num_entities, kg.num_relations)


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_update_inside_the_captured_step(bits):
    """Each replay's update is AdamW's on that replay's gradients, capturing takes no step, and the new
    weights are what the next replay runs with."""
    from minikg_dev_b200.proof import ProofRunner
    kg, g = small_graph()
    B, L, K, E, n = 4, 2, 2, kg.num_entities, 2 * kg.num_relations + 1
    torch.manual_seed(0)
    heads = torch.randint(0, E, (B,), device="cuda")
    w = torch.nn.Parameter(torch.softmax(torch.randn(K, B, L, n, device="cuda"), -1))
    scores = torch.nn.Parameter(torch.rand(kg.num_triples, device="cuda"))
    out, msgs = torch.zeros(B, E, device="cuda"), torch.zeros(K, dtype=torch.int64, device="cuda")
    grad_out = torch.randn(B, E, device="cuda")
    gw, ge = torch.zeros_like(w), torch.zeros_like(scores)
    w.grad, scores.grad = gw, ge
    lr = torch.tensor(0.01, device="cuda")
    opt = AdamW([{"params": [w], "lr": lr}, {"params": [scores], "lr": 0.02}], weight_decay=0.1, state_bits=bits)
    before = w.detach().clone(), scores.detach().clone()
    graph = ProofRunner(g, B, L, K).capture(heads, w, out, msgs, grad_out, scores, gw, ge, optimizer=opt)
    assert torch.equal(w, before[0]) and torch.equal(scores, before[1])
    assert [int(opt.state[p]["step"]) for p in (w, scores)] == [0, 0]
    twins = [torch.nn.Parameter(x.clone()) for x in before]
    ref = AdamW([{"params": twins[:1], "lr": 0.01}, {"params": twins[1:], "lr": 0.02}], weight_decay=0.1, state_bits=bits)
    eager = ProofRunner(g, B, L, K)
    for i in range(3):
        rate = float(torch.tensor(0.01 / (i + 1)))
        lr.fill_(rate)
        ref.param_groups[0]["lr"] = rate
        g.set_edge_factor(None, twins[1], True, 1.0)
        want, _ = eager.forward(heads, twins[0])  # with the weights before this replay's update
        graph.replay()
        torch.cuda.synchronize()
        torch.testing.assert_close(out, want, rtol=1e-5, atol=1e-6)
        assert gw.abs().max() > 0 and ge.abs().max() > 0
        twins[0].grad, twins[1].grad = gw.clone(), ge.clone()
        ref.step()
        assert torch.equal(w, twins[0]) and torch.equal(scores, twins[1])
    assert not torch.equal(w, before[0]) and int(opt.state[w]["step"]) == 3


@gpu
def test_capture_refuses_other_optimizers():
    from minikg_dev_b200.proof import ProofRunner
    kg, g = small_graph()
    B, L, K, n = 2, 1, 1, 2 * kg.num_relations + 1
    w = torch.nn.Parameter(torch.rand(K, B, L, n, device="cuda"))
    scores = torch.rand(kg.num_triples, device="cuda")
    args = (torch.zeros(B, dtype=torch.int64, device="cuda"), w, torch.zeros(B, kg.num_entities, device="cuda"),
            torch.zeros(K, dtype=torch.int64, device="cuda"), torch.zeros(B, kg.num_entities, device="cuda"), scores)
    gw = torch.zeros_like(w)
    runner = ProofRunner(g, B, L, K)
    with pytest.raises(ValueError, match="AdamW"):
        runner.capture(*args, gw, optimizer=torch.optim.AdamW([w]))
    with pytest.raises(ValueError, match="gradient"):
        runner.capture(*args, gw, optimizer=AdamW([w]))  # no gradient set
    w.grad = torch.zeros_like(w)
    with pytest.raises(ValueError, match="gradient"):
        runner.capture(*args, gw, optimizer=AdamW([w]))  # another buffer
    other = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    w.grad, other.grad = gw, torch.zeros(5, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        runner.capture(*args, gw, optimizer=AdamW([w, other]))


@gpu
@pytest.mark.parametrize("bits", (32, 8))
def test_training_run(bits):
    """A producer trained towards given rule bodies: log probabilities, their gradient and the update, five
    steps, against the same in float64 (torch's LSTM, log_softmax and the update's definition)."""
    torch.manual_seed(7)
    model = Producer()
    twin = model.exact()
    rel = torch.randint(0, model.relation_count, (32,))
    bodies = bodies_of(rel, 2, model.step, 2 * model.relation_count + 1, seed=3)
    lr, eps, wd, steps = 1e-2, 1e-2, 0.05, 5
    opt = AdamW(model.parameters(), lr=lr, eps=eps, weight_decay=wd, state_bits=bits)
    ref = torch.optim.AdamW(twin.parameters(), lr=lr, eps=eps, weight_decay=wd, foreach=False)
    biggest = 0.0
    for _ in range(steps):
        opt.zero_grad()
        out = rules.rule_logprobs(model, rel.cuda(), bodies.cuda())
        loss = -out.logprobs.logsumexp(2).mean() - 0.01 * out.entropy.mean()
        loss.backward()
        opt.step()
        ref.zero_grad()
        lp, ent, _ = body_logprobs64(twin.logits64(rel), bodies, model.tau_1)
        want = -lp.logsumexp(2).mean() - 0.01 * ent.mean()
        want.backward()
        ref.step()
        if bits == 32:
            assert abs(float(loss.detach()) - float(want.detach())) < 1e-4 * abs(float(want.detach()))
        biggest = max(biggest, max(float(p.grad.abs().max()) for p in twin.parameters()))
    assert torch.isfinite(loss)
    # One step moves a parameter by lr m / (sqrt(v) + eps).  A gradient off by d moves that by at most
    # 2 lr d / eps, and the gradients are off by 1e-4 of the largest.  Held in 8 bits, m is off by 2^-4 and
    # sqrt(v) by 2^-5 of themselves from the second step on; both meet a bias correction of at most
    # (1 - b1) / (1 - b1^2) and the quotient is at most sqrt((1 - b1)^2 / (1 - b2)) < 3.2, so a step is off by
    # lr * 3.2 * (2^-4 + 2^-5) and the errors of m carry on with b1 = 0.9: below 10 times one of them.
    tol = steps * 2 * lr * 1e-4 * biggest / eps
    if bits == 8:
        tol += steps * lr * 3.2 * (2.0 ** -4 + 2.0 ** -5)
    for (name, p), (_, q) in zip(model.named_parameters(), twin.named_parameters()):
        assert float((p.double().cpu() - q).abs().max()) <= tol, name
    assert {int(opt.state[p]["step"]) for p in model.parameters()} == {steps}


@gpu
def test_a_captured_update_keeps_what_it_reads():
    """A rate's tensor that is taken out of the optimizer after the capture, and moments that a new group
    moves, are not handed to others while the graph is there.  Nothing is replayed."""
    from minikg_dev_b200.proof import ProofRunner
    kg, g = small_graph()
    B, L, K, E, n = 2, 1, 1, kg.num_entities, 2 * kg.num_relations + 1
    w = torch.nn.Parameter(torch.rand(K, B, L, n, device="cuda"))
    w.grad = torch.zeros_like(w)
    opt = AdamW([w], lr=torch.full((1,), 0.01, device="cuda"))
    graph = ProofRunner(g, B, L, K).capture(
        torch.zeros(B, dtype=torch.int64, device="cuda"), w, torch.zeros(B, E, device="cuda"),
        torch.zeros(K, dtype=torch.int64, device="cuda"), torch.zeros(B, E, device="cuda"),
        torch.rand(kg.num_triples, device="cuda"), w.grad, optimizer=opt)
    old = [(b.data_ptr(), b.numel(), b.dtype) for b in (*opt._buffers.values(), opt.param_groups[0]["lr"])]
    opt.param_groups[0]["lr"] = 0.5
    opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(300, device="cuda"))]})
    others = [torch.empty(k, dtype=t, device="cuda") for _, k, t in old for _ in range(200)]
    assert not {x.data_ptr() for x in others} & {at for at, _, _ in old}
    del graph


@gpu
def test_tail_logprobs_of_scores_below_the_least_normal_number():
    """They are candidates like others, at their own weight.  log of a score down to 2^-149 is at most 104
    in size: half a step of fp32 there is 2^-18, and its own error twice that; two of them, and the sum's
    log, make a log probability: 2^-15."""
    raw = torch.tensor([[1e-40, 3e-40, 0.0, 6e-40], [8e-39, 4e-39, 0.0, 0.0], [2e-38, 8e-39, 0.5, 0.0], [0.0, 1e-44, 0.0, 0.0]],
                       device="cuda", requires_grad=True)
    tails = torch.tensor([[0, 1, 3], [0, 1, 2], [0, 1, 2], [0, 1, -1]], device="cuda")
    out = tail_logprobs(raw, tails, topk=3)
    x = raw.detach().double().cpu()
    logp = torch.log(x / x.sum(1, keepdim=True))
    want = torch.where(tails.cpu() < 0, 0.0, logp.gather(1, tails.cpu().clamp_min(0)))
    assert torch.equal(out.logprobs.isinf().cpu(), want.isinf())
    fine = want.isfinite()
    assert float((out.logprobs.double().cpu() - want)[fine].abs().max()) <= 2.0 ** -15
    assert out.top_ids[0].tolist() == [3, 1, 0] and out.top_ids[1].tolist() == [0, 1, -1]
    # d log p_t / d raw_j = (j == t) / raw_j - 1 / sum over the candidates, 0 elsewhere
    grad, = torch.autograd.grad(out.logprobs[1, 0], raw)
    want = torch.tensor([1 / x[1, 0] - 1 / x[1].sum(), -1 / x[1].sum(), 0.0, 0.0], dtype=torch.float64)
    assert not grad[[0, 2, 3]].any()
    assert float((grad[1].double().cpu() - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max())


@gpu
def test_rule_logprobs_of_a_trained_temperature():
    """tau gets no gradient here: a temperature that asks for one is refused, a frozen one is read."""
    model = Producer()
    rel, bodies = torch.tensor([0, 1], device="cuda"), torch.zeros((2, 1, 2), dtype=torch.int64, device="cuda")
    want = rules.rule_logprobs(model, rel, bodies).logprobs
    model.tau_1 = torch.nn.Parameter(torch.tensor(0.8))
    with pytest.raises(NotImplementedError, match="tau"):
        rules.rule_logprobs(model, rel, bodies)
    model.tau_1.requires_grad_(False)
    torch.testing.assert_close(rules.rule_logprobs(model, rel, bodies).logprobs, want, rtol=4 * U, atol=16 * U)
