"""The recurrent policy's operators together, as a learner uses them: dense gates, the recurrence over padded episodes, logits, the
clipped policy loss, the gradients back through time and an AdamW step, against torch's float64 autograd of the same formulas on
the CPU; then acting step by step with the trained weights."""
import numpy as np
import pytest
import torch

import rl_gan_amd as R

pytestmark = pytest.mark.gpu

B, T, K, UNITS, ACTIONS = 5, 37, 12, 16, 8
LR, BETAS, EPS, DECAY = 1e-2, (0.9, 0.999), 1e-8, 0.01
LOSS = dict(clip=0.2, kl_coef=0.1, entropy_coef=0.01)


def _data(seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    lengths = torch.tensor([T, 0, 20, 1, T - 1], dtype=torch.int32)
    live = torch.arange(T)[None] < lengths[:, None]
    return dict(x=torch.randn(B, T, K, generator=g), state=torch.randn(B, UNITS, generator=g), starts=torch.rand(B, T, generator=g) < 0.1,
                lengths=lengths, live=live, actions=torch.where(live, torch.randint(0, ACTIONS, (B, T), generator=g), torch.tensor(-1)),
                old=torch.full((B, T), -2.0) + 0.1 * torch.randn(B, T, generator=g), ref=torch.full((B, T), -2.1),
                adv=torch.randn(B, T, generator=g), weights=live.float() / live.sum())


def _float64(d, w, wo, steps):
    """torch autograd in float64: the losses and the parameters after each step."""
    w, wo = w.double().cpu().clone().requires_grad_(), wo.double().cpu().clone().requires_grad_()
    opt = torch.optim.AdamW([w, wo], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
    losses, grads = [], []
    for _ in range(steps):
        gates = d["x"].double() @ w[:K * 2 * UNITS].view(K, 2 * UNITS) + w[K * 2 * UNITS:]
        f, s, hs = torch.sigmoid(gates[..., :UNITS]), d["state"].double(), []
        for t in range(T):
            p = torch.where(d["starts"][:, t, None], torch.zeros_like(s), s)
            new = f[:, t] * p + (1 - f[:, t]) * gates[:, t, UNITS:]
            on = d["live"][:, t, None]
            s = torch.where(on, new, s)
            hs.append(torch.where(on, new, torch.zeros_like(new)))
        logits = torch.stack(hs, 1) @ wo[:UNITS * ACTIONS].view(UNITS, ACTIONS) + wo[UNITS * ACTIONS:]
        lp = torch.log_softmax(logits, -1)
        a = d["actions"].clamp(min=0)[..., None]
        la = lp.gather(-1, a)[..., 0]
        r, q = (la - d["old"].double()).exp(), d["ref"].double() - la
        adv = d["adv"].double()
        row = -torch.minimum(r * adv, r.clamp(0.8, 1.2) * adv) + 0.1 * (q.exp() - q - 1) + 0.01 * (lp.exp() * lp).sum(-1)
        loss = (d["weights"].double() * row).sum()
        opt.zero_grad()
        loss.backward()
        losses.append(loss.item())
        grads.append((w.grad.clone(), wo.grad.clone()))
        opt.step()
    return losses, grads, (w.detach(), wo.detach())


@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps_and_acting(bits):
    d = _data(1)
    rng = np.random.RandomState(2)
    memory = R.GatedUnit(K, UNITS, rng=rng)
    head = R.DenseLayer(UNITS, ACTIONS, rng=rng)
    start = (memory.gates.canon.clone(), head.canon.clone())
    opt = R.AdamW([memory.gates.canon, head.canon], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=bits)
    c = {k: v.cuda() for k, v in d.items()}
    flat = lambda v: v.reshape(-1)
    steps = 3
    losses, grads = [], []
    for _ in range(steps):
        h, last = memory.forward(c["x"], c["state"], c["starts"], c["lengths"])
        rows = h.reshape(B * T, UNITS)
        logits = head.forward(rows, act=False)
        r = R.policy_loss(logits, flat(c["actions"]), flat(c["old"]), flat(c["adv"]), weights=flat(c["weights"]), ref_logp=flat(c["ref"]), **LOSS)
        dh = head.backward(rows, logits, r.dlogits, act=False)
        memory.backward(dh.view(B, T, UNITS), need_dx=False)
        losses.append(float(r.loss))
        grads.append((memory.gates.grad.clone(), head.grad.clone()))
        opt.step([memory.gates.grad, head.grad])
    ref_losses, ref_grads, ref_params = _float64(d, *start, steps)
    # the first pass sees the same parameters: products and sums of at most some hundred terms in fp32
    assert abs(losses[0] - ref_losses[0]) <= 1e-5 * max(1.0, abs(ref_losses[0]))
    for g, q in zip(grads[0], ref_grads[0]):
        q = q.numpy()
        assert np.abs(g.double().cpu().numpy() - q).max() <= 2e-5 * np.abs(q).max()
    assert all(np.isfinite(losses))
    if bits == 32:
        for k in range(1, steps):                                # later passes: what Adam's division leaves of the differences
            assert abs(losses[k] - ref_losses[k]) <= 1e-3 * max(1.0, abs(ref_losses[k]))
    # acting: one step at a time gives what the sequence pass gives
    h, last = memory.forward(c["x"], c["state"], c["starts"], None)
    state = c["state"].clone()
    for t in range(T):
        ht = memory.step(c["x"][:, t].contiguous(), state, c["starts"][:, t])
        assert (ht - h[:, t]).abs().max() <= 2e-5 * max(1.0, float(h.abs().max()))
    assert (state - last).abs().max() <= 2e-5 * max(1.0, float(last.abs().max()))


def test_captured_training_step():
    """A whole training step captured into a graph: every replay leaves the parameters that the same eager step leaves."""
    d = {k: v.cuda() for k, v in _data(3).items()}
    flat = lambda v: v.reshape(-1)

    def make():
        rng = np.random.RandomState(4)
        memory, head = R.GatedUnit(K, UNITS, rng=rng), R.DenseLayer(UNITS, ACTIONS, rng=rng)
        opt = R.AdamW([memory.gates.canon, head.canon], lr=LR)

        def step():
            h, _ = memory.forward(d["x"], d["state"], d["starts"], d["lengths"])
            rows = h.reshape(B * T, UNITS)
            logits = head.forward(rows, act=False)
            r = R.policy_loss(logits, flat(d["actions"]), flat(d["old"]), flat(d["adv"]), weights=flat(d["weights"]), ref_logp=flat(d["ref"]), **LOSS)
            memory.backward(head.backward(rows, logits, r.dlogits, act=False).view(B, T, UNITS), need_dx=False)
            opt.step([memory.gates.grad, head.grad])
            return r.loss
        return memory, head, step
    a, b = make(), make()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a[2]()
    stream.synchronize()
    b[2]()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        loss = a[2]()
    for _ in range(4):
        d["x"].mul_(0.9)
        graph.replay()
        want = b[2]()
        torch.cuda.synchronize()
        assert torch.equal(loss, want)
        assert torch.equal(a[0].gates.canon, b[0].gates.canon) and torch.equal(a[1].canon, b[1].canon)
