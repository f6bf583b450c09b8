"""The operators of policies over large action sets as a training program uses them: draw, log-probability with gradient,
clipping of the global gradient norm, on their own and inside PPO(fused_policy=True).  -m gpu."""
import math

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu


class _Policy(nn.Module):
    """a table of states, a hidden layer, two heads"""

    def __init__(self, states, actions, hidden=32):
        super().__init__()
        self.table = nn.Embedding(states, hidden)
        self.fc = nn.Linear(hidden, hidden)
        self.policy_head = nn.Linear(hidden, actions)
        self.value_head = nn.Linear(hidden, 1)

    def trunk(self, obs):
        return torch.tanh(self.fc(self.table(obs)))

    def policy(self, obs):
        return self.policy_head(self.trunk(obs))

    def value(self, obs):
        return self.value_head(self.trunk(obs))


def _objective(logp, entropy, old_logp, adv, live):
    ratio = torch.exp(logp - old_logp)
    surrogate = torch.minimum(ratio * adv, ratio.clamp(0.9, 1.1) * adv)
    return -((surrogate + 0.01 * entropy) * live).sum() / live.sum()


@pytest.mark.parametrize('A', [18, 3000, 20011])
def test_draw_learn_clip_step_against_float64(A, dev):
    """a padded batch of sequences: actions drawn with the actor's temperature and filters, three updates on them; every
    update's gradients, their norm and the clipped gradients against float64 on the CPU"""
    from parl_amd import ops
    torch.manual_seed(A)
    T = 0.8
    model = _Policy(50, A).to(dev)
    twin = _Policy(50, A).double()
    with torch.no_grad():
        model.policy_head.weight.mul_(20.0)   # a policy that has learnt something
    g = torch.Generator(device=dev).manual_seed(1)
    obs = torch.randint(0, 50, (6, 11), generator=g, device=dev)
    length = torch.tensor([11, 7, 1, 0, 11, 3], device=dev)
    live = torch.arange(11, device=dev).view(1, -1) < length.view(-1, 1)
    with torch.no_grad():
        logits = model.policy(obs)
        logits = logits.masked_fill(~live.unsqueeze(-1), float('-inf'))   # behind a sequence's end nothing can be taken
        u = torch.rand(6, 11, generator=g, dtype=torch.float64, device=dev)
        actions, old_logp = ops.logits_sample(logits, u, temperature=T, top_k=200, top_p=0.95)
    assert ((actions == -1) == ~live).all() and (old_logp[~live] == 0).all()
    adv = torch.randn(6, 11, generator=g, device=dev) * 3
    opt = torch.optim.Adam(model.parameters(), lr=3e-3)
    for update in range(3):
        opt.zero_grad()
        logp, entropy = ops.logits_log_prob(model.policy(obs), actions, temperature=T)
        _objective(logp, entropy, old_logp, adv, live.float()).backward()
        # the same in float64, with the same parameters
        twin.load_state_dict({k: v.double().cpu() for k, v in model.state_dict().items()})
        twin.zero_grad()
        z = torch.log_softmax(twin.policy(obs.cpu()) / T, -1)
        want_logp = z.gather(-1, actions.cpu().clamp(min=0).unsqueeze(-1)).squeeze(-1) * live.cpu()
        want_ent = -(z.exp() * z).sum(-1) * live.cpu()
        _objective(want_logp, want_ent, old_logp.double().cpu(), adv.double().cpu(), live.double().cpu()).backward()
        if update == 0:   # the actor's log-probabilities are the learner's
            # float32 logits of magnitude M = 16 or less through two matrix products: 2^-24 (33 M + A / 256 + 40) and the scale
            tol = 2.0**-24 * (33 * 16 + A / 256 + 40) * 2
            assert (logp - old_logp).abs().max() <= tol and (logp.double().cpu() - want_logp).abs().max() <= tol * 4
        learnt = [p for p in model.parameters() if p.grad is not None]   # the value head takes no part
        grads = [p.grad.clone() for p in learnt]
        wants = [p.grad for p in twin.parameters() if p.grad is not None]
        assert len(grads) == len(wants) == 5
        # A float32 gradient through the kernels, exp, tanh and the products: each element a sum of up to 66 rows or A terms of
        # relative error 2^-24 (A / 256 + 600) each (the logits' own error moves every probability); as norms
        for a, b in zip(grads, wants):
            bound = 2.0**-24 * (A / 256 + 600) * 4
            assert (a.double().cpu() - b).norm() <= bound * b.norm() + 1e-9
        norm = ops.clip_grad_norm_(model.parameters(), 0.05)
        want_norm = math.sqrt(sum(float(a.double().square().sum()) for a in grads))
        assert float(norm) == pytest.approx(want_norm, rel=2.0**-22)
        clip = min(1.0, 0.05 / (want_norm + 1e-6))
        for p, a in zip(learnt, grads):
            torch.testing.assert_close(p.grad, a * clip, rtol=2.0**-22, atol=1e-30)
        opt.step()


def test_log_prob_gradient_is_stale_proof_and_first_order(dev):
    from parl_amd import ops
    x = torch.randn(4, 300, device=dev, requires_grad=True)
    a = torch.zeros(4, dtype=torch.int64, device=dev)
    y = x * 1.0
    lp, _ = ops.logits_log_prob(y, a)
    with torch.no_grad():
        y.mul_(2.0)                      # what the backward pass would read is gone
    with pytest.raises(RuntimeError):
        lp.sum().backward()
    lp, ent = ops.logits_log_prob(x, a)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(lp.sum(), x, create_graph=True)
    # through the graph twice gives the same
    lp, ent = ops.logits_log_prob(x, a)
    g1, = torch.autograd.grad(lp.sum() + ent.sum(), x, retain_graph=True)
    g2, = torch.autograd.grad(lp.sum() + ent.sum(), x)
    assert torch.equal(g1, g2)
    with torch.no_grad():
        assert not ops.logits_log_prob(x, a)[0].requires_grad
    with torch.inference_mode():
        z = x.detach() * 1.0
        assert torch.equal(ops.logits_log_prob(z, a)[0], lp)
        ops.logits_sample(z, torch.zeros(4, dtype=torch.float64, device=dev))
        p = nn.Parameter(torch.zeros(3, device=dev))
        p.grad = torch.ones(3, device=dev)
        ops.clip_grad_norm_([p], 1.0)


def test_clip_bumps_the_version_of_what_it_writes(dev):
    """a gradient that a graph still needs is not replaced behind its back"""
    from parl_amd import ops
    p = nn.Parameter(torch.ones(5, device=dev))
    p.grad = torch.full((5, ), 2.0, device=dev)
    w = torch.ones(5, device=dev, requires_grad=True)
    y = (w * p.grad).sum()
    ops.clip_grad_norm_([p], 0.1)
    with pytest.raises(RuntimeError):
        y.backward()


@pytest.mark.parametrize('A', [6, 700, 9000])
def test_ppo_with_the_fused_policy_learns_what_the_framework_path_learns(A, dev):
    from parl_amd.algorithms import PPO
    import parl_amd as parl

    class Model(_Policy, parl.Model):
        pass

    def make(fused):
        torch.manual_seed(3)
        return PPO(Model(20, A), clip_param=0.2, value_loss_coef=0.5, entropy_coef=0.01, initial_lr=1e-2, eps=1e-5,
                   max_grad_norm=0.2, fused_policy=fused)

    one, two = make(True), make(False)
    g = torch.Generator(device=dev).manual_seed(5)
    obs = torch.randint(0, 20, (64, ), generator=g, device=dev)
    value, action, logp, ent = one.sample(obs)
    assert action.dtype == torch.int64 and action.shape == (64, ) and logp.shape == (64, ) and ent.shape == (64, )
    dist = torch.distributions.Categorical(logits=two.model.policy(obs))
    # float32 on both sides: sums of A terms, log-probabilities of a few units
    tol = 2.0**-24 * (A / 256 + 60) * 2 * (math.log(A) + 4)
    torch.testing.assert_close(logp, dist.log_prob(action).detach(), rtol=0, atol=tol)
    torch.testing.assert_close(ent, dist.entropy().detach(), rtol=0, atol=tol)
    assert torch.equal(one.predict(obs), two.predict(obs))
    adv = torch.randn(64, generator=g, device=dev)
    ret = torch.randn(64, generator=g, device=dev)
    before = [p.detach().clone() for p in one.model.parameters()]
    for p, q in zip(one.model.parameters(), two.model.parameters()):
        assert torch.equal(p, q)
    losses = [alg.learn(obs, action, value.view(-1), ret, logp, adv) for alg in (one, two)]
    for a, b in zip(*losses):
        assert a == pytest.approx(b, rel=1e-4, abs=tol)
    for p, q, b in zip(one.model.parameters(), two.model.parameters(), before):
        # the clipped gradients left in .grad agree as float32 sums do
        assert (p.grad - q.grad).norm() <= 2.0**-24 * (A / 256 + 600) * 4 * q.grad.norm() + 1e-9
        assert (p - b).abs().max() <= 1.01e-2    # Adam's first step is at most the learning rate


def test_ppo_refuses_a_fused_policy_over_continuous_actions():
    from parl_amd.algorithms import PPO
    import parl_amd as parl

    class Model(_Policy, parl.Model):
        pass

    with pytest.raises(AssertionError):
        PPO(Model(3, 4), continuous_action=True, fused_policy=True)


def _table_ppo(logits, values, fused, **kw):
    """PPO over a table: state s has the logits logits[s] and the value values[s]"""
    from parl_amd.algorithms import PPO
    import parl_amd as parl

    class Model(parl.Model):
        def __init__(self):
            super().__init__()
            self.logits = nn.Parameter(logits.clone())
            self.values = nn.Parameter(values.clone())

        def policy(self, obs):
            return self.logits[obs]

        def value(self, obs):
            return self.values[obs].unsqueeze(-1)

    args = dict(clip_param=0.2, value_loss_coef=0.5, entropy_coef=0.01, initial_lr=1e-2, eps=1e-5, max_grad_norm=0.2)
    return PPO(Model(), fused_policy=fused, **dict(args, **kw))


def _batch(alg, states, dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    obs = torch.arange(states, device=dev)
    value, action, logp, _ = alg.sample(obs)
    rand = lambda: torch.randn(states, generator=g, device=dev)  # noqa: E731
    return [obs, action, value.view(-1) + rand(), rand(), logp + 0.1 * rand(), rand()]


@pytest.mark.parametrize('A', [6, 700, 9000])
def test_ppo_says_that_a_policy_has_diverged(A, dev):
    """a row with NaN or +inf stops sample, predict and learn, as the NaN does without fused_policy; a row where nothing may be
    taken is action -1 in sample and predict alike"""
    from parl_amd import ops
    logits = torch.randn(6, A, device=dev)
    logits[1, A // 2] = float('nan')
    logits[2] = float('nan')
    logits[3, 0] = float('inf')
    logits[4] = float('-inf')
    alg, plain = (_table_ppo(logits, torch.zeros(6, device=dev), f) for f in (True, False))
    at = lambda *s: torch.tensor(s, device=dev)  # noqa: E731
    for s in (1, 2):
        for a in (alg, plain):
            with pytest.raises(ValueError):
                a.sample(at(0, s))
            with pytest.raises(ValueError):
                a.predict(at(s, 0))
    with pytest.raises(ValueError):
        alg.sample(at(0, 3, 5))
    with pytest.raises(ValueError):
        alg.predict(at(0, 3, 5))
    value, action, logp, entropy = alg.sample(at(0, 4, 5))
    assert int(action[1]) == -1 and float(logp[1]) == 0 and float(entropy[1]) == 0
    assert int(action[0]) >= 0 and int(action[2]) >= 0 and torch.isfinite(logp).all() and torch.isfinite(entropy).all()
    best = alg.predict(at(0, 4, 5))
    assert best.shape == (3, 1) and best.dtype == torch.int64
    assert best.view(-1).tolist() == [int(logits[0].argmax()), -1, int(logits[5].argmax())]
    z = torch.zeros(2, device=dev)
    for s in (1, 2, 3):
        before = [p.detach().clone() for p in alg.model.parameters()]
        with pytest.raises(ValueError):
            alg.learn(at(0, s), at(0, 1), z, z, z, torch.tensor([1.0, -1.0], device=dev))
        for p, b in zip(alg.model.parameters(), before):
            assert p.grad is None and torch.equal(p.detach().nan_to_num(7.0), b.nan_to_num(7.0))
    # a row of padding is not looked at, whatever it holds
    losses = alg.learn(at(0, 5, 1, 3), at(0, 1, -1, -1), *torch.zeros(3, 4, device=dev),
                       torch.tensor([1.0, -1.0, 0.0, 0.0], device=dev))
    assert all(math.isfinite(v) for v in losses)
    assert torch.isfinite(alg.model.logits[0]).all() and torch.isfinite(alg.model.values).all()
    assert ops.consume_device_errors() > 0   # the draws' flag is up as well


@pytest.mark.parametrize('A', [6, 700, 9000])
def test_ppo_refuses_actions_outside_the_set(A, dev):
    from parl_amd import ops
    ops.consume_device_errors()
    alg, plain = (_table_ppo(torch.randn(4, A, device=dev), torch.zeros(4, device=dev), f) for f in (True, False))
    before = [p.detach().clone() for p in alg.model.parameters()]
    z, adv = torch.zeros(2, device=dev), torch.tensor([1.0, -1.0], device=dev)
    for bad in (A, A + 5, -2):
        for a in (alg, plain):
            with pytest.raises(ValueError):
                a.learn(torch.tensor([0, 1], device=dev), torch.tensor([0, bad], device=dev), z, z, z, adv)
    for a in (alg, plain):
        with pytest.raises(ValueError):
            a.learn(torch.tensor([0, 1], device=dev), torch.tensor([0.0, 1.5], device=dev), z, z, z, adv)
    for p, b in zip(alg.model.parameters(), before):
        assert p.grad is None and torch.equal(p, b)
    alg.learn(torch.tensor([0, 1], device=dev), torch.tensor([0.0, 2.0], device=dev), z, z, z, adv)   # whole numbers in any type
    assert ops.consume_device_errors() == 0   # refused before any kernel saw them


@pytest.mark.parametrize('norm_adv', [True, False])
@pytest.mark.parametrize('clipped', [True, False])
@pytest.mark.parametrize('A', [6, 700])
def test_rows_of_action_minus_one_change_no_update(A, clipped, norm_adv, dev):
    """a batch, and the same one with rows of padding between whose returns, advantages and old values are anything: the same
    losses, gradients and parameters"""
    g = torch.Generator(device=dev).manual_seed(A)
    logits, values = torch.randn(40, A, generator=g, device=dev), torch.randn(40, generator=g, device=dev)
    one, two = (_table_ppo(logits, values, True, use_clipped_value_loss=clipped, norm_adv=norm_adv) for _ in range(2))
    batch = _batch(one, 24, dev)
    at = torch.arange(24, device=dev) + torch.arange(24, device=dev) // 2   # every third row is padding
    padded = []
    for i, t in enumerate(batch):
        p = torch.full((36, ), [30, -1, float('nan'), 1e30, float('nan'), float('-inf')][i], dtype=t.dtype, device=dev)
        p[at] = t
        padded.append(p)
    for _ in range(2):
        a, b = one.learn(*batch), two.learn(*padded)
        # the same numbers through the same operations, but for the order of sums over 24 rows
        assert a == pytest.approx(b, rel=24 * 2.0**-23, abs=24 * 2.0**-23)
        for p, q in zip(one.model.parameters(), two.model.parameters()):
            # one row of the batch for each row of the tables: a few products, the norm's factor
            torch.testing.assert_close(p.grad, q.grad, rtol=2.0**-19, atol=1e-12)
            torch.testing.assert_close(p, q, rtol=2.0**-20, atol=1e-2 * 2.0**-15)
        assert (two.model.logits.grad[30] == 0).all() and float(two.model.values.grad[30]) == 0


def test_a_batch_of_nothing_but_padding_teaches_nothing(dev):
    alg = _table_ppo(torch.randn(4, 9, device=dev), torch.zeros(4, device=dev), True)
    obs, none = torch.arange(4, device=dev), torch.full((4, ), -1, device=dev)
    x = torch.full((4, ), float('nan'), device=dev)
    assert alg.learn(obs, none, x, x, x, x) == (0.0, 0.0, 0.0)
    for p in alg.model.parameters():
        assert (p.grad == 0).all() and torch.isfinite(p).all()


def test_one_decision_among_padding_is_learnt_from(dev):
    """one advantage has no deviation to be divided by: it is its own mean, so it counts as 0 there"""
    alg = _table_ppo(torch.randn(4, 9, device=dev), torch.zeros(4, device=dev), True)
    obs, a = torch.arange(4, device=dev), torch.tensor([-1, 3, -1, -1], device=dev)
    z = torch.zeros(4, device=dev)
    losses = alg.learn(obs, a, z, z + 1, z, z + 5)
    assert all(math.isfinite(v) for v in losses) and losses[0] == pytest.approx(0.5) and losses[1] == 0
    assert float(alg.model.values[1]) != 0 and all(torch.isfinite(p).all() for p in alg.model.parameters())


def test_ppo_sample_in_a_graph_marks_what_it_cannot_raise(dev):
    """a captured call cannot look at its results: the row of a diverged policy has no log-probability and no entropy"""
    from parl_amd import ops
    logits = torch.randn(4, 300, device=dev)
    alg = _table_ppo(logits, torch.zeros(4, device=dev), True)
    obs = torch.arange(4, device=dev)
    alg.sample(obs)
    alg.predict(obs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, action, logp, entropy = alg.sample(obs)
        best = alg.predict(obs)
    for bad in (False, True, False):
        with torch.no_grad():
            alg.model.logits.copy_(logits)
            if bad:
                alg.model.logits[2, 7] = float('nan')
        graph.replay()
        torch.cuda.synchronize()
        row = torch.tensor([False, False, bad, False], device=dev)
        assert torch.equal(torch.isnan(logp), row) and torch.equal(torch.isnan(entropy), row)
        assert torch.equal(action == -1, row) and torch.equal(best.view(-1) == -1, row)
    assert ops.consume_device_errors() > 0


@pytest.mark.parametrize('fused', [True, False])
@pytest.mark.parametrize('A', [6, 700, 9000])
def test_ppo_moves_every_parameter_by_its_clipped_gradient(A, fused, dev):
    """Adam's first step from the gradients that learn() leaves: lr g / (|g| + eps)"""
    alg = _table_ppo(torch.randn(20, A, device=dev), torch.randn(20, device=dev), fused)
    batch = _batch(alg, 20, dev)
    before = [p.detach().double().clone() for p in alg.model.parameters()]
    alg.learn(*batch)
    for p, b in zip(alg.model.parameters(), before):
        g = p.grad.double()
        step = 1e-2 * g / (g.abs() + 1e-5)
        # float32: the parameter's own rounding, and a few roundings of the step (the square root of g^2 and its sum with
        # eps, the two bias corrections); squares under the normal range leave a gradient of less than 1e-19 without effect
        tol = 2.0**-23 * b.abs() + 2.0**-18 * step.abs() + 1e-2 * 1e-19 / 1e-5
        assert ((p.double() - b + step).abs() <= tol).all()
        assert (p.double() - b).abs().max() > 1e-3


def test_old_values_that_no_loss_reads_may_be_missing(dev):
    alg = _table_ppo(torch.randn(6, 9, device=dev), torch.zeros(6, device=dev), True, use_clipped_value_loss=False)
    obs, action, _, ret, logp, adv = _batch(alg, 6, dev)
    for a in (action, torch.where(obs == 3, -1, action)):
        assert all(math.isfinite(v) for v in alg.learn(obs, a, None, ret, logp, adv))


def test_actions_in_any_memory_order(dev):
    """a batch [T, B] that lies transposed, with padding: as the flat one"""
    logits = torch.randn(12, 9, device=dev)
    one, two = (_table_ppo(logits, torch.zeros(12, device=dev), True) for _ in range(2))
    obs, action, value, ret, logp, adv = _batch(one, 12, dev)
    action[5] = -1
    flat = one.learn(obs, action, value, ret, logp, adv)
    t = lambda x: x.view(3, 4).t().contiguous().t()  # noqa: E731
    assert not t(action).is_contiguous()
    assert two.learn(t(obs), t(action), t(value), t(ret), t(logp), t(adv)) == pytest.approx(flat, rel=12 * 2.0**-23)
