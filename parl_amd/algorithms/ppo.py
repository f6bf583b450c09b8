"""PPO — parl/algorithms/torch/ppo.py:27-206 (same constructor, same learn / sample / predict /
value contract; the Paddle twin parl/algorithms/paddle/ppo.py:28-216 has identical arithmetic).

What runs where: the model forward / backward, Normal / Categorical log-probabilities, the clipped
surrogate and Adam are PyTorch-ROCm; the per-minibatch advantage normalisation
`(adv - adv.mean()) / (adv.std() + 1e-8)` (ppo.py:124-127, unbiased std) is the HIP kernel
`parlhip_adv_normalize_f32` (advantages carry no gradient).  The GAE scan and the minibatch
gather that feed learn() live in parl_amd.storage.RolloutStorage.

`fused_policy=True` (discrete actions on the device) is for action sets the size of a vocabulary: log-probabilities,
entropies and their gradient (`ops.logits_log_prob`), the draw (`ops.logits_sample`, with uniforms of torch's generator) and
the clipping of the global gradient norm (`ops.clip_grad_norm_`) are the library's kernels instead of torch's
Categorical and clip_grad_norm_, which materialise several arrays of the logits' size.  The policy may return float32,
bfloat16 or float16 logits, and an action of -1 marks a row that is no decision: sample() gives it log-probability and
entropy 0, learn() takes its losses, their means and the advantages' normalisation over the other rows alone (one such row
counts with the advantage 0, none with losses of 0).  sample() and predict() give it to a row whose every logit is -inf.  A row with NaN or +inf is a
ValueError in sample(), predict() and learn(), as NaN is in Categorical; a call that is being captured into a graph
cannot look at its results, there the row gets action -1 and, from sample(), NaN for log-probability and entropy.
An action that is neither -1 nor one of the set is a ValueError in learn()."""
import torch
import torch.nn as nn
from torch.distributions import Categorical, Normal

from .. import ops
from ..core import Algorithm

__all__ = ['PPO']


class PPO(Algorithm):
    def __init__(self,
                 model,
                 clip_param=0.1,
                 value_loss_coef=0.5,
                 entropy_coef=0.01,
                 initial_lr=2.5e-4,
                 eps=1e-5,
                 max_grad_norm=0.5,
                 use_clipped_value_loss=True,
                 norm_adv=True,
                 continuous_action=False,
                 fused_policy=False):
        for m in ('value', 'policy'):  # check_model_method, parl/utils/utils.py:217-243
            assert callable(getattr(model, m, None)), '%s: model needs a `%s` method' % (self.__class__.__name__, m)
        # the argument checks of ppo.py:57-65
        assert isinstance(clip_param, float)
        assert isinstance(value_loss_coef, float)
        assert isinstance(entropy_coef, float)
        assert isinstance(initial_lr, float)
        assert isinstance(eps, float)
        assert isinstance(max_grad_norm, float)
        assert isinstance(use_clipped_value_loss, bool)
        assert isinstance(norm_adv, bool)
        assert isinstance(continuous_action, bool)
        assert isinstance(fused_policy, bool)
        assert not (fused_policy and continuous_action), 'fused_policy: discrete actions only'
        super(PPO, self).__init__(model)
        self.clip_param = clip_param
        self.value_loss_coef = value_loss_coef
        self.entropy_coef = entropy_coef
        self.max_grad_norm = max_grad_norm
        self.use_clipped_value_loss = use_clipped_value_loss
        self.norm_adv = norm_adv
        self.continuous_action = continuous_action
        self.fused_policy = fused_policy
        if torch.cuda.is_available():  # ppo.py:75-76
            self.model = model.to(torch.device('cuda'))
        self.optimizer = torch.optim.Adam(self.model.parameters(), lr=initial_lr, eps=eps)
        self.grad_hook = None  # parl_amd.dist.FlatGradAllReduce(model, average=True) for data-parallel learners

    def _dist(self, obs):
        if self.continuous_action:
            mean, std = self.model.policy(obs)
            return Normal(mean, std)
        return Categorical(logits=self.model.policy(obs))

    @staticmethod
    def _refuse(bad, rows, what='the policy has logits with NaN or +inf'):
        if bad:
            raise ValueError('PPO(fused_policy=True): %s in %d of %d rows' % (what, bad, rows))

    def _refuse_diverged(self, bad):
        """ValueError where `bad` holds anywhere (waits for the device, as Categorical's own checks do).  False if the call is
        being captured, so that nothing can be known."""
        if torch.cuda.is_current_stream_capturing():
            return False
        self._refuse(int(bad.sum()), bad.numel())
        return True

    def _fused_log_prob(self, obs, action):
        """log-probabilities and entropies, and the rows that are decisions (None: all are)"""
        logits, taken = self.model.policy(obs), action.to(torch.int64)
        outside = (taken < -1) | (taken >= logits.shape[-1]) | (taken != action)
        taken = taken.masked_fill(outside, -1)
        logp, entropy = ops.logits_log_prob(logits, taken)
        live = (taken >= 0).reshape(-1)
        n_outside, n_nan, n_live = torch.stack((outside.sum(), torch.isnan(logp).sum(), live.sum())).tolist()
        self._refuse(n_outside, live.numel(), 'actions that are none')
        self._refuse(n_nan, live.numel())
        return logp, entropy, None if n_live == live.numel() else live.nonzero().view(-1)

    def _losses(self, obs, action, old_value, ret, old_logp, adv):
        """the three terms of the PPO objective for one minibatch (ppo.py:104-148)"""
        rows = None   # where not all are decisions: those that are
        if self.fused_policy:
            logp, entropy, rows = self._fused_log_prob(obs, action)
            if rows is not None:
                logp, entropy, ret, old_logp, adv = (t.reshape(-1)[rows] for t in (logp, entropy, ret, old_logp, adv))
                if self.use_clipped_value_loss:
                    old_value = old_value.reshape(-1)[rows]
        else:
            dist = self._dist(obs)
            logp, entropy = dist.log_prob(action), dist.entropy()
        if self.continuous_action:  # independent Normal per action dimension
            logp, entropy = logp.sum(1), entropy.sum(1)
        if self.norm_adv:  # ppo.py:124-127 on the device kernel (unbiased std, + 1e-8); no gradient
            if self.fused_policy and adv.numel() == 1:   # it is its own mean, and there is no deviation
                adv = torch.zeros_like(adv)
            else:
                adv = ops.adv_normalize(adv.detach(), eps=1e-8).view_as(adv)
        mean = torch.sum if self.fused_policy and not adv.numel() else torch.mean   # of no decisions: 0
        eps = self.clip_param
        ratio = torch.exp(logp - old_logp)
        policy_loss = -mean(torch.minimum(ratio * adv, ratio.clamp(1.0 - eps, 1.0 + eps) * adv))
        value = self.model.value(obs).reshape(-1)
        if rows is not None:
            value = value[rows]
        if self.use_clipped_value_loss:
            clipped = old_value + (value - old_value).clamp(-eps, eps)
            value_loss = 0.5 * mean(torch.maximum((value - ret)**2, (clipped - ret)**2))
        else:
            value_loss = 0.5 * mean((ret - value)**2)
        return value_loss, policy_loss, mean(entropy)

    def learn(self, batch_obs, batch_action, batch_value, batch_return, batch_logprob, batch_adv, lr=None):
        """ppo.py:81-158: one clipped-surrogate update on a minibatch.  Returns
        (value_loss, action_loss, entropy_loss) as python floats."""
        value_loss, action_loss, entropy_loss = self._losses(batch_obs, batch_action, batch_value, batch_return,
                                                             batch_logprob, batch_adv)
        loss = value_loss * self.value_loss_coef + action_loss - entropy_loss * self.entropy_coef
        if lr:
            for group in self.optimizer.param_groups:
                group['lr'] = lr
        self._zero_grad()
        loss.backward()
        if self.grad_hook is not None:
            self.grad_hook(self.model)
        clip_grad_norm_ = ops.clip_grad_norm_ if self.fused_policy else nn.utils.clip_grad_norm_
        clip_grad_norm_(self.model.parameters(), self.max_grad_norm)
        self.optimizer.step()
        return value_loss.item(), action_loss.item(), entropy_loss.item()

    @torch.no_grad()
    def sample(self, obs):
        """ppo.py:160-187: (value, action, action_log_probs, action_entropy)"""
        value = self.model.value(obs)
        if self.fused_policy:
            logits = self.model.policy(obs)
            uniforms = torch.rand(logits.shape[:-1], dtype=torch.float64, device=logits.device)
            action, drawn = ops.logits_sample(logits, uniforms)
            log_probs, entropy = ops.logits_log_prob(logits, action)   # the learner's own: its first ratio is 1
            diverged = torch.isnan(drawn)
            if not self._refuse_diverged(diverged):
                log_probs, entropy = (t.masked_fill(diverged, float('nan')) for t in (log_probs, entropy))
            return value, action, log_probs, entropy
        dist = self._dist(obs)
        action = dist.sample()
        if self.continuous_action:
            return value, action, dist.log_prob(action).sum(1), dist.entropy().sum(1)
        return value, action, dist.log_prob(action), dist.entropy()

    @torch.no_grad()
    def predict(self, obs):
        """ppo.py:189-203: the mean action / the argmax of the probabilities (keepdim)"""
        if self.continuous_action:
            action, _ = self.model.policy(obs)
            return action
        if self.fused_policy:
            logits = self.model.policy(obs)
            best = logits.amax(dim=-1, keepdim=True)
            self._refuse_diverged(~(best < float('inf')))
            legal = (best > float('-inf')) & (best < float('inf'))
            return logits.argmax(dim=-1, keepdim=True).masked_fill(~legal, -1)
        return Categorical(logits=self.model.policy(obs)).probs.argmax(dim=-1, keepdim=True)

    @torch.no_grad()
    def value(self, obs):
        return self.model.value(obs)
