"""A policy with memory on the operators of `ops.py`, and PPO over whole rollouts for it.

`MemoryAC` is the Nature-CNN actor-critic of `ppo.py` (src/fast_mario_env/ppo/model.py:13-30 in the reference) with group norm
and SiLU after each convolution and, between the trunk and the heads, a layer of decayed linear attention: every env carries one
(head_dim, head_dim) matrix per head, which an episode's start clears. Acting takes one token a step
(`decay_attention_step`); learning runs the same recurrence over the rollout at once (`decay_attention`) and keeps the
normalised activations' inputs in 8 bits (`group_norm_act(..., checkpoint="u8")`).

    net = MemoryAC(7).cuda()
    state = net.initial_state(n_envs)
    logits, value = net.step(obs, state, reset)          # obs (N, 4, 84, 84) uint8; state updated in place
    logits, value, state = net(obs_seq, state0, resets)  # obs_seq (T, N, 4, 84, 84), resets (T, N)
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import ops
from .ppo import STAT_NAMES, PPOConfig, Storage, adv_norm, gae


class GroupNormAct(nn.Module):
    """`ops.group_norm_act` with its weight and bias."""

    def __init__(self, channels: int, groups: int, act: str = "silu", checkpoint: str = "full", eps: float = 1e-5):
        super().__init__()
        self.groups, self.act, self.checkpoint, self.eps = groups, act, checkpoint, eps
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels))

    def forward(self, x):
        return ops.group_norm_act(x, self.groups, self.weight, self.bias, eps=self.eps, act=self.act, checkpoint=self.checkpoint)


class MemoryAC(nn.Module):
    def __init__(self, n_actions: int = 7, in_ch: int = 4, heads: int = 8, head_dim: int = 64, groups: int = 8, checkpoint: str = "u8"):
        super().__init__()
        self.heads, self.head_dim, self.width = heads, head_dim, 512
        inner = heads * head_dim
        self.convs = nn.ModuleList([nn.Conv2d(in_ch, 32, 8, 4), nn.Conv2d(32, 64, 4, 2), nn.Conv2d(64, 64, 3, 1)])
        self.norms = nn.ModuleList([GroupNormAct(c, groups, checkpoint=checkpoint) for c in (32, 64, 64)])
        self.fc = nn.Linear(3136, self.width)
        self.qkv = nn.Linear(self.width, 3 * inner, bias=False)
        self.head_norm = GroupNormAct(inner, heads, act="none")
        self.out = nn.Linear(inner, self.width, bias=False)
        self.pi = nn.Linear(self.width, n_actions)
        self.vf = nn.Linear(self.width, 1)
        # horizons from 4 to 512 steps over the heads
        self.register_buffer("log_decay", torch.log1p(-torch.exp2(-torch.linspace(2.0, 9.0, heads))))
        for m in [*self.convs, self.fc, self.pi, self.vf]:
            nn.init.orthogonal_(m.weight, 0.01 if m is self.pi else 1.0 if m is self.vf else math.sqrt(2.0))
            nn.init.zeros_(m.bias)
        for c in self.convs:   # channels-last weights: the convolutions' outputs then are what the norms read
            c.weight.data = c.weight.data.contiguous(memory_format=torch.channels_last)

    def initial_state(self, n: int):
        d = self.head_dim
        return torch.zeros((n, self.heads, d, d), dtype=torch.float32, device=self.log_decay.device)

    def encode(self, obs_u8):
        x = obs_u8.float().mul_(1.0 / 255.0).contiguous(memory_format=torch.channels_last)
        for conv, norm in zip(self.convs, self.norms):
            x = norm(conv(x).contiguous(memory_format=torch.channels_last))
        return F.silu(self.fc(x.flatten(1)))

    def _heads(self, x, o):
        h = x + self.out(self.head_norm(o))
        return self.pi(h), self.vf(h).squeeze(-1)

    def forward(self, obs, state=None, reset=None):
        """A time-major rollout: obs (T, N, C, 84, 84) uint8, reset (T, N) bool (set where obs[t] starts an episode), state before
        it. Returns logits (T, N, A), values (T, N) and the state after it."""
        t, n = obs.shape[:2]
        x = self.encode(obs.flatten(0, 1))
        q, k, v = self.qkv(x).view(t, n, 3, self.heads, self.head_dim).transpose(0, 1).unbind(2)   # (N, T, H, D) views
        o, last = ops.decay_attention(q, k, v, self.log_decay, reset=None if reset is None else reset.t(), state=state)
        o = o.transpose(0, 1).reshape(t * n, -1)
        logits, values = self._heads(x, o)
        return logits.view(t, n, -1), values.view(t, n), last

    @torch.no_grad()
    def step(self, obs, state, reset=None):
        """One step of N envs: obs (N, C, 84, 84) uint8, reset (N,) bool; state is updated in place. Returns logits and values."""
        x = self.encode(obs)
        q, k, v = self.qkv(x).view(obs.shape[0], 3, self.heads, self.head_dim).unbind(1)
        o = ops.decay_attention_step(q, k, v, self.log_decay, state, reset=reset)
        return self._heads(x, o.view(obs.shape[0], -1))


class MemoryTrainer:
    """PPO with whole rollouts of some envs as minibatches (GAE, advantage normalisation, clipping and the losses as in
    `ppo.py`; src/fast_mario_env/ppo/train.py:112-247 in the reference). cfg.batch counts samples, so a minibatch holds
    cfg.batch // cfg.n_steps envs.

    Every step runs eagerly: cfg.graph is not used. Nor is cfg.trunc_budget (all envs that a time limit cuts are bootstrapped, at
    one look from the host a step) or cfg.channels_last (the norms need that layout). Gradients are not averaged over ranks."""

    def __init__(self, env, cfg: PPOConfig, dev, seed: int = 0, net: MemoryAC | None = None):
        torch.manual_seed(seed)
        if cfg.batch % cfg.n_steps or cfg.n_envs % (cfg.batch // cfg.n_steps):
            raise ValueError("cfg.batch must be whole rollouts, and the envs whole minibatches")
        self.env, self.cfg, self.dev = env, cfg, dev
        self.net = (net if net is not None else MemoryAC()).to(dev)
        self.params = list(self.net.parameters())
        self.opt = torch.optim.Adam(self.params, lr=cfg.lr, eps=cfg.adam_eps, fused=True)
        self.buf = Storage(cfg.n_steps, cfg.n_envs, dev)
        self.adv, self.ret = torch.zeros_like(self.buf.rew), torch.zeros_like(self.buf.rew)
        self.obs = env.reset().clone()
        self.reset = torch.ones(cfg.n_envs, dtype=torch.bool, device=dev)
        self.state = self.net.initial_state(cfg.n_envs)
        self.state0 = torch.zeros_like(self.state)

    @torch.no_grad()
    def collect(self):
        """One rollout: obs, actions, log-probs, values, rewards, done flags, and the state that it began with."""
        c, b = self.cfg, self.buf
        self.state0.copy_(self.state)
        for t in range(c.n_steps):
            b.obs[t].copy_(self.obs)
            b.done[t].copy_(self.reset)
            logits, v = self.net.step(self.obs, self.state, self.reset)
            logp = F.log_softmax(logits, -1)
            a = (logp - torch.log(-torch.log(torch.rand_like(logp).clamp_(1e-20, 1.0)))).argmax(-1)
            b.act[t].copy_(a); b.val[t].copy_(v); b.logp[t].copy_(logp.gather(-1, a[:, None]).squeeze(-1))
            obs, rew, term, trunc, info = self.env.step(a)
            b.rew[t].copy_(rew)
            cut = (trunc & ~term).bool()
            if bool(cut.any()):   # the time limit is no end: add the discounted value of where it cut, with the memory it had
                i = cut.nonzero().squeeze(-1)
                _, nv = self.net.step(info["final_obs"][i], self.state[i])
                b.rew[t].index_add_(0, i, c.gamma * nv)
            self.obs.copy_(obs)
            self.reset.copy_((term | trunc).bool())
        b.next_done.copy_(self.reset)
        _, nv = self.net.step(self.obs, self.state.clone(), self.reset)   # the memory itself moves on in the next rollout
        b.next_val.copy_(nv)

    def minibatch(self, envs):
        """One step on the whole rollouts of the given envs (int64 indices)."""
        c, b = self.cfg, self.buf
        logits, v, _ = self.net(b.obs[:, envs], self.state0[envs], b.done[:, envs].bool())
        logp_all = F.log_softmax(logits, -1)
        logp = logp_all.gather(-1, b.act[:, envs, None]).squeeze(-1)
        entropy = -(logp_all.exp() * logp_all).sum(-1).mean()
        adv = self.adv[:, envs].reshape(-1)
        adv = adv_norm(adv).view_as(logp)
        lr = (logp - b.logp[:, envs]).clamp(-20.0, 20.0)
        ratio = lr.exp()
        pg = -torch.min(adv * ratio, adv * ratio.clamp(1 - c.clip, 1 + c.clip)).mean()
        vl = F.mse_loss(self.ret[:, envs], v)
        loss = pg - c.ent * entropy + c.vf * vl
        self.opt.zero_grad(set_to_none=True)
        loss.backward()
        norm = nn.utils.clip_grad_norm_(self.params, c.max_grad_norm)
        ok = torch.isfinite(norm)
        for p in self.params:   # a non-finite minibatch is skipped
            p.grad.copy_(torch.where(ok, p.grad, torch.zeros_like(p.grad)))
        self.opt.step()
        with torch.no_grad():
            return torch.stack([pg, vl, entropy, ((ratio - 1).abs() > c.clip).float().mean(), ((ratio - 1) - lr).mean(), (~ok).float()])

    def iterate(self):
        """A rollout and cfg.epochs passes over it. Returns the mean statistics, named by ppo.STAT_NAMES."""
        c, b = self.cfg, self.buf
        self.collect()
        gae(b.rew, b.val, b.done, b.next_val, b.next_done, c.gamma, c.lam, self.adv, self.ret)
        per, stats = c.batch // c.n_steps, []
        for _ in range(c.epochs):
            for envs in torch.randperm(c.n_envs, device=self.dev).split(per):
                stats.append(self.minibatch(envs))
        return dict(zip(STAT_NAMES, torch.stack(stats).mean(0).tolist()))
