"""The policy with memory: acting step by step and learning over the rollout are one function, its gradients are those of a plain
torch computation of the same network, and the example runs."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F
from conftest import ROOT, fme  # noqa: F401  (loads the package)

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_tf32():
    old = (torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32)
    torch.backends.cuda.matmul.allow_tf32 = False
    torch.backends.cudnn.allow_tf32 = False
    yield
    torch.backends.cuda.matmul.allow_tf32, torch.backends.cudnn.allow_tf32 = old


def make(checkpoint, t=7, n=5):
    from fast_mario_env_b200.memory import MemoryAC
    torch.manual_seed(0)
    net = MemoryAC(7, heads=4, head_dim=32, checkpoint=checkpoint).cuda()
    torch.nn.init.normal_(net.pi.weight, std=0.1)
    r = torch.Generator().manual_seed(1)
    obs = torch.randint(0, 256, (t, n, 4, 84, 84), generator=r, dtype=torch.uint8).cuda()
    reset = (torch.rand((t, n), generator=r) < 0.3).cuda()
    state = torch.randn((n, 4, 32, 32), generator=r).cuda()
    return net, obs, reset, state


def test_steps_and_rollout_agree():
    """Both are float32 in other orders: 1e-4 of the values' size, the bar for network outputs here."""
    net, obs, reset, state = make("full")
    s = state.clone()
    out = [net.step(obs[t], s, reset[t]) for t in range(obs.shape[0])]
    with torch.no_grad():
        logits, values, last = net(obs, state, reset)
    for a, b in ((torch.stack([o[0] for o in out]), logits), (torch.stack([o[1] for o in out]), values), (s, last)):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()


def plain(net, obs, reset, state):
    """The same network from torch's own functions, the recurrence token by token."""
    t, n = obs.shape[:2]
    x = obs.flatten(0, 1).float() / 255.0
    for conv, norm in zip(net.convs, net.norms):
        x = F.silu(F.group_norm(conv(x), norm.groups, norm.weight, norm.bias, norm.eps))
    x = F.silu(net.fc(x.flatten(1)))
    q, k, v = net.qkv(x).view(t, n, 3, net.heads, net.head_dim).unbind(2)
    s, o = state, []
    for i in range(t):
        s = torch.where(reset[i][:, None, None, None], torch.zeros_like(s), s * net.log_decay.exp()[None, :, None, None])
        s = s + k[i][..., :, None] * v[i][..., None, :]
        o.append((q[i][..., :, None] * s).sum(-2) * net.head_dim ** -0.5)
    o = torch.stack(o).reshape(t * n, -1)
    o = F.group_norm(o, net.heads, net.head_norm.weight, net.head_norm.bias, net.head_norm.eps)
    h = x + net.out(o)
    return net.pi(h).view(t, n, -1), net.vf(h).view(t, n), s


def test_gradients_match_plain_torch():
    """float32 both ways: 1e-3 of each gradient's size, the bar for a network's gradients here."""
    net, obs, reset, state = make("full")

    def grads(f):
        net.zero_grad(set_to_none=True)
        logits, values, last = f()
        (F.log_softmax(logits, -1)[..., 2].mean() + values.square().mean() + 1e-3 * last.square().mean()).backward()
        return {k: p.grad.clone() for k, p in net.named_parameters()}

    got, want = grads(lambda: net(obs, state, reset)), grads(lambda: plain(net, obs, reset, state))
    for k in want:
        assert (got[k] - want[k]).norm() <= 1e-3 * want[k].norm(), k


def test_eight_bit_checkpoints_keep_the_outputs_and_nearly_the_gradients():
    """The forward pass is the same; a kept value is off by at most 1/510 of its group's range, some 2 % of its spread, and
    evenly, so the gradients of sums over thousands of them stay within 5 %."""
    net, obs, reset, state = make("full")
    low, _, _, _ = make("u8")
    low.load_state_dict(net.state_dict())

    def grads(m):
        logits, values, _ = m(obs, state, reset)
        (F.log_softmax(logits, -1)[..., 2].mean() + values.square().mean()).backward()
        return logits.detach(), {k: p.grad for k, p in m.named_parameters()}

    (la, a), (lb, b) = grads(net), grads(low)
    assert torch.equal(la, lb)
    for k in a:
        assert (a[k] - b[k]).norm() <= 0.05 * a[k].norm(), k


def test_example_trains(capsys):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import memory_ppo
    finally:
        sys.path.pop(0)
    history = memory_ppo.main(["--envs", "32", "--steps", "16", "--iterations", "2", "--minibatch-envs", "16"])
    assert len(history) == 2
    for h in history:
        assert h["nonfinite_skips"] == 0 and all(abs(v) < 1e6 for v in h.values()) and 0 < h["entropy"] <= 1.9460
