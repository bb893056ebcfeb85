"""The float64 oracle of the memory policy's operators against differences, and the refusals that need no GPU."""
import ctypes

import pytest
import torch
from conftest import fme  # noqa: F401  (loads the package)

import memory_oracle as mo
from fast_mario_env_b200 import _native as N
from fast_mario_env_b200 import ops


def _case(seed=0, n=2, t=7, h=2, d=4):
    r = torch.Generator().manual_seed(seed)
    z = lambda *s: torch.randn(s, generator=r, dtype=torch.float64)  # noqa: E731
    reset = torch.rand((n, t), generator=r) < 0.3
    return dict(q=z(n, t, h, d), k=z(n, t, h, d), v=z(n, t, h, d), state=z(n, h, d, d)), -torch.rand(h, generator=r, dtype=torch.float64), \
        reset, z(n, t, h, d), z(n, h, d, d)


@pytest.mark.parametrize("seed", [0, 1])
def test_attention_gradients_match_differences(seed):
    """o and the last state are linear in each of q, k, v and the first state, so a difference is exact."""
    x, g, reset, do, dl = _case(seed)
    dq, dk, dv, ds = mo.attn_backward(x["q"], x["k"], x["v"], g, do, reset, x["state"], dl, 0.7)

    def loss(**y):
        z = {**x, **y}
        o, last, _ = mo.attn_forward(z["q"], z["k"], z["v"], g, reset, z["state"], 0.7)
        return (o * do).sum() + (last * dl).sum()

    for name, grad in (("q", dq), ("k", dk), ("v", dv), ("state", ds)):
        u = torch.randn(x[name].shape, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
        got = loss(**{name: x[name] + u}) - loss(**{name: x[name] - u})
        assert torch.allclose(got, 2 * (grad * u).sum(), rtol=1e-11, atol=1e-11), name


@pytest.mark.parametrize("name", ["none", "relu", "silu"])
def test_norm_gradients_match_differences(name):
    r = torch.Generator().manual_seed(3)
    z = lambda *s: torch.randn(s, generator=r, dtype=torch.float64)  # noqa: E731
    x, w, b, dy = z(3, 6, 5), z(6), z(6), z(3, 6, 5)
    dx, dw, db = mo.norm_backward(x, 2, w, b, 1e-5, name, dy)
    loss = lambda x, w, b: (mo.norm_forward(x, 2, w, b, 1e-5, name) * dy).sum()  # noqa: E731
    e = 1e-6
    for i, (t, grad) in enumerate(((x, dx), (w, dw), (b, db))):
        u = z(*t.shape)
        a, c = [x, w, b], [x, w, b]
        a[i], c[i] = t + e * u, t - e * u
        assert torch.allclose((loss(*a) - loss(*c)) / (2 * e), (grad * u).sum(), rtol=1e-7, atol=1e-7)


def test_operators_refuse_cpu_tensors():
    q = torch.zeros(1, 2, 1, 32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.decay_attention(q, q, q, torch.zeros(1))
    with pytest.raises(ValueError, match="CUDA"):
        ops.decay_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(1), torch.zeros(1, 1, 32, 32))
    with pytest.raises(ValueError, match="CUDA"):
        ops.group_norm_act(torch.zeros(2, 8), 2)


def test_rows_of_an_output_that_overlap_are_found():
    """Against counting: (n, h, d) views of a buffer, shared axes, interleaved rows and rows that run into each other."""
    flat = torch.arange(4096)
    seen = set()
    for n in (1, 2, 3, 5):
        for h in (1, 2, 4):
            for sn in (0, 4, 8, 12, 16, 24, 32, 36, 64):
                for sh in (0, 4, 8, 12, 16, 20, 24, 40, 64):
                    x = flat.as_strided((n, h, 8), (sn, sh, 1))
                    shared = x.unique().numel() < x.numel()
                    assert ops._shares_memory(x) == shared, (n, h, sn, sh)
                    seen.add(shared)
    assert seen == {True, False}
    assert ops._shares_memory(torch.empty(1, 2, 64).expand(5, 2, 64)) and not ops._shares_memory(torch.empty(5, 4, 64)[:, ::2])


def _attn(**kw):
    a = N.FmeDecayAttn(n=1, t=1, h=1, d=64, dtype=N.FME_F32, scale=1.0, log_decay=256)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw, said", [
    (dict(n=-1), ">= 0"), (dict(t=-1), ">= 0"), (dict(h=0), "h >= 1"), (dict(d=48), "32, 64 or 128"), (dict(dtype=7), "dtype"),
    (dict(n=1 << 20, h=1 << 12), "pairs"), (dict(log_decay=None), "log_decay"), (dict(s_in=264), "16-byte"),
    (dict(), "q, k, v"), (dict(q=(260, 64, 64, 64), k=(256, 64, 64, 64), v=(256, 64, 64, 64)), "16-byte"),
    (dict(q=(256, 64, 64, 63), k=(256, 64, 64, 64), v=(256, 64, 64, 64)), "16-byte")])
def test_library_refuses_bad_attention_arguments(kw, said):
    """Refused on the host, before anything is launched."""
    kw = {k: N.FmeAttnTensor(*v) if isinstance(v, tuple) else v for k, v in kw.items()}
    a = _attn(**kw)
    for f in (N.lib().fme_decay_attn_fwd, N.lib().fme_decay_attn_bwd, N.lib().fme_decay_attn_step):
        assert f(ctypes.byref(a), None) == -1
        assert said in N.last_error()


def test_library_refuses_bad_step_and_missing_outputs():
    rows = N.FmeAttnTensor(256, 64, 64, 64)
    L = N.lib()
    assert L.fme_decay_attn_step(ctypes.byref(_attn(t=2, q=rows, k=rows, v=rows)), None) == -1 and "t must be 1" in N.last_error()
    assert L.fme_decay_attn_step(ctypes.byref(_attn(q=rows, k=rows, v=rows)), None) == -1 and "s_in and s_out" in N.last_error()
    assert L.fme_decay_attn_fwd(ctypes.byref(_attn(q=rows, k=rows, v=rows)), None) == -1 and "o must be given" in N.last_error()
    assert L.fme_decay_attn_bwd(ctypes.byref(_attn(q=rows, k=rows, v=rows)), None) == -1 and "gradients" in N.last_error()
    assert L.fme_decay_attn_fwd(None, None) == -1
    assert L.fme_decay_attn_bytes(None, 0) == -1 and L.fme_decay_attn_bytes(ctypes.byref(_attn()), 3) == -1


@pytest.mark.parametrize("kw, said", [
    (dict(n=-1), "sizes"), (dict(p=-1), "sizes"), (dict(g=3), "divide"), (dict(g=0), "divide"), (dict(c=8192, g=2), "4096"), (dict(dtype=5), "dtype"),
    (dict(act=3), "activation"), (dict(), "required")])
def test_library_refuses_bad_norm_arguments(kw, said):
    a = N.FmeGroupNorm(n=1, p=1, c=8, g=2, dtype=N.FME_F32, act=0, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    for f in (N.lib().fme_group_norm_fwd, N.lib().fme_group_norm_bwd):
        assert f(ctypes.byref(a), None) == -1
        assert said in N.last_error()
    a = N.FmeGroupNorm(n=1, p=1, c=8, g=2, dtype=N.FME_F32, act=0, eps=1e-5, dw=256)
    assert N.lib().fme_group_norm_bwd(ctypes.byref(a), None) == -1 and "together" in N.last_error()


def test_packed_arguments_have_the_structures_layout():
    for packed, struct in ((N.ATTN, N.FmeDecayAttn), (N.NORM, N.FmeGroupNorm)):
        assert packed.size == ctypes.sizeof(struct)
        n = len(packed.unpack(bytes(packed.size)))
        raw = struct.from_buffer_copy(packed.pack(*range(1, n + 1)))
        flat = []
        for name, _ in struct._fields_:
            v = getattr(raw, name)
            flat += [v.p, v.sn, v.st, v.sh] if isinstance(v, N.FmeAttnTensor) else [v]
        assert [int(v) for v in flat] == list(range(1, n + 1))


def test_empty_calls_need_no_buffers():
    assert N.lib().fme_decay_attn_fwd(ctypes.byref(_attn(n=0)), None) == 0
    a = N.FmeGroupNorm(n=0, p=1, c=8, g=2, dtype=N.FME_F32, act=0, eps=1e-5)
    assert N.lib().fme_group_norm_fwd(ctypes.byref(a), None) == 0


LARGE_SAMPLES = [((8, 64, 112, 112), 32, False, 1), ((8, 192, 64, 64), 16, False, 1), ((8, 192, 64, 64), 32, False, 1), ((8, 110, 84, 84), 10, False, 1),
                 ((8, 128, 112, 112), 32, False, 0), ((8, 192, 74, 74), 16, True, 1), ((4, 192, 75, 75), 16, True, 1), ((36, 192, 65, 65), 16, False, 1)]


@pytest.mark.parametrize("shape, groups, u8, which", LARGE_SAMPLES)
def test_samples_that_a_cluster_just_holds_leave_room_for_their_sums(shape, groups, u8, which):
    """bfloat16 samples between what 16 CTAs hold with the sums and without them are split into parts, whose sums a workspace
    holds; they used to be left to one thread a channel (no workspace forward, 592 rows of dw and db backward)."""
    n, c = shape[:2]
    p = shape[2] * shape[3]
    got = ops._norm_size(n, p, c, groups, N.FME_BF16, u8, True, p * c, True, p * c, which)
    each, row = (16, 0) if which == 0 else (8, 8 * c)   # bytes of a (sample, part, group), and a part's dw and db
    parts, rest = divmod(got - n * groups * each, n * (groups * each + row))
    assert rest == 0 and parts > 16
