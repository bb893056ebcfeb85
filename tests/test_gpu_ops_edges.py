"""The memory policy's operators where a call is easily answered wrongly: derivatives and traces that pass a kernel by, outputs
that overlap themselves, tensors off their boundary or of another layout, and values at the ends of the range."""
import pytest
import torch
from conftest import fme  # noqa: F401  (loads the package)
from test_gpu_ops import DEV, U, check_norm, last_dense, make, norm_case, on_gpu, oracle

from fast_mario_env_b200 import ops

pytestmark = pytest.mark.gpu


def seq(t=5, d=64, dtype=torch.float32, seed=40):
    c = make(2, t, 2, d, dtype, None, True, seed=seed)
    return [c[x].to(DEV) for x in ("q", "k", "v")], c["g"].to(DEV), c["state"].to(DEV)


# ---------------------------------------------------------------------------------------------- derivatives and traces
@pytest.mark.parametrize("which", ["q", "v", "state", "log_decay"])
def test_forward_mode_is_refused(which):
    """A dual tensor wants a tangent of the output, which no kernel computes."""
    fw = torch.autograd.forward_ad
    (q, k, v), g, s = seq()
    with fw.dual_level():
        kw = dict(q=q, k=k, v=v, log_decay=g, state=s)
        assert ops.decay_attention(**kw)[0].isfinite().all()        # no tangent: nothing to refuse
        kw[which] = fw.make_dual(kw[which], torch.ones_like(kw[which]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.decay_attention(**kw)
        one = {**kw, **{x: kw[x][:, 0] for x in ("q", "k", "v")}}
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops.decay_attention_step(**one)
        x, w = torch.randn(4, 16, device=DEV), torch.ones(16, device=DEV)
        assert ops.group_norm_act(x, 2, w).isfinite().all()
        for a in ((fw.make_dual(x, x), 2, w), (x, 2, fw.make_dual(w, w)), (x, 2, w, fw.make_dual(w, w))):
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.group_norm_act(*a)


@pytest.mark.filterwarnings("ignore")
def test_a_trace_computes_and_does_not_replay_empty_outputs():
    (q, k, v), g, s = seq()
    f = torch.jit.trace(lambda q, k, v: ops.decay_attention(q, k, v, g, state=s)[0], (q, k, v), check_trace=False)
    assert torch.equal(f(2 * q, k, v), ops.decay_attention(2 * q, k, v, g, state=s)[0])
    x = torch.randn(4, 16, device=DEV)
    f = torch.jit.trace(lambda x: ops.group_norm_act(x, 2), (x,), check_trace=False)
    y = torch.randn(4, 16, device=DEV)
    assert torch.equal(f(y), ops.group_norm_act(y, 2))
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda q: ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s), (q,), check_trace=False)


def test_make_fx_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    (q, k, v), g, s = seq()
    for f in (lambda q: ops.decay_attention(q, k, v, g)[0], lambda q: ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s),
              lambda q: ops.group_norm_act(q[:, 0, 0], 2)):
        with pytest.raises(RuntimeError, match="make_fx"):
            make_fx(f)(q)


# ---------------------------------------------------------------------------------------------- layouts
def off_by_one(x):
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x)


def test_states_and_their_gradients_off_a_boundary():
    (q, k, v), g, s = seq()
    q.requires_grad_()
    want_o, want = ops.decay_attention(q, k, v, g, state=s)
    o, last = ops.decay_attention(q, k, v, g, state=off_by_one(s))
    assert torch.equal(o, want_o) and torch.equal(last, want)
    dl = torch.randn_like(last)
    a = torch.autograd.grad(want, q, dl, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(last, q, off_by_one(dl))[0], a)
    b = torch.autograd.grad(torch.cat([torch.ones(1, device=DEV), want.flatten()]), q, torch.cat([torch.ones(1, device=DEV), dl.flatten()]))[0]
    assert torch.equal(b, a)
    with pytest.raises(ValueError, match="16-byte"):   # updated in place: a copy would not do
        ops.decay_attention_step(q[:, 0].detach(), k[:, 0], v[:, 0], g, off_by_one(s))


def test_saved_tensors_that_come_back_in_another_layout():
    """Hooks may hand back what was saved with other strides, as torch's own pinned offloading does."""
    x, w, b, dy = norm_case((3, 16, 5, 4), 4, torch.float32, seed=41)
    (q, k, v), g, s = seq(t=70)
    r = (torch.rand(2, 70, device=DEV) < 0.1).t().contiguous().t()
    qs = [i.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for i in (q, k, v)]
    gx, gw, gb = last_dense(x.to(DEV)).requires_grad_(), w.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()

    def grads():
        y = ops.group_norm_act(gx, 4, gw, gb)
        o, _ = ops.decay_attention(*qs, g, reset=r, state=s)
        return lambda: (*torch.autograd.grad(y, (gx, gw, gb), last_dense(dy.to(DEV))), *torch.autograd.grad(o, qs, torch.ones_like(o)))

    want = grads()()
    with torch.autograd.graph.save_on_cpu(pin_memory=True):
        later = grads()
    for a, c in zip(want, later()):
        assert torch.equal(a, c)


def test_an_output_whose_rows_overlap_is_refused():
    (q, k, v), g, s = seq()
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    keep = s.clone()
    for out in (torch.zeros(1, 2, 64, device=DEV).expand(2, 2, 64), torch.zeros(2, 1, 64, device=DEV).expand(2, 2, 64),
                torch.zeros(256, device=DEV).as_strided((2, 2, 64), (32, 64, 1))):
        with pytest.raises(ValueError, match="overlap"):
            ops.decay_attention_step(q, k, v, g, s, out=out)
    assert torch.equal(s, keep)
    want = ops.decay_attention_step(q, k, v, g, keep)
    assert torch.equal(ops.decay_attention_step(q, k, v, g, s, out=v), want) and torch.equal(s, keep)


# ---------------------------------------------------------------------------------------------- values
def test_silu_slope_of_large_values():
    """silu'(z) is 1 for large z and 0 for very negative ones, however large |z| is; one value a group keeps x^ at 1 and -1."""
    x = torch.tensor([[1.0, -1.0, 3.0, -3.0]], device=DEV).repeat(6, 1)
    for shape, p in (((6, 4), 1), ((6, 4, 8), 8)):
        gx = (x if p == 1 else last_dense(x[:, :, None].repeat(1, 1, p))).requires_grad_()
        for scale in (30.0, 1e4, 2.0 ** 25, 1e12):
            w, b = torch.full((4,), scale, device=DEV), torch.zeros(4, device=DEV, requires_grad=True)
            y = ops.group_norm_act(gx, 2, w, b)
            db = torch.autograd.grad(y, b, torch.ones_like(y))[0]
            want = 6 * p * torch.tensor([1.0, 0.0, 1.0, 0.0], device=DEV)   # silu' - (1 or 0) is below 30 e^-30 = 3e-12
            assert ((db - want).abs() <= 6 * p * 16 * U).all(), (shape, scale, db)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("u8", [False, True])
@pytest.mark.parametrize("shape, groups", [((2, 515, 64, 64), 5), ((2, 2052, 2), 1), ((3, 2055, 1, 2), 3)])
def test_constant_groups_of_many_channels(shape, groups, u8, dtype):
    """A constant group: each rounding of a long sum in the same direction moves the mean off it."""
    x, w, b, dy = norm_case(shape, groups, dtype, seed=42)
    x[0] = 1000.1
    x[1, : shape[1] // groups] = -7.3
    check_norm(x, groups, w, b, dy, "none", u8)


@pytest.mark.parametrize("shape, groups, u8", [((2, 64, 112, 112), 32, False), ((1, 192, 64, 64), 16, False), ((2, 110, 84, 84), 10, False),
                                               ((2, 128, 112, 112), 32, False), ((1, 192, 74, 74), 16, True), ((1, 192, 75, 75), 16, True)])
def test_samples_that_a_cluster_just_holds(shape, groups, u8):
    """bfloat16 samples that 16 CTAs hold without the sums and not with them."""
    x, w, b, dy = norm_case(shape, groups, torch.bfloat16, seed=43)
    check_norm(x, groups, w, b, dy, "silu", u8)


@pytest.mark.parametrize("t, p_reset", [(2, None), (67, 0.02), (799, None), (1500, 0.003)])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_float32_products_lose_no_digits_along_their_sums(d, t, p_reset):
    """Relative to its norm a float32 result is off by 16 * 2^-24 at most: an operand in two tf32 numbers and the dropped product of
    the remainders are 3 * 2^-24 of a term, through two products in a row 6; each of the three sums (scores, their product, the
    state's) adds at most 16 partial sums, each addition off by 2^-25 of what there is, together 2 * 2^-24 as they are independent."""
    c = make(1, t, 2, d, torch.float32, p_reset, True, seed=44)
    want = oracle(c, d ** -0.5)
    for name, x in on_gpu(c).items():
        err = (x.detach().double().cpu() - want[name]).norm() / want[name].norm()
        assert err <= 16 * U, (name, float(err))
