"""The memory policy's operators against the float64 oracle.

Error bounds, from the operations and not from what comes out. `A` is the operator applied to the absolute values of its
inputs, i.e. the sum of the magnitudes that each output adds up.
* float32: every term carries at most D + T + 16 roundings or truncations of 2^-23 (sums over features and tokens, powers of
  the decay, the scale), so |error| <= (D + T + 16) 2^-23 A.
* bfloat16 (8 bits, so a rounding is off by 2^-8 at most): a term may be rounded to it as a decayed product of q and k or of do and v, as a decayed row,
  as a state read by a matrix product, and the result once more: 4 * 2^-8 A, plus one for products of such roundings.
* states are float32 whatever the inputs: their decayed rows keep 16 bits at least (2^-16 each way), so 2^-15 A plus the
  float32 term."""
import pytest
import torch
from conftest import fme  # noqa: F401  (loads the package)

import memory_oracle as mo
from fast_mario_env_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bound(a, d, t, dtype, state=False):
    f = (d + t + 16) * 2.0 ** -23
    return a * (f if dtype == torch.float32 else f + 2.0 ** -15 if state else f + 5 * 2.0 ** -8) + 1e-30


def decays(h):
    return torch.log1p(-torch.exp2(-torch.linspace(1.0, 9.0, h)))


def make(n, t, h, d, dtype, p_reset, carry, seed=0):
    r = torch.Generator().manual_seed(seed)
    z = lambda *s: torch.randn(s, generator=r)  # noqa: E731
    c = dict(q=z(n, t, h, d).to(dtype), k=z(n, t, h, d).to(dtype), v=z(n, t, h, d).to(dtype), do=z(n, t, h, d).to(dtype), g=decays(h))
    c["reset"] = None if p_reset is None else torch.rand((n, t), generator=r) < p_reset
    c["state"], c["dlast"] = (z(n, h, d, d), z(n, h, d, d)) if carry else (None, None)
    return c


def oracle(c, scale, absolute=False):
    f = (lambda x: None if x is None else x.double().abs()) if absolute else (lambda x: None if x is None else x.double())
    q, k, v, do, s, dl = (f(c[x]) for x in ("q", "k", "v", "do", "state", "dlast"))
    o, last, _ = mo.attn_forward(q, k, v, c["g"].double(), c["reset"], s, scale)
    dq, dk, dv, ds = mo.attn_backward(q, k, v, c["g"].double(), do, c["reset"], s, dl, scale)
    return dict(o=o, last=last, dq=dq, dk=dk, dv=dv, ds=ds)


def on_gpu(c, scale=None, view=lambda x: x):
    leaf = {x: None if c[x] is None else view(c[x].to(DEV)).detach().requires_grad_() for x in ("q", "k", "v")}
    leaf["state"] = None if c["state"] is None else c["state"].to(DEV).requires_grad_()
    reset = None if c["reset"] is None else c["reset"].to(DEV)
    o, last = ops.decay_attention(leaf["q"], leaf["k"], leaf["v"], c["g"].to(DEV), reset=reset, state=leaf["state"], scale=scale)
    outs, grads = ([o, last], [c["do"].to(DEV), c["dlast"].to(DEV)]) if c["dlast"] is not None else ([o], [c["do"].to(DEV)])
    ask = [leaf[x] for x in ("q", "k", "v", "state") if leaf[x] is not None]
    got = torch.autograd.grad(outs, ask, grads)
    return dict(zip(("o", "last", "dq", "dk", "dv", "ds"), (o, last, *got)))


def compare(got, want, size, d, t, dtype):
    for name, x in got.items():
        err = (x.detach().double().cpu() - want[name]).abs()
        lim = bound(size[name], d, t, dtype, state=name in ("last", "ds"))
        assert x.isfinite().all(), name
        assert (err <= lim).all(), (name, float((err / lim).max()))


LENGTHS = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 321]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("t", LENGTHS)
def test_attention_and_gradients(t, d, dtype):
    i = LENGTHS.index(t)
    n, h = [(2, 3), (3, 1), (1, 2)][i % 3]
    c = make(n, t, h, d, dtype, [0.02, None, 0.3][i % 3], carry=i % 2 == 0, seed=t + d)
    scale = d ** -0.5
    compare(on_gpu(c), oracle(c, scale), oracle(c, scale, True), d, t, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_sequences_of_few_rows(dtype):
    """Few (sequence, head) pairs: the time axis is split."""
    n, t, h, d = 1, 1500, 2, 64
    c = make(n, t, h, d, dtype, 0.003, True, seed=5)
    compare(on_gpu(c), oracle(c, d ** -0.5), oracle(c, d ** -0.5, True), d, t, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(dtype):
    """More (sequence, head) pairs than the GPU runs at once."""
    n, t, h, d = 700, 70, 3, 32
    c = make(n, t, h, d, dtype, 0.05, True, seed=6)
    compare(on_gpu(c), oracle(c, d ** -0.5), oracle(c, d ** -0.5, True), d, t, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("g", [0.0, -1e-4, -30.0, -200.0, float("-inf")])
def test_extreme_decays(g, dtype):
    c = make(2, 90, 2, 64, dtype, 0.05, True, seed=7)
    c["g"] = torch.tensor([g, -0.1])
    compare(on_gpu(c), oracle(c, 0.125), oracle(c, 0.125, True), 64, 90, dtype)


@pytest.mark.parametrize("p_reset", [0.0, 1.0])
def test_no_and_only_restarts(p_reset):
    c = make(2, 130, 2, 64, torch.bfloat16, p_reset, True, seed=8)
    got = on_gpu(c)
    compare(got, oracle(c, 0.125), oracle(c, 0.125, True), 64, 130, torch.bfloat16)
    if p_reset == 1.0:
        assert (got["ds"] == 0).all()


def test_restart_as_bytes_and_time_major():
    c = make(3, 70, 2, 64, torch.float32, 0.1, False, seed=9)
    want = on_gpu(c)["o"]
    q, k, v = (c[x].to(DEV) for x in ("q", "k", "v"))
    tm = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731  (a time-major rollout, seen as (N, T, ...))
    r = tm(c["reset"].to(DEV).to(torch.uint8) * 255)
    o, _ = ops.decay_attention(tm(q), tm(k), tm(v), c["g"].to(DEV), reset=r)
    assert torch.equal(o, want)
    step = ops.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], c["g"].to(DEV), torch.zeros(3, 2, 64, 64, device=DEV), reset=r[:, 0])
    assert torch.allclose(step, want[:, 0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strided_and_misaligned_inputs(dtype):
    """Slices of one fused projection, and rows that start off a 16-byte boundary."""
    n, t, h, d = 2, 75, 2, 64
    c = make(n, t, h, d, dtype, 0.05, False, seed=10)
    want = on_gpu(c)
    fused = torch.stack([c["q"], c["k"], c["v"]], 2).to(DEV)
    o, _ = ops.decay_attention(fused[:, :, 0], fused[:, :, 1], fused[:, :, 2], c["g"].to(DEV), reset=c["reset"].to(DEV))
    assert torch.equal(o, want["o"])

    def off_by_one(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
        return y.copy_(x)

    got = on_gpu(c, view=off_by_one)
    for name in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[name], want[name])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_shared_heads_get_the_sum_of_their_gradients(dtype):
    n, t, h, d = 2, 70, 4, 32
    c = make(n, t, h, d, dtype, 0.05, False, seed=11)
    for x in ("k", "v"):
        c[x] = c[x][:, :, :1].expand(n, t, h, d)
    k, v = (c[x][:, :, :1].to(DEV).requires_grad_() for x in ("k", "v"))
    q = c["q"].to(DEV).requires_grad_()
    o, _ = ops.decay_attention(q, k.expand(n, t, h, d), v.expand(n, t, h, d), c["g"].to(DEV), reset=c["reset"].to(DEV))
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), c["do"].to(DEV))
    want, size = oracle(c, d ** -0.5), oracle(c, d ** -0.5, True)
    for name in ("dk", "dv"):
        want[name], size[name] = want[name].sum(2, keepdim=True), size[name].sum(2, keepdim=True)
    compare(dict(o=o, dq=dq, dk=dk, dv=dv), want, size, d, t, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_numbers_stay_in_their_episode(bad, dtype):
    """Nothing reaches the tokens before them or those after the next restart; gradients neither."""
    n, t, h, d = 2, 150, 2, 64
    c = make(n, t, h, d, dtype, None, True, seed=12)
    c["reset"] = torch.zeros(n, t, dtype=torch.bool)
    c["reset"][0, [30, 100]] = True
    c["reset"][1, 64] = True
    clean = on_gpu(c)
    c["k"][0, 40, 0, 3] = bad
    c["v"][0, 50, 0, 5] = bad
    c["state"][1, 0, 2, 2] = bad
    got = on_gpu(c)
    size, want = oracle({**c, "k": c["k"].nan_to_num(0, 0, 0), "v": c["v"].nan_to_num(0, 0, 0), "state": c["state"].nan_to_num(0, 0, 0)}, 0.125, True), clean
    ok = torch.ones(n, t, h, dtype=torch.bool)
    ok[0, 30:100, 0] = False
    ok[1, :64, 0] = False
    for name in ("o", "dq", "dk", "dv"):
        err = (got[name].double().cpu() - want[name].double().cpu()).abs()
        lim = 2 * bound(size[name], d, t, dtype)
        assert (err[ok] <= lim[ok]).all(), name
    assert got["o"][0, 30:40].isfinite().all() and not got["o"][0, 40:100, 0].isfinite().all()
    assert got["last"].isfinite().all() and got["ds"][0].isfinite().all()
    # gradients that are not numbers: they reach the tokens of their own episode up to theirs
    c = make(n, t, h, d, dtype, None, False, seed=12)
    c["reset"] = torch.zeros(n, t, dtype=torch.bool)
    c["reset"][0, [30, 100]] = True
    clean = on_gpu(c)
    c["do"][0, 60, 1, 7] = bad
    got = on_gpu(c)
    ok = torch.ones(n, t, h, dtype=torch.bool)
    ok[0, 30:61, 1] = False
    for name in ("dk", "dv", "dq"):
        err = (got[name].double().cpu() - clean[name].double().cpu()).abs()
        assert (err[ok] <= 2 * bound(size[name], d, t, dtype)[ok]).all(), name


def test_two_halves_make_the_whole():
    c = make(2, 200, 2, 64, torch.float32, 0.02, True, seed=13)
    g, r = c["g"].to(DEV), c["reset"].to(DEV)
    q, k, v, s = (c[x].to(DEV) for x in ("q", "k", "v", "state"))
    whole, last = ops.decay_attention(q, k, v, g, reset=r, state=s)
    a, mid = ops.decay_attention(q[:, :90], k[:, :90], v[:, :90], g, reset=r[:, :90], state=s)
    b, end = ops.decay_attention(q[:, 90:], k[:, 90:], v[:, 90:], g, reset=r[:, 90:], state=mid)
    size = oracle(c, 0.125, True)
    assert ((torch.cat([a, b], 1) - whole).abs().cpu() <= 2 * bound(size["o"], 64, 200, torch.float32)).all()
    assert ((end - last).abs().cpu() <= 2 * bound(size["last"], 64, 200, torch.float32, True)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n, h, d", [(1, 1, 32), (5, 3, 64), (33, 2, 128), (300, 8, 32)])
def test_steps_follow_the_oracle(n, h, d, dtype):
    t = 6
    c = make(n, t, h, d, dtype, 0.3, True, seed=14)
    size, want = oracle(c, d ** -0.5, True), oracle(c, d ** -0.5)
    state, g, reset = c["state"].to(DEV), c["g"].to(DEV), c["reset"].to(DEV)
    place = state.data_ptr()
    for i in range(t):
        o = ops.decay_attention_step(*(c[x][:, i].to(DEV) for x in ("q", "k", "v")), g, state, reset=reset[:, i])
        assert ((o.double().cpu() - want["o"][:, i]).abs() <= bound(size["o"][:, i], d, t, dtype)).all()
    assert state.data_ptr() == place
    assert ((state.double().cpu() - want["last"]).abs() <= bound(size["last"], d, t, torch.float32)).all()


def test_step_with_strides_out_and_bad_values():
    n, h, d = 7, 3, 64
    c = make(n, 1, h, d, torch.bfloat16, None, True, seed=15)
    fused = torch.stack([c["q"][:, 0], c["k"][:, 0], c["v"][:, 0]], 1).to(DEV)
    state, g = c["state"].to(DEV), c["g"].to(DEV)
    state[2, 1, 0, 0] = float("nan")
    reset = torch.zeros(n, dtype=torch.bool, device=DEV)
    reset[2] = True
    out = torch.zeros(n, 2 * h, d, dtype=torch.bfloat16, device=DEV)[:, ::2]
    assert ops.decay_attention_step(fused[:, 0], fused[:, 1], fused[:, 2], g, state, reset=reset, out=out) is out
    c["reset"], c["state"] = reset.cpu()[:, None], c["state"]
    want, size = oracle(c, 0.125), oracle(c, 0.125, True)
    assert ((out.double().cpu() - want["o"][:, 0]).abs() <= bound(size["o"][:, 0], d, 1, torch.bfloat16)).all()
    assert state.isfinite().all()


def test_a_state_that_a_backward_pass_needs_is_not_changed_unnoticed():
    c = make(2, 5, 2, 64, torch.float32, None, True, seed=19)
    q, k, v, g, s = (c[x].to(DEV) for x in ("q", "k", "v", "g", "state"))
    q.requires_grad_()
    o, _ = ops.decay_attention(q, k, v, g, state=s)
    ops.decay_attention_step(q[:, 0].detach(), k[:, 0], v[:, 0], g, s)
    with pytest.raises(RuntimeError, match="inplace"):
        o.sum().backward()


def test_empty_sequences():
    g = decays(2).to(DEV)
    z = torch.zeros(3, 0, 2, 64, device=DEV, requires_grad=True)
    s = torch.randn(3, 2, 64, 64, device=DEV, requires_grad=True)
    o, last = ops.decay_attention(z, z, z, g, state=s)
    assert o.shape == (3, 0, 2, 64) and torch.equal(last, s)
    assert torch.equal(torch.autograd.grad(last, s, torch.ones_like(s))[0], torch.ones_like(s))
    e = torch.zeros(0, 5, 2, 64, device=DEV)
    assert ops.decay_attention(e, e, e, g)[0].shape == (0, 5, 2, 64)
    _, last = ops.decay_attention(z.detach(), z.detach(), z.detach(), g)
    assert (last == 0).all()
    assert ops.decay_attention_step(e[:, 0], e[:, 0], e[:, 0], g, torch.zeros(0, 2, 64, 64, device=DEV)).shape == (0, 2, 64)


def test_offsets_past_32_bits():
    """Two sequences more than 2^31 elements apart in one buffer."""
    t, h, d = 3, 1, 32
    far = 2 ** 31 + 64
    buf = torch.zeros(far + t * d, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((2, t, h, d), (far, d, d, 1))
    c = make(2, t, h, d, torch.bfloat16, None, False, seed=16)
    x.copy_(c["q"].to(DEV))
    o, _ = ops.decay_attention(x, x, x, c["g"].to(DEV))
    y = c["q"].to(DEV)
    assert torch.equal(o, ops.decay_attention(y, y, y, c["g"].to(DEV))[0])
    n = 131073                      # states of 2^31 + 16384 elements in all
    del buf, x
    state = torch.zeros(n, 1, 128, 128, device=DEV)
    q = torch.zeros(n, 1, 128, device=DEV)
    q[-1] = 1.0
    o = ops.decay_attention_step(q, q, q, torch.zeros(1, device=DEV), state, scale=1.0)
    assert (o[-1] == 128).all() and (state[-1] == 1).all() and (o[:-1] == 0).all() and (state[-2] == 0).all()


def test_same_bits_again_and_on_another_stream():
    c = make(3, 140, 2, 64, torch.bfloat16, 0.02, True, seed=17)
    one = on_gpu(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = on_gpu(c)
    side.synchronize()
    for name in one:
        assert torch.equal(one[name], two[name]), name


def test_operators_in_a_captured_graph():
    """Acting and learning are captured by the trainers: the same bits as outside, on inputs that change between replays."""
    n, t, h, d = 3, 600, 2, 64   # few rows: the joined segments are part of it
    c = make(n, t, h, d, torch.bfloat16, 0.01, True, seed=18)
    x, w, b, dy = norm_case((8, 16, 6, 6), 4, torch.float32, seed=18)
    g, reset = c["g"].to(DEV), c["reset"].to(DEV)
    q, k, v = (c[i].to(DEV).requires_grad_() for i in ("q", "k", "v"))
    do, gx, gw, gb, gd = c["do"].to(DEV), last_dense(x.to(DEV)).requires_grad_(), w.to(DEV), b.to(DEV), last_dense(dy.to(DEV))
    state = c["state"].to(DEV)

    def work(s):
        o, last = ops.decay_attention(q, k, v, g, reset=reset, state=c_state)
        y = ops.group_norm_act(gx, 4, gw, gb, checkpoint="u8")
        one = ops.decay_attention_step(q[:, 0].detach(), k[:, 0].detach(), v[:, 0].detach(), g, s, reset=reset[:, 0])
        return (o, last, *torch.autograd.grad(o, (q, k, v), do), y, *torch.autograd.grad(y, gx, gd), one, s)

    c_state, s = state.clone(), state.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work(s)
    with torch.no_grad():
        for i in (q, k, v, gx):
            i.mul_(0.5)
    s.copy_(state)
    graph.replay()
    got = [i.detach().clone() for i in out]
    for a, b in zip(got, work(state.clone())):
        assert torch.equal(a, b)


def test_attention_refusals():
    q = torch.zeros(2, 4, 2, 64, device=DEV)
    g = torch.zeros(2, device=DEV)
    s = torch.zeros(2, 2, 64, 64, device=DEV)
    ok = dict(q=q, k=q, v=q, log_decay=g)
    for kw, said in ((dict(q=q[0]), "axes"), (dict(q=q.half()), "float32 or bfloat16"), (dict(k=q[:1]), "shape"), (dict(v=q.bfloat16()), "dtype"),
                     (dict(q=q[..., :48], k=q[..., :48], v=q[..., :48]), "head size"), (dict(log_decay=g[:1]), "log_decay"),
                     (dict(log_decay=g.double()), "log_decay"), (dict(log_decay=g.clone().requires_grad_()), "no gradient"),
                     (dict(reset=torch.zeros(2, 3, device=DEV, dtype=torch.bool)), "reset"), (dict(reset=torch.zeros(2, 4, device=DEV)), "reset"),
                     (dict(state=s[:1]), "state"), (dict(state=s.bfloat16()), "state"), (dict(state=s.cpu()), "state")):
        with pytest.raises(ValueError, match=said):
            ops.decay_attention(**{**ok, **kw})
    x = q[:, 0]
    with pytest.raises(ValueError, match="contiguous"):
        ops.decay_attention_step(x, x, x, g, s.transpose(2, 3))
    with pytest.raises(ValueError, match="out"):
        ops.decay_attention_step(x, x, x, g, s, out=torch.zeros(2, 2, 64, device=DEV, dtype=torch.bfloat16))


# ---------------------------------------------------------------------------------------------- group norm
# x^ = (x - mean) rstd: the mean carries at most log2-many, here < 16, roundings of the largest magnitude in the sum, the
# variance twice that relative to itself, so x^ is off by at most 32 * 2^-24 (1 + |x^|) + 16 * 2^-24 max|x| rstd =: e. Then
# y is off by act' <= 1.1 times |w| e plus the roundings of z, and dx, with the group means of dz w and dz w x^ (each a sum
# of terms that carry e), by a small multiple K of u' = 64 * 2^-24 times the terms' sizes; each bfloat16 output once by 2^-8.
U = 2.0 ** -24


def norm_case(shape, groups, dtype, seed=0, mean=0.5, spread=1.5):
    r = torch.Generator().manual_seed(seed)
    b, c = shape[:2]
    x = (torch.randn(shape, generator=r) * spread + mean * torch.randn(c, generator=r).view(1, c, *[1] * (len(shape) - 2))).to(dtype)
    return x, 1 + 0.3 * torch.randn(c, generator=r), 0.3 * torch.randn(c, generator=r), torch.randn(shape, generator=r).to(dtype)


def last_dense(x):
    return x.movedim(1, -1).contiguous().movedim(-1, 1)


def check_norm(x, groups, w, b, dy, act, u8=False, eps=1e-5, put=last_dense):
    flat = lambda t: t.reshape(t.shape[0], t.shape[1], -1)  # noqa: E731
    gx, gw, gb = put(x.to(DEV)).requires_grad_(), w.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
    y = ops.group_norm_act(gx, groups, gw, gb, eps=eps, act=act, checkpoint="u8" if u8 else "full")
    assert y.shape == x.shape and y.dtype == x.dtype and ops._channels_last(y)
    dx, dw, db = torch.autograd.grad(y, (gx, gw, gb), last_dense(dy.to(DEV)))
    xd, wd, bd, dyd = flat(x).double(), w.double(), b.double(), flat(dy).double()
    kept = mo.codes(flat(x).float(), groups).double() if u8 else None
    want_y = mo.norm_forward(xd, groups, wd, bd, eps, act)
    want = mo.norm_backward(xd, groups, wd, bd, eps, act, dyd, kept)
    xg, mean, rstd = mo.norm_parts(xd, groups, eps)
    big = xg.abs().amax((2, 3), keepdim=True)
    kg = xg if kept is None else kept.reshape(xg.shape)
    xh = ((kg - mean) * rstd).abs()
    e = (32 * U * (1 + xh) + 16 * U * big * rstd)
    z = (xh.reshape(xd.shape) * wd.abs()[None, :, None] + bd.abs()[None, :, None])
    ez = 1.1 * (wd.abs()[None, :, None] * e.reshape(xd.shape) + 4 * U * z)
    out = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -24
    err = (flat(y.detach()).double().cpu() - want_y).abs()
    assert (err <= ez + out * want_y.abs() + 1e-30).all(), float((err / ez).max())
    # gradients: dz off by |dy| (0.5 ez + 8 U) at most (|act''| <= 0.5 for silu)
    edz = dyd.abs() * (0.5 * ez + 8 * U) if act == "silu" else dyd.abs() * 2 * U
    adz = dyd.abs() * 1.1
    n_sum = x.shape[0] * xd.shape[2]
    more = (16 + min(n_sum, 256)) * U      # roundings of a blocked sum
    for got, ref, lim in ((db, want[2], (edz + more * adz).sum((0, 2))),
                          (dw, want[1], ((edz + more * adz) * xh.reshape(xd.shape) + adz * e.reshape(xd.shape)).sum((0, 2)))):
        err = (got.double().cpu() - ref).abs()
        assert (err <= lim + 1e-30).all(), float((err / lim).max())
    gw_ = wd.abs()[None, :, None]
    dh, edh = (adz * gw_).reshape(xg.shape), ((edz + 4 * U * adz) * gw_).reshape(xg.shape)
    avg = lambda t: t.mean((2, 3), keepdim=True)  # noqa: E731
    lim = rstd * (edh + avg(edh + more * dh) + (xh * avg((edh + more * dh) * xh + dh * e) + e * avg(dh * xh)) + 64 * U * (dh + avg(dh) + xh * avg(dh * xh)))
    err = (flat(dx).double().cpu() - want[0]).abs()
    assert (err <= lim.reshape(xd.shape) + out * want[0].abs() + 1e-30).all(), float((err / lim.reshape(xd.shape)).max())
    return y


SHAPES = [((3, 12, 5, 4), 4), ((2, 32, 20, 20), 8), ((5, 64, 9, 9), 8), ((4, 64, 7, 7), 1), ((3, 6, 3, 3), 6), ((7, 512), 8), ((1, 4096, 2), 16),
          ((9, 35, 6, 5), 5), ((2, 48, 84, 84), 6), ((700, 16, 2, 3), 2), ((3, 33, 11), 1), ((2, 5, 1, 9), 5), ((2, 1000, 3, 3), 125), ((1300, 64), 4),
          ((1, 32, 150, 149), 4), ((2, 20, 1, 1), 2)]


@pytest.mark.parametrize("u8", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape, groups", SHAPES)
def test_norm_and_gradients(shape, groups, dtype, u8):
    x, w, b, dy = norm_case(shape, groups, dtype, seed=len(shape) + shape[1])
    check_norm(x, groups, w, b, dy, ("silu", "none")[(shape[0] + shape[1]) % 2], u8)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("u8", [False, True])
def test_norm_with_relu_away_from_zero(u8, dtype):
    """dy is zero where |z| is near 0: there the side that rounding picks decides."""
    shape, groups = (4, 24, 8, 7), 3
    x, w, b, dy = norm_case(shape, groups, dtype, seed=21)
    f = x.reshape(4, 24, -1)
    kept = mo.codes(f.float(), groups).double() if u8 else f.double()
    _, mean, rstd = mo.norm_parts(f.double(), groups, 1e-5)
    z = ((kept.reshape(4, groups, 8, -1) - mean) * rstd).reshape(f.shape) * w.double()[None, :, None] + b.double()[None, :, None]
    dy = torch.where(z.reshape(shape).abs() < 1e-3, torch.zeros_like(dy), dy)
    check_norm(x, groups, w, b, dy, "relu", u8)


def test_norm_without_weight_and_bias_and_forward_alone():
    x, _, _, dy = norm_case((4, 32, 6, 6), 4, torch.float32, seed=22)
    one, zero = torch.ones(32), torch.zeros(32)
    y = check_norm(x, 4, one, zero, dy, "silu")
    gx = last_dense(x.to(DEV))
    with torch.no_grad():
        assert torch.equal(ops.group_norm_act(gx, 4), y)
    gx.requires_grad_()
    z = ops.group_norm_act(gx, 4)
    a = torch.autograd.grad(z, gx, last_dense(dy.to(DEV)))[0]
    z = ops.group_norm_act(gx, 4, one.to(DEV), zero.to(DEV))
    assert torch.equal(a, torch.autograd.grad(z, gx, last_dense(dy.to(DEV)))[0])


def test_norm_of_offset_and_constant_groups():
    x, w, b, dy = norm_case((3, 16, 9, 9), 4, torch.float32, seed=23, mean=0.0, spread=1.0)
    check_norm(x + 1000.0, 4, w, b, dy, "none")
    x[1, 4:8] = 3.25
    for u8 in (False, True):
        check_norm(x, 4, w, b, dy, "silu", u8)


def test_norm_of_sliced_and_misaligned_samples():
    x, w, b, dy = norm_case((8, 24, 5, 5), 3, torch.bfloat16, seed=24)
    y = check_norm(x[::2], 3, w, b, dy[::2], "silu")
    gx = last_dense(x.to(DEV))[::2]
    assert torch.equal(ops.group_norm_act(gx, 3, w.to(DEV), b.to(DEV)), y)

    def off_by_one(t):
        t = t.movedim(1, -1).contiguous()
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape).copy_(t).movedim(-1, 1)

    for u8 in (False, True):
        check_norm(x[::2], 3, w, b, dy[::2], "silu", u8, put=off_by_one)


def test_norm_gradient_of_a_broadcast_sum():
    x, w, b, _ = norm_case((4, 8, 3, 3), 2, torch.float32, seed=25)
    gx = last_dense(x.to(DEV)).requires_grad_()
    ops.group_norm_act(gx, 2, w.to(DEV), b.to(DEV)).sum().backward()
    want = mo.norm_backward(x.reshape(4, 8, 9).double(), 2, w.double(), b.double(), 1e-5, "silu", torch.ones(4, 8, 9, dtype=torch.float64))[0]
    assert torch.allclose(gx.grad.reshape(4, 8, 9).double().cpu(), want, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("u8", [False, True])
def test_norm_keeps_bad_values_in_their_sample_and_group(bad, u8):
    x, w, b, dy = norm_case((3, 16, 6, 6), 4, torch.float32, seed=26)
    how = dict(act="silu", checkpoint="u8" if u8 else "full")
    gw, gb, gd = w.to(DEV), b.to(DEV), last_dense(dy.to(DEV))
    a = last_dense(x.to(DEV)).requires_grad_()
    ya = ops.group_norm_act(a, 4, gw, gb, **how)
    x[1, 5, 2, 2] = bad
    c = last_dense(x.to(DEV)).requires_grad_()
    yc = ops.group_norm_act(c, 4, gw, gb, **how)
    da, dc = torch.autograd.grad(ya, a, gd)[0], torch.autograd.grad(yc, c, gd)[0]
    ok = torch.ones(3, 16, dtype=torch.bool)
    ok[1, 4:8] = False
    assert torch.equal(ya.detach()[ok], yc.detach()[ok]) and torch.equal(da[ok], dc[ok])
    assert yc.detach()[1, 4:8].isnan().all() and dc[1, 4:8].isnan().all()


def test_norm_same_bits_again_and_empty_calls():
    x, w, b, dy = norm_case((600, 32, 6, 6), 4, torch.bfloat16, seed=27)
    runs = []
    for _ in range(2):
        gx, gw, gb = last_dense(x.to(DEV)).requires_grad_(), w.to(DEV).requires_grad_(), b.to(DEV).requires_grad_()
        y = ops.group_norm_act(gx, 4, gw, gb, checkpoint="u8")
        runs.append((y, *torch.autograd.grad(y, (gx, gw, gb), last_dense(dy.to(DEV)))))
    for one, two in zip(*runs):
        assert torch.equal(one, two)
    for shape in ((0, 8, 3, 3), (3, 8, 0, 5)):
        e = torch.zeros(shape, device=DEV).contiguous(memory_format=torch.channels_last).requires_grad_()
        w = torch.ones(8, device=DEV, requires_grad=True)
        y = ops.group_norm_act(e, 2, w)
        y.sum().backward()
        assert y.shape == shape and (w.grad == 0).all()


def test_norm_past_32_bit_offsets():
    """A last sample whose offset passes 2^31 elements."""
    c, far = 8, 2 ** 31 + 32
    buf = torch.zeros(far + 4 * c, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((2, c, 4), (far, 1, c))
    r = torch.Generator().manual_seed(28)
    v = torch.randn((2, c, 4), generator=r).to(torch.bfloat16).to(DEV)
    x.copy_(v)
    assert torch.equal(ops.group_norm_act(x, 2), ops.group_norm_act(last_dense(v), 2))


def test_norm_gradient_against_differences():
    """L(x + e u) - L(x - e u) over 2 e, e = 2^-6: the third-order term is e^2 |L'''| / 6 and float32 rounding of L is
    divided by e, together well under 1 % of a derivative of this size."""
    x, w, b, dy = norm_case((2, 16, 6, 6), 4, torch.float32, seed=29)
    u = torch.randn(x.shape, generator=torch.Generator().manual_seed(30))
    w, b, dy = w.to(DEV), b.to(DEV), last_dense(dy.to(DEV))
    gx = last_dense(x.to(DEV)).requires_grad_()
    dx = torch.autograd.grad(ops.group_norm_act(gx, 4, w, b), gx, dy)[0]
    loss = lambda t: (ops.group_norm_act(last_dense(t.to(DEV)), 4, w, b).double() * dy).sum()  # noqa: E731
    e = 2.0 ** -6
    got, want = float(loss(x + e * u) - loss(x - e * u)) / (2 * e), float((dx.double().cpu() * u).sum())
    assert abs(got - want) <= 0.01 * float(dx.double().norm().cpu() * u.double().norm()) / (u.numel() ** 0.5)


def test_attention_gradient_against_differences():
    """o and the last state are linear in each input, so a difference of any size is exact up to rounding."""
    c = make(2, 100, 2, 64, torch.float32, 0.03, True, seed=31)
    got = on_gpu(c)
    size = oracle(c, 0.125, True)
    g, reset = c["g"].to(DEV), c["reset"].to(DEV)

    def loss(**y):
        z = {**c, **y}
        o, last = ops.decay_attention(*(z[x].to(DEV) for x in ("q", "k", "v")), g, reset=reset, state=z["state"].to(DEV))
        return float((o.double().cpu() * c["do"]).sum() + (last.double().cpu() * c["dlast"]).sum())

    total = float((size["o"] * c["do"].abs()).sum() + (size["last"] * c["dlast"].abs()).sum())
    for name, d in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("state", "ds")):
        u = c[name].sign()   # as large as the input: L(x + u) and L(x - u) stay of L's size
        diff = loss(**{name: c[name] + u}) - loss(**{name: c[name] - u})
        want = 2 * float((got[d].double().cpu() * u).sum())
        assert abs(diff - want) <= 8 * (64 + 100 + 16) * 2.0 ** -23 * total, name


def test_norm_refusals():
    x = torch.zeros(2, 8, 4, 4, device=DEV).contiguous(memory_format=torch.channels_last)
    w = torch.ones(8, device=DEV)
    for args, kw, said in (((x[0, 0, 0], 2), {}, r"\(N, C"), ((x.half(), 2), {}, "float32 or bfloat16"), ((x, 3), {}, "groups"), ((x, 0), {}, "groups"),
                           ((x.contiguous(), 2), {}, "channels-last"), ((x, 2, w[:4]), {}, "weight"), ((x, 2, w, w.double()), {}, "bias"),
                           ((x, 2), dict(act="gelu"), "act"), ((x, 2), dict(checkpoint="u4"), "checkpoint"),
                           ((torch.zeros(1, 5000, device=DEV), 1), {}, "channels must be")):
        with pytest.raises(ValueError, match=said):
            ops.group_norm_act(*args, **kw)
