"""Operators of a policy with memory, on the library's kernels (`include/fme.h`): decayed linear attention over whole
rollouts and one token at a time, and group norm with an activation for channels-last activations.

    o, state = decay_attention(q, k, v, log_decay, reset=done, state=state)      # (N, T, H, D); learning
    o = decay_attention_step(q, k, v, log_decay, state, reset=done)              # (N, H, D); acting, state in place
    y = group_norm_act(x, groups, weight, bias, act="silu", checkpoint="u8")     # (N, C, H, W), channels last

All of them run on the caller's current stream, allocate through torch, take float32 and bfloat16, and compute in 32
bits. `decay_attention` and `group_norm_act` have gradients (once differentiable); sums are taken in a fixed order, so the
same inputs give the same bits. There is no CPU path. The reference has no counterpart: its policy has no memory
(src/fast_mario_env/ppo/model.py:13-30).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

_DTYPES = {torch.float32: N.FME_F32, torch.bfloat16: N.FME_BF16}
_ACTS = {"none": N.FME_ACT_NONE, "relu": N.FME_ACT_RELU, "silu": N.FME_ACT_SILU}
HEAD_DIMS = (32, 64, 128)
MAX_CHANNELS = 4096


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _call(name, args, dev):
    """One library call on the current stream of dev, with dev current."""
    if torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev):
            return _call(name, args, dev)
    N.check(getattr(N.lib(), name)(ctypes.byref(args), torch.cuda.current_stream(dev).cuda_stream), name)


def _bytes(name, args, which):
    n = getattr(N.lib(), name)(ctypes.byref(args), which)
    if n < 0:
        N.check(int(n), name)
    return n


def _scratch(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _p(t):
    return None if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------- decayed attention
def _rows(x):
    """x itself if the kernels can read its rows (last axis contiguous, rows on 16-byte boundaries), else a copy."""
    e = x.element_size()
    ok = x.stride(-1) == 1 and x.data_ptr() % 16 == 0
    ok = ok and all(x.size(i) == 1 or x.stride(i) * e % 16 == 0 for i in range(x.dim() - 1))
    return x if ok else x.clone(memory_format=torch.contiguous_format)


def _t4(x):
    """(pointer, strides) of an (N, T, H, D) tensor; the stride of an axis of one element is not used and given as 0."""
    s = x.stride()
    return (x.data_ptr(), s[0] if x.size(0) > 1 else 0, s[1] if x.size(1) > 1 else 0, s[2] if x.size(2) > 1 else 0)


_NO4 = (None, 0, 0, 0)


def _check_qkv(q, k, v, log_decay, reset, state, lead):
    _need(q.is_cuda, "decay attention runs on a CUDA device (there is no CPU path)")
    _need(q.dim() == lead + 2, f"q must have {lead + 2} axes")
    _need(q.dtype in _DTYPES, "q must be float32 or bfloat16")
    for x, name in ((k, "k"), (v, "v")):
        _need(x.shape == q.shape, f"{name} must have q's shape {tuple(q.shape)}")
        _need(x.dtype == q.dtype and x.device == q.device, f"{name} must have q's dtype and device")
    h, d = q.shape[-2], q.shape[-1]
    _need(d in HEAD_DIMS, f"the head size must be one of {HEAD_DIMS}")
    _need(h >= 1, "at least one head is needed")
    _need(log_decay.shape == (h,) and log_decay.dtype == torch.float32 and log_decay.device == q.device,
          f"log_decay must be a float32 ({h},) tensor on q's device")
    _need(not log_decay.requires_grad, "log_decay is fixed for each head: it has no gradient")
    if reset is not None:
        _need(reset.shape == q.shape[:lead], f"reset must have shape {tuple(q.shape[:lead])}")
        _need(reset.dtype in (torch.bool, torch.uint8) and reset.device == q.device, "reset must be bool or uint8 on q's device")
    if state is not None:
        _need(state.shape == (q.shape[0], h, d, d) and state.dtype == torch.float32 and state.device == q.device,
              f"state must be a float32 {(q.shape[0], h, d, d)} tensor on q's device")


def _attn_args(q, k, v, o, log_decay, reset, s_in, s_out, scale):
    n, t, h, d = q.shape
    return N.FmeDecayAttn(n, t, h, d, _DTYPES[q.dtype], scale, _t4(q), _t4(k), _t4(v), _t4(o), log_decay.data_ptr(),
                          _p(reset), 0 if reset is None else reset.stride(0), 0 if reset is None else reset.stride(1),
                          _p(s_in), _p(s_out))


def _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, keep):
    """o, the state after the last token, and what the backward pass wants of the states in between."""
    n, t, h, d = q.shape
    o = torch.empty_like(q)
    if o.stride() != q.stride():      # q had a shared or overlapping axis
        o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    last = torch.empty((n, h, d, d), dtype=torch.float32, device=q.device) if return_state else None
    a = _attn_args(q, k, v, o, log_decay, reset, state, last, scale)
    ws = _scratch(_bytes("fme_decay_attn_bytes", a, 0), q.device)
    saved = _scratch(_bytes("fme_decay_attn_bytes", a, 2), q.device) if keep else None
    a.saved, a.ws, a.ws_bytes = _p(saved), _p(ws), 0 if ws is None else ws.numel()
    _call("fme_decay_attn_fwd", a, q.device)
    return o, last, saved


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, reset, state, scale, return_state):
        ctx.set_materialize_grads(False)
        o, last, saved = _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, True)
        ctx.save_for_backward(q, k, v, log_decay, reset, state, saved)
        ctx.scale = scale
        return o, last

    @staticmethod
    @once_differentiable
    def backward(ctx, do, dlast):
        q, k, v, log_decay, reset, state, saved = ctx.saved_tensors
        do = torch.zeros_like(q) if do is None else _rows(do)
        dlast = None if dlast is None else dlast.contiguous()
        dq, dk, dv = (torch.empty(q.shape, dtype=q.dtype, device=q.device) for _ in range(3))
        ds = torch.empty_like(state) if state is not None and ctx.needs_input_grad[5] else None
        a = _attn_args(q, k, v, q, log_decay, reset, state, None, ctx.scale)
        a.d_o, a.dq, a.dk, a.dv = (N.FmeAttnTensor(*_t4(x)) for x in (do, dq, dk, dv))
        ws = _scratch(_bytes("fme_decay_attn_bytes", a, 1), q.device)
        a.ds_out, a.ds_in, a.saved, a.ws, a.ws_bytes = _p(dlast), _p(ds), _p(saved), _p(ws), 0 if ws is None else ws.numel()
        _call("fme_decay_attn_bwd", a, q.device)
        return dq, dk, dv, None, None, ds, None, None


def decay_attention(q, k, v, log_decay, *, reset=None, state=None, scale=None, return_state=True):
    """Decayed linear attention over N sequences of T tokens:

        S_t = (0 where reset[n, t] else exp(log_decay[h]) S_{t-1}) + k_t v_t^T,      o_t = scale * q_t S_t

    q, k, v: (N, T, H, D), float32 or bfloat16, D one of 32, 64, 128, any strides (a time-major rollout is passed as a
    transposed view, heads that are shared as an expanded one). log_decay: (H,) float32, <= 0, without a gradient.
    reset: (N, T) bool or uint8, set where a token starts an episode (the rollout's `done`). state: (N, H, D, D) float32
    before the first token, default zeros. scale: default D ** -0.5. Returns (o, state after the last token), the state
    None unless return_state. Gradients for q, k, v and state."""
    _check_qkv(q, k, v, log_decay, reset, state, 2)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, reset, state, scale, return_state)
    o, last, _ = _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, False)
    return o, last


@torch.no_grad()
def decay_attention_step(q, k, v, log_decay, state, *, reset=None, scale=None, out=None):
    """One token of `decay_attention` for each of N envs, for acting: q, k, v (N, H, D), reset (N,), and state
    (N, H, D, D) float32 contiguous, which is updated in place. Returns o (N, H, D), in `out` where given. No gradient."""
    _check_qkv(q, k, v, log_decay, reset, state, 1)
    _need(state is not None and state.is_contiguous(), "state must be contiguous: it is updated in place")
    n, h, d = q.shape
    if out is None:
        out = torch.empty((n, h, d), dtype=q.dtype, device=q.device)
    else:
        _need(out.shape == q.shape and out.dtype == q.dtype and out.device == q.device and _rows(out) is out,
              "out must have q's shape, dtype and device, with 16-byte aligned rows")
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    t3 = lambda x: (x.data_ptr(), x.stride(0) if n > 1 else 0, 0, x.stride(1) if h > 1 else 0)  # noqa: E731
    a = N.FmeDecayAttn(n, 1, h, d, _DTYPES[q.dtype], d ** -0.5 if scale is None else scale, t3(q), t3(k), t3(v), t3(out),
                       log_decay.data_ptr(), _p(reset), 0 if reset is None else reset.stride(0), 0, state.data_ptr(), state.data_ptr())
    _call("fme_decay_attn_step", a, q.device)
    return out


# ---------------------------------------------------------------------------------------------- group norm
def _channels_last(x):
    """Whether each sample of x (N, C, ...) is dense with its channels innermost."""
    want = 1
    for i in (1, *range(x.dim() - 1, 1, -1)):
        if x.size(i) != 1 and x.stride(i) != want:
            return False
        want *= x.size(i)
    return True


def _like(x):
    """A dense channels-last tensor of x's shape and dtype."""
    if x.dim() == 2:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return torch.empty((x.size(0), *x.shape[2:], x.size(1)), dtype=x.dtype, device=x.device).movedim(-1, 1)


def _norm_args(x, groups, weight, bias, eps, act):
    n, c = x.shape[0], x.shape[1]
    p = 1
    for s in x.shape[2:]:
        p *= s
    a = N.FmeGroupNorm(n, p, c, groups, _DTYPES[x.dtype], act, eps)
    a.w, a.b = _p(weight), _p(bias)
    return a


def _norm_forward(x, groups, weight, bias, eps, act, keep, u8):
    a = _norm_args(x, groups, weight, bias, eps, act)
    y = _like(x)
    n, dev = x.shape[0], x.device
    a.x, a.y, a.x_sn = x.data_ptr(), y.data_ptr(), x.stride(0)
    stats = codes = None
    if keep:
        stats = torch.empty((4 if u8 else 2, n, groups), dtype=torch.float32, device=dev)
        a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * n * groups
        if u8:
            codes = torch.empty((n, a.p, a.c), dtype=torch.uint8, device=dev)
            a.codes, a.lo, a.hi = codes.data_ptr(), a.mean + 8 * n * groups, a.mean + 12 * n * groups
    ws = _scratch(_bytes("fme_group_norm_bytes", a, 0), dev)
    a.ws, a.ws_bytes = _p(ws), 0 if ws is None else ws.numel()
    _call("fme_group_norm_fwd", a, dev)
    return y, stats, codes


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, u8):
        y, stats, codes = _norm_forward(x, groups, weight, bias, eps, act, True, u8)
        ctx.save_for_backward(codes if u8 else x, weight, bias, stats)
        ctx.how = (groups, eps, act, u8)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        kept, weight, bias, stats = ctx.saved_tensors
        groups, eps, act, u8 = ctx.how
        if not _channels_last(dy):
            dy = dy.movedim(1, -1).contiguous().movedim(-1, 1)
        n, dev = dy.shape[0], dy.device
        a = _norm_args(dy, groups, weight, bias, eps, act)
        dx = _like(dy)
        a.mean, a.rstd = stats.data_ptr(), stats.data_ptr() + 4 * n * groups
        if u8:
            a.codes, a.lo, a.hi = kept.data_ptr(), a.mean + 8 * n * groups, a.mean + 12 * n * groups
        else:
            a.x, a.x_sn = kept.data_ptr(), kept.stride(0)
        a.dy, a.dy_sn, a.dx = dy.data_ptr(), dy.stride(0), dx.data_ptr()
        dw = db = None
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            dw, db = torch.empty((2, a.c), dtype=torch.float32, device=dev).unbind()
            a.dw, a.db = dw.data_ptr(), db.data_ptr()
        ws = _scratch(_bytes("fme_group_norm_bytes", a, 1), dev)
        a.ws, a.ws_bytes = _p(ws), 0 if ws is None else ws.numel()
        _call("fme_group_norm_bwd", a, dev)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None, None, None, None


def group_norm_act(x, groups, weight=None, bias=None, *, eps=1e-5, act="silu", checkpoint="full"):
    """act(group norm of x): each sample's channels in `groups` groups, normalised over the group's channels and all
    pixels, times weight plus bias (float32, (C,)), then act, one of "none", "relu", "silu".

    x: (N, C) or (N, C, ...) with channels-last memory, float32 or bfloat16; a row of (N, C) with one group a head
    normalises heads. checkpoint: what the backward pass keeps of x: "full" x itself, "u8" one byte a value, with the
    range of each (sample, group); gradients then are those at the values the codes stand for (an error of at most
    1/510 of that range). Gradients for x, weight and bias."""
    _need(x.is_cuda, "group norm runs on a CUDA device (there is no CPU path)")
    _need(x.dim() >= 2, "x must be (N, C, ...)")
    _need(x.dtype in _DTYPES, "x must be float32 or bfloat16")
    c = x.shape[1]
    _need(1 <= c <= MAX_CHANNELS, f"the number of channels must be in 1..{MAX_CHANNELS}")
    _need(isinstance(groups, int) and groups >= 1 and c % groups == 0, f"groups must divide the {c} channels")
    _need(act in _ACTS, f"act must be one of {tuple(_ACTS)}")
    _need(checkpoint in ("full", "u8"), 'checkpoint must be "full" or "u8"')
    _need(_channels_last(x), "x must have channels-last memory (x.contiguous(memory_format=torch.channels_last))")
    for t, name in ((weight, "weight"), (bias, "bias")):
        _need(t is None or (t.shape == (c,) and t.dtype == torch.float32 and t.device == x.device and t.is_contiguous()),
              f"{name} must be a contiguous float32 ({c},) tensor on x's device")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _GroupNormAct.apply(x, weight, bias, groups, eps, _ACTS[act], checkpoint == "u8")
    return _norm_forward(x, groups, weight, bias, eps, _ACTS[act], False, False)[0]
