"""Operators of a policy with memory, on the library's kernels (`include/fme.h`): decayed linear attention over whole
rollouts and one token at a time, and group norm with an activation for channels-last activations.

    o, state = decay_attention(q, k, v, log_decay, reset=done, state=state)      # (N, T, H, D); learning
    o = decay_attention_step(q, k, v, log_decay, state, reset=done)              # (N, H, D); acting, state in place
    y = group_norm_act(x, groups, weight, bias, act="silu", checkpoint="u8")     # (N, C, H, W), channels last

All of them run on the caller's current stream, allocate through torch and take float32 and bfloat16. Sums, states and
statistics are float32 and taken in a fixed order, so the same inputs give the same bits; `decay_attention` says what its
matrix products round. `decay_attention` and `group_norm_act` have gradients (once differentiable). Forward-mode derivatives are
refused; `torch.jit.trace` records a call as a call. There is no CPU path. The reference has no counterpart: its policy has no memory
(src/fast_mario_env/ppo/model.py:13-30).
"""
from __future__ import annotations

import ctypes
import sys
from functools import lru_cache

import torch
import torch.autograd.forward_ad as _fw
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

from . import _native as N

_DTYPES = {torch.float32: N.FME_F32, torch.bfloat16: N.FME_BF16}
_ACTS = {"none": N.FME_ACT_NONE, "relu": N.FME_ACT_RELU, "silu": N.FME_ACT_SILU}
HEAD_DIMS = (32, 64, 128)
MAX_CHANNELS = 4096
_fns = {}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice
_modes = torch._C._len_torch_dispatch_stack


def _followed(size, *tensors):
    """Whether forward-mode differentiation or torch.jit.trace follows this call. To both, an output that a kernel writes is
    an empty tensor without a history; the autograd function refuses the one and stands in the other's record as a call.
    make_fx looks inside that function too, so it is refused here. size: one of an argument's sizes, a tensor while a trace is
    recorded and a plain int otherwise (asking torch for the trace takes 0.1 us of a call of 13)."""
    if type(size) is int and _fw._current_level < 0 and not _modes():
        return False
    if _modes():
        proxies = sys.modules.get("torch.fx.experimental.proxy_tensor")
        if proxies is not None and proxies.get_proxy_mode() is not None:
            raise RuntimeError("make_fx cannot record this operator: it would replay its outputs empty")
    return type(size) is not int or _fw._current_level >= 0 and any(t is not None and _fw.unpack_dual(t).tangent is not None for t in tensors)


def _call(name, args, index):
    """One library call (args: the packed structure) on the current stream of device `index`, with that device current."""
    if _current() != index:
        with torch.cuda.device(index):
            return _call(name, args, index)
    f = _fns.get(name)
    if f is None:
        f = _fns[name] = getattr(N.lib(), name)
    rc = f(args, _raw_stream(index))
    if rc:
        N.check(rc, name)


def _size(name, args, which):
    n = getattr(N.lib(), name)(ctypes.byref(args), which)
    if n < 0:
        N.check(int(n), name)
    return n


def _scratch(nbytes, dev):
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _ptr(t):
    return 0 if t is None else t.data_ptr()


# ---------------------------------------------------------------------------------------------- decayed attention
def _rows(x):
    """x itself if the kernels can read its rows (last axis contiguous, rows on 16-byte boundaries), else a copy."""
    if x.data_ptr() & 15 == 0:
        if x.is_contiguous():
            return x
        e = x.element_size()
        if x.stride(-1) == 1 and all(x.size(i) == 1 or x.stride(i) * e % 16 == 0 for i in range(x.dim() - 1)):
            return x
    return x.clone(memory_format=torch.contiguous_format)


def _matrices(x):
    """x itself if it is contiguous on a 16-byte boundary, else a copy (a state, or its gradient)."""
    return x if x.is_contiguous() and x.data_ptr() & 15 == 0 else x.clone(memory_format=torch.contiguous_format)


def _t4(x):
    """(pointer, strides) of an (N, T, H, D) tensor; the stride of an axis of one element is not used and given as 0."""
    n, t, h, _ = x.shape
    sn, st, sh, _ = x.stride()
    return x.data_ptr(), sn if n > 1 else 0, st if t > 1 else 0, sh if h > 1 else 0


_NO4 = (0, 0, 0, 0)


def _check_qkv(q, k, v, log_decay, reset, state, lead):
    if not q.is_cuda:
        raise ValueError("decay attention runs on a CUDA device (there is no CPU path)")
    shape, dtype, dev = q.shape, q.dtype, q.get_device()
    if len(shape) != lead + 2:
        raise ValueError(f"q must have {lead + 2} axes")
    if dtype not in _DTYPES:
        raise ValueError("q must be float32 or bfloat16")
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"k and v must have q's shape {tuple(shape)}")
    if k.dtype != dtype or v.dtype != dtype or k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k and v must have q's dtype and device")
    n, h, d = shape[0], shape[-2], shape[-1]
    if d not in HEAD_DIMS:
        raise ValueError(f"the head size must be one of {HEAD_DIMS}")
    if h < 1:
        raise ValueError("at least one head is needed")
    if log_decay.shape != (h,) or log_decay.dtype != torch.float32 or log_decay.get_device() != dev:
        raise ValueError(f"log_decay must be a float32 ({h},) tensor on q's device")
    if log_decay.requires_grad:
        raise ValueError("log_decay is fixed for each head: it has no gradient")
    if reset is not None:
        if reset.shape != shape[:lead]:
            raise ValueError(f"reset must have shape {tuple(shape[:lead])}")
        if reset.dtype not in (torch.bool, torch.uint8) or reset.get_device() != dev:
            raise ValueError("reset must be bool or uint8 on q's device")
    if state is not None and (state.shape != (n, h, d, d) or state.dtype != torch.float32 or state.get_device() != dev):
        raise ValueError(f"state must be a float32 {(n, h, d, d)} tensor on q's device")


@lru_cache(maxsize=4096)
def _attn_sizes(n, t, h, d, dtype):
    """Bytes of the forward workspace, the backward workspace, and of what the forward pass keeps for the backward pass."""
    a = N.FmeDecayAttn(n=n, t=t, h=h, d=d, dtype=dtype)
    return tuple(_size("fme_decay_attn_bytes", a, i) for i in range(3))


def _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, keep):
    """o, the state after the last token, and what the backward pass wants of the states in between."""
    n, t, h, d = q.shape
    dev, dtype = q.device, _DTYPES[q.dtype]
    o = torch.empty_like(q)
    if not q.is_contiguous() and o.stride() != q.stride():      # q had a shared or overlapping axis
        o = torch.empty(q.shape, dtype=q.dtype, device=dev)
    last = torch.empty((n, h, d, d), dtype=torch.float32, device=dev) if return_state else None
    sizes = _attn_sizes(n, t, h, d, dtype)
    ws = _scratch(sizes[0], dev)
    saved = _scratch(sizes[2], dev) if keep else None
    rs = (0, 0) if reset is None else reset.stride()
    _call("fme_decay_attn_fwd",
          N.ATTN.pack(n, t, h, d, dtype, scale, *_t4(q), *_t4(k), *_t4(v), *_t4(o), log_decay.data_ptr(), _ptr(reset), *rs, _ptr(state), _ptr(last),
                      *_NO4, *_NO4, *_NO4, *_NO4, 0, 0, _ptr(saved), _ptr(ws), sizes[0]), q.get_device())
    return o, last, saved


def _attn_backward(ctx, do, dlast):
    q, k, v, log_decay, reset, state, saved = ctx.saved_tensors
    q, k, v = _rows(q), _rows(k), _rows(v)   # a hook on saved tensors may hand them back in another layout
    n, t, h, d = q.shape
    dev, dtype = q.device, _DTYPES[q.dtype]
    do = torch.zeros_like(q) if do is None else _rows(do)
    dlast = None if dlast is None else _matrices(dlast)
    state = None if state is None else _matrices(state)
    if q.is_contiguous():
        dq, dk, dv = torch.empty_like(q), torch.empty_like(q), torch.empty_like(q)
    else:
        dq, dk, dv = (torch.empty(q.shape, dtype=q.dtype, device=dev) for _ in range(3))
    ds = torch.empty_like(state) if state is not None and ctx.needs_input_grad[5] else None
    sizes = _attn_sizes(n, t, h, d, dtype)
    ws = _scratch(sizes[1], dev)
    rs = (0, 0) if reset is None else reset.stride()
    _call("fme_decay_attn_bwd",
          N.ATTN.pack(n, t, h, d, dtype, ctx.scale, *_t4(q), *_t4(k), *_t4(v), *_NO4, log_decay.data_ptr(), _ptr(reset), *rs, _ptr(state), 0,
                      *_t4(do), *_t4(dq), *_t4(dk), *_t4(dv), _ptr(dlast), _ptr(ds), _ptr(saved), _ptr(ws), sizes[1]), q.get_device())
    return dq, dk, dv, None, None, ds, None, None


_attn_backward_once = once_differentiable(_attn_backward)


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, reset, state, scale, return_state):
        ctx.set_materialize_grads(False)
        o, last, saved = _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, True)
        ctx.save_for_backward(q, k, v, log_decay, reset, state, saved)
        ctx.scale = scale
        return o, last

    @staticmethod
    def backward(ctx, do, dlast):   # under create_graph a second derivative has to be refused
        return (_attn_backward_once if torch.is_grad_enabled() else _attn_backward)(ctx, do, dlast)


def decay_attention(q, k, v, log_decay, *, reset=None, state=None, scale=None, return_state=True):
    """Decayed linear attention over N sequences of T tokens:

        S_t = (0 where reset[n, t] else exp(log_decay[h]) S_{t-1}) + k_t v_t^T,      o_t = scale * q_t S_t

    q, k, v: (N, T, H, D), float32 or bfloat16, D one of 32, 64, 128, any strides (a time-major rollout is passed as a
    transposed view, heads that are shared as an expanded one). log_decay: (H,) float32, <= 0, without a gradient.
    reset: (N, T) bool or uint8, set where a token starts an episode (the rollout's `done`). state: (N, H, D, D) float32
    before the first token, default zeros. scale: default D ** -0.5. Returns (o, state after the last token), the state
    None unless return_state. Gradients for q, k, v and state.

    Products are taken by the matrix units and summed in float32. float32 operands count with 22 bits (error of a result
    at most 6e-7 of its norm over the sizes measured, 2e-7 to 4e-7 being that of sums in float32). With bfloat16 tensors what a product reads is rounded to bfloat16: the scores, and the state
    (a given one too, and its gradient) where q, k, v or a gradient meets it (error about 0.0024 of a result's norm, of
    which its own rounding is 0.0017); tokens enter a state with 16 bits, with 24 where the state or its gradient is asked for.

    A call that a backward pass follows keeps a state for every 64 tokens (32 with D = 32, and with D = 128 in float32),
    in the tensors' type: 1, 1 or 2 (float32: 1, 1 or 4) times q's memory for D = 32, 64 or 128."""
    _check_qkv(q, k, v, log_decay, reset, state, 2)
    d = q.shape[-1]
    scale = float(d ** -0.5 if scale is None else scale)
    follow = _followed(d, q, k, v, log_decay, state)
    q, k, v, log_decay = _rows(q), _rows(k), _rows(v), log_decay.contiguous()
    if state is not None:
        state = _matrices(state)
    if follow or torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or (state is not None and state.requires_grad)):
        return _DecayAttention.apply(q, k, v, log_decay, reset, state, scale, return_state)
    o, last, _ = _attn_forward(q, k, v, log_decay, reset, state, scale, return_state, False)
    return o, last


def decay_attention_step(q, k, v, log_decay, state, *, reset=None, scale=None, out=None):
    """One token of `decay_attention` for each of N envs, for acting: q, k, v (N, H, D), reset (N,), and state
    (N, H, D, D) float32 contiguous, which is updated in place. Returns o (N, H, D), in `out` where given
    (which may be q, k or v itself, but may not overlap them or the state otherwise). No gradient."""
    _check_qkv(q, k, v, log_decay, reset, state, 1)
    if state is None or not state.is_contiguous() or state.requires_grad:
        raise ValueError("state must be contiguous and without a gradient: it is updated in place")
    s = state.data_ptr()
    if s & 15:
        raise ValueError("state must start on a 16-byte boundary: it is updated in place")
    n, h, d = q.shape
    if _followed(n, q, k, v, log_decay, state):
        raise RuntimeError("a step has no forward-mode derivative and leaves no trace: it updates its state in place")
    if out is None:
        out = torch.empty((n, h, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.get_device() != q.get_device() or _rows(out) is not out:
        raise ValueError("out must have q's shape, dtype and device, with 16-byte aligned rows")
    elif _shares_memory(out):
        raise ValueError("rows of out must not overlap")
    q, k, v = _rows(q), _rows(k), _rows(v)
    log_decay = log_decay.contiguous()
    _call("fme_decay_attn_step",
          N.ATTN.pack(n, 1, h, d, _DTYPES[q.dtype], d ** -0.5 if scale is None else scale, *_t3(q), *_t3(k), *_t3(v), *_t3(out), log_decay.data_ptr(),
                      _ptr(reset), 0 if reset is None else reset.stride(0), 0, s, s, *_NO4, *_NO4, *_NO4, *_NO4, 0, 0, 0, 0, 0), q.get_device())
    increment_version((state, out))   # a backward pass that kept either notices
    return out


def _shares_memory(x):
    """Whether two rows of an (n, h, d) tensor overlap: n CTAs would write one place in no order."""
    n, h, d = x.shape
    sn, sh = (x.stride(0) if n > 1 else 0), (x.stride(1) if h > 1 else 0)
    if (n == 1 or sn >= (h - 1) * sh + d) and (h == 1 or sh >= d) or (h == 1 or sh >= (n - 1) * sn + d) and (n == 1 or sn >= d):
        return False
    if n > 1 and sn == 0:
        return True
    # rows i sn + j sh: some difference of two, j heads and as many sequences as come nearest, is less than a row
    return any(abs(i * sn - j * sh) < d for j in range(h) for i in ((j * sh // sn, j * sh // sn + 1) if n > 1 else (0,)) if (i or j) and i < n)


def _t3(x):
    n, h, _ = x.shape
    sn, sh, _ = x.stride()
    return x.data_ptr(), sn if n > 1 else 0, 0, sh if h > 1 else 0


# ---------------------------------------------------------------------------------------------- group norm
def _channels_last(x):
    """Whether each sample of x (N, C, ...) is dense with its channels innermost."""
    if x.dim() == 4 and x.is_contiguous(memory_format=torch.channels_last) or x.dim() == 2 and x.is_contiguous():
        return True
    want = 1
    for i in (1, *range(x.dim() - 1, 1, -1)):
        if x.size(i) != 1 and x.stride(i) != want:
            return False
        want *= x.size(i)
    return True


def _relaid(x):
    """x itself if it has channels-last memory, else a copy that does."""
    return x if _channels_last(x) else x.movedim(1, -1).contiguous().movedim(-1, 1)


def _like(x):
    """A dense channels-last tensor of x's shape and dtype."""
    if x.dim() == 4:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device, memory_format=torch.channels_last)
    if x.dim() == 2:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    return torch.empty((x.size(0), *x.shape[2:], x.size(1)), dtype=x.dtype, device=x.device).movedim(-1, 1)


def _pixels(shape):
    p = 1
    for s in shape[2:]:
        p *= s
    return p


@lru_cache(maxsize=4096)
def _norm_size(n, p, c, groups, dtype, u8, x_aligned, x_sn, dy_aligned, dy_sn, which):
    """Workspace bytes of a call; they depend on whether x and dy can be read in 16-byte pieces."""
    at = lambda ok: 256 if ok else 257  # noqa: E731
    a = N.FmeGroupNorm(n=n, p=p, c=c, g=groups, dtype=dtype, x=at(x_aligned), x_sn=x_sn, dy=at(dy_aligned), dy_sn=dy_sn, y=256, dx=256,
                       codes=256 if u8 else None)
    return _size("fme_group_norm_bytes", a, which)


def _norm_forward(x, groups, weight, bias, eps, act, keep, u8):
    shape = x.shape
    n, c, p = shape[0], shape[1], _pixels(shape)
    dtype, dev, xp, sn = _DTYPES[x.dtype], x.device, x.data_ptr(), x.stride(0)
    y = _like(x)
    stats = codes = None
    mean = codes_p = lo = 0
    if keep:      # rows: mean, rstd, and the ranges of the codes
        stats = torch.empty((4 if u8 else 2) * n * groups, dtype=torch.float32, device=dev)
        mean = stats.data_ptr()
        if u8:
            codes = torch.empty(n * p * c, dtype=torch.uint8, device=dev)
            codes_p, lo = codes.data_ptr(), mean + 8 * n * groups
    need = _norm_size(n, p, c, groups, dtype, u8, xp & 15 == 0, sn, True, 0, 0)
    ws = _scratch(need, dev)
    _call("fme_group_norm_fwd",
          N.NORM.pack(n, p, c, groups, dtype, act, eps, xp, sn, 0, y.data_ptr(), _ptr(weight), _ptr(bias), mean, mean and mean + 4 * n * groups, codes_p,
                      lo, lo and lo + 4 * n * groups, 0, 0, 0, 0, _ptr(ws), need), x.get_device())
    return y, stats, codes


def _norm_backward(ctx, dy):
    kept, weight, bias, stats = ctx.saved_tensors
    groups, eps, act, u8 = ctx.how
    dy = _relaid(dy)
    if not u8:
        kept = _relaid(kept)   # a hook on saved tensors (pinned offloading) may hand it back in another layout
    shape = dy.shape
    n, c, p = shape[0], shape[1], _pixels(shape)
    dtype, dev, dyp, dy_sn, mean = _DTYPES[dy.dtype], dy.device, dy.data_ptr(), dy.stride(0), stats.data_ptr()
    dx = _like(dy)
    if u8:
        xp, x_sn, codes, lo = 0, 0, kept.data_ptr(), mean + 8 * n * groups
    else:
        xp, x_sn, codes, lo = kept.data_ptr(), kept.stride(0), 0, 0
    need = _norm_size(n, p, c, groups, dtype, u8, xp & 15 == 0, x_sn, dyp & 15 == 0, dy_sn, 1)
    wants_w, wants_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
    dw = db = None
    dwp = 0
    if wants_w or wants_b:
        dw, db = torch.empty((2, c), dtype=torch.float32, device=dev).unbind()
        dwp = dw.data_ptr()
    ws = _scratch(need, dev)
    _call("fme_group_norm_bwd",
          N.NORM.pack(n, p, c, groups, dtype, act, eps, xp, x_sn, dy_sn, 0, _ptr(weight), _ptr(bias), mean, mean + 4 * n * groups, codes, lo,
                      lo and lo + 4 * n * groups, dyp, dx.data_ptr(), dwp, dwp and dwp + 4 * c, _ptr(ws), need), dy.get_device())
    return dx, dw if wants_w else None, db if wants_b else None, None, None, None, None


_norm_backward_once = once_differentiable(_norm_backward)


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, u8):
        y, stats, codes = _norm_forward(x, groups, weight, bias, eps, act, True, u8)
        ctx.save_for_backward(codes if u8 else x, weight, bias, stats)
        ctx.how = (groups, eps, act, u8)
        return y

    @staticmethod
    def backward(ctx, dy):
        return (_norm_backward_once if torch.is_grad_enabled() else _norm_backward)(ctx, dy)


def group_norm_act(x, groups, weight=None, bias=None, *, eps=1e-5, act="silu", checkpoint="full"):
    """act(group norm of x): each sample's channels in `groups` groups, normalised over the group's channels and all
    pixels, times weight plus bias (float32, (C,)), then act, one of "none", "relu", "silu".

    x: (N, C) or (N, C, ...) with channels-last memory, float32 or bfloat16; a row of (N, C) with one group a head
    normalises heads. checkpoint: what the backward pass keeps of x: "full" x itself, "u8" one byte a value, with the
    range of each (sample, group); gradients then are those at the values the codes stand for (an error of at most
    1/510 of that range). Gradients for x, weight and bias."""
    if not x.is_cuda:
        raise ValueError("group norm runs on a CUDA device (there is no CPU path)")
    if x.dim() < 2:
        raise ValueError("x must be (N, C, ...)")
    if x.dtype not in _DTYPES:
        raise ValueError("x must be float32 or bfloat16")
    c = x.size(1)
    if not 1 <= c <= MAX_CHANNELS:
        raise ValueError(f"the number of channels must be in 1..{MAX_CHANNELS}")
    if not isinstance(groups, int) or groups < 1 or c % groups:
        raise ValueError(f"groups must divide the {c} channels")
    if act not in _ACTS:
        raise ValueError(f"act must be one of {tuple(_ACTS)}")
    if checkpoint not in ("full", "u8"):
        raise ValueError('checkpoint must be "full" or "u8"')
    if not _channels_last(x):
        raise ValueError("x must have channels-last memory (x.contiguous(memory_format=torch.channels_last))")
    grad = x.requires_grad
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            if t.shape != (c,) or t.dtype != torch.float32 or t.get_device() != x.get_device() or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous float32 ({c},) tensor on x's device")
            grad = grad or t.requires_grad
    if _followed(c, x, weight, bias) or grad and torch.is_grad_enabled():
        return _GroupNormAct.apply(x, weight, bias, groups, eps, _ACTS[act], checkpoint == "u8")
    return _norm_forward(x, groups, weight, bias, eps, _ACTS[act], False, False)[0]
