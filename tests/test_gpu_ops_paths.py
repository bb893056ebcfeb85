"""The memory policy's operators on every kernel that their sizes choose: the time axis in several joined segments (heads of each
size, more than 17 segments, values that are not numbers, a captured graph), samples split into parts, groups in a row of every
width, and calls without a plan. Each case asserts from the library's own workspace sizes that it takes the path it is for.
Error bounds are those of test_gpu_ops."""
import pytest
import torch
from conftest import fme  # noqa: F401  (loads the package)
from test_gpu_ops import DEV, bound, check_norm, compare, last_dense, make, norm_case, on_gpu, oracle

from fast_mario_env_b200 import _native as N
from fast_mario_env_b200 import ops

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])


def segments(n, t, h, d, dtype):
    """Segments of the forward and the backward pass: the workspace holds a matrix and a factor for all but one."""
    sizes = ops._attn_sizes(n, t, h, d, ops._DTYPES[dtype])
    return [s // (n * h * (4 * d * d + 4)) + 1 for s in sizes[:2]]


# ---------------------------------------------------------------------------------------------- segments
@BOTH
@pytest.mark.parametrize("carry", [True, False])
@pytest.mark.parametrize("t, h, d, least, most", [(1100, 2, 128, 3, 17), (1500, 2, 64, 3, 17), (1300, 2, 32, 3, 17), (3000, 1, 32, 18, 40), (6000, 1, 64, 18, 40)])
def test_joined_segments(t, h, d, least, most, carry, dtype):
    """Without a state asked for, decayed rows keep fewer bits and the state's gradient is not computed: other kernels."""
    assert all(least <= s <= most for s in segments(1, t, h, d, dtype))
    c = make(1, t, h, d, dtype, 0.004, carry, seed=t + d)
    if carry:
        got = on_gpu(c)
    else:
        q, k, v = (c[x].to(DEV).requires_grad_() for x in ("q", "k", "v"))
        o, last = ops.decay_attention(q, k, v, c["g"].to(DEV), reset=c["reset"].to(DEV), return_state=False)
        assert last is None
        got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, (q, k, v), c["do"].to(DEV)))))
    compare(got, oracle(c, d ** -0.5), oracle(c, d ** -0.5, True), d, t, dtype)


@BOTH
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_numbers_stay_in_their_episode_across_segments(bad, d, dtype):
    """In the first, a middle and the last segment, in the chunk of a restart and far from one, in a state and in gradients."""
    n, t, h = 2, 1500, 2
    assert min(segments(n, t, h, d, dtype)) >= 3
    c = make(n, t, h, d, dtype, None, True, seed=50)
    c["reset"] = torch.zeros(n, t, dtype=torch.bool)
    c["reset"][0, [300, 710, 1400, 1470]] = True
    c["reset"][1, 500] = True
    clean = on_gpu(c)
    c["k"][0, 40, 0, 3] = bad       # first segment
    c["k"][0, 290, 0, 1] = bad      # ten tokens before a restart
    c["v"][0, 800, 0, 5] = bad      # in the middle
    c["v"][0, 1460, 0, 5] = bad     # last segment, ten tokens before a restart
    c["state"][1, 0, 2, 2] = bad
    got = on_gpu(c)
    size = oracle({**c, **{x: c[x].nan_to_num(0, 0, 0) for x in ("k", "v", "state")}}, d ** -0.5, True)
    ok = torch.ones(n, t, h, dtype=torch.bool)
    ok[0, :300, 0] = False
    ok[0, 710:1470, 0] = False
    ok[1, :500, 0] = False
    for name in ("o", "dq", "dk", "dv"):
        err = (got[name].double().cpu() - clean[name].double().cpu()).abs()
        lim = 2 * bound(size[name], d, t, dtype)
        assert (err[ok] <= lim[ok]).all(), name
    assert got["o"][0, :40, 0].isfinite().all() and got["o"][0, 710:800, 0].isfinite().all() and got["o"][0, 1400:1460, 0].isfinite().all()
    for bad_rows in (got["o"][0, 40:300, 0], got["o"][0, 800:1400, 0], got["o"][0, 1460:1470, 0], got["o"][1, :500, 0]):
        assert not bad_rows.isfinite().all(-1).any()
    assert got["last"].isfinite().all() and got["ds"].isfinite().all()
    c = make(n, t, h, d, dtype, None, True, seed=50)
    c["reset"] = torch.zeros(n, t, dtype=torch.bool)
    c["reset"][0, [300, 710, 1400, 1470]] = True
    c["do"][0, 715, 1, 7] = bad     # five tokens after a restart
    c["do"][0, 1300, 0, 7] = bad    # an episode over several segments
    c["dlast"][1, 1, 0, 0] = bad    # the whole second sequence
    got = on_gpu(c)
    ok = torch.ones(n, t, h, dtype=torch.bool)
    ok[0, 710:716, 1] = False
    ok[0, 710:1301, 0] = False
    ok[1, :, 1] = False
    clean = on_gpu({**c, "do": c["do"].nan_to_num(0, 0, 0), "dlast": c["dlast"].nan_to_num(0, 0, 0)})
    size = oracle({**c, "do": c["do"].nan_to_num(0, 0, 0), "dlast": c["dlast"].nan_to_num(0, 0, 0)}, d ** -0.5, True)
    for name in ("dq", "dk", "dv"):
        err = (got[name].double().cpu() - clean[name].double().cpu()).abs()
        assert (err[ok] <= 2 * bound(size[name], d, t, dtype)[ok]).all(), name
    assert got["ds"][0].isfinite().all() and got["ds"][1, 0].isfinite().all()


def test_joined_segments_in_a_captured_graph():
    n, t, h, d = 2, 1500, 2, 64
    assert min(segments(n, t, h, d, torch.bfloat16)) >= 3
    c = make(n, t, h, d, torch.bfloat16, 0.004, True, seed=51)
    q, k, v, s = (c[x].to(DEV).requires_grad_() for x in ("q", "k", "v", "state"))
    g, reset, do, dl = (c[x].to(DEV) for x in ("g", "reset", "do", "dlast"))

    def work():
        o, last = ops.decay_attention(q, k, v, g, reset=reset, state=s)
        return (o, last, *torch.autograd.grad((o, last), (q, k, v, s), (do, dl)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    with torch.no_grad():
        for x in (q, k, v, s, do, dl):
            x.mul_(0.5)
        reset.logical_xor_(torch.rand(reset.shape, device=DEV) < 0.004)
    graph.replay()
    got = [x.detach().clone() for x in out]
    for a, b in zip(got, work()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------- group norm
def norm_bytes(shape, groups, dtype, u8, which, aligned=True):
    n, c = shape[:2]
    p = ops._pixels(shape)
    return ops._norm_size(n, p, c, groups, ops._DTYPES[dtype], u8, aligned, p * c, True, p * c, which)


def off_by_one(x):
    x = x.movedim(1, -1).contiguous()
    return torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape).copy_(x).movedim(-1, 1)


@BOTH
@pytest.mark.parametrize("u8", [False, True])
@pytest.mark.parametrize("shape, groups, put", [((1, 256, 84, 84), 16, last_dense), ((2, 64, 180, 180), 8, last_dense), ((2, 48, 188, 189), 16, last_dense),
                                                ((1, 33, 301, 301), 3, last_dense), ((1, 32, 330, 330), 8, off_by_one)])
def test_samples_in_parts(shape, groups, put, u8, dtype):
    """Larger than a cluster holds. Groups of whole vectors, of a power of two of them, of 3 channels; odd counts; misaligned."""
    x, w, b, dy = norm_case(shape, groups, dtype, seed=52)
    assert norm_bytes(shape, groups, dtype, u8, 0, put is last_dense) > 0
    check_norm(x, groups, w, b, dy, "silu", u8, put=put)


@BOTH
@pytest.mark.parametrize("u8", [False, True])
@pytest.mark.parametrize("shape, groups, across", [((50, 24), 6, 1), ((50, 48), 6, 1), ((40, 240), 3, 1), ((33, 640), 4, 1), ((21, 1280), 4, 1), ((9, 2048), 4, 1),
                                                   ((5, 4096), 4, 1), ((2500, 512), 1, 1), ((700, 1024), 1, 1), ((30, 1280), 16, 2), ((19, 2560), 16, 2),
                                                   ((400, 1536), 24, 2), ((18, 1920), 12, 2), ((7, 3840), 12, 2), ((5, 2048), 512, 2), ((1, 512), 1, 1)])
def test_groups_in_a_row_of_every_width(shape, groups, across, u8, dtype):
    """Groups of 1 to 128 vectors of 16 bytes, and more groups than a CTA takes (`across` CTAs for a sample, in one of the types)."""
    n, c = shape
    x, w, b, dy = norm_case(shape, groups, dtype, seed=53)
    vec = 4 if dtype == torch.float32 else 8
    wide = c // groups // vec
    if c // groups % vec == 0 and wide <= 128:
        lanes = min(32, 1 << (wide - 1).bit_length())
        per = 256 // lanes
        rows, rest = divmod(norm_bytes(shape, groups, dtype, u8, 1), 8 * c)
        assert rest == 0
        if per < groups:   # a row of dw and db for each of the CTAs across, for at most n samples at once
            assert across == 2 and rows % 2 == 0 and rows // 2 <= n
        else:
            assert rows <= -(-n // (per // groups))
    check_norm(x, groups, w, b, dy, ("silu", "none")[n % 2], u8)


@BOTH
@pytest.mark.parametrize("u8", [False, True])
@pytest.mark.parametrize("shape, groups", [((600, 515, 2), 5), ((1300, 515), 1), ((3, 1029, 5, 3), 7), ((2, 2047, 3), 2047)])
def test_calls_without_a_plan(shape, groups, u8, dtype):
    """Odd channel counts above 512, more samples than CTAs among them."""
    assert norm_bytes(shape, groups, dtype, u8, 1) == 592 * 8 * shape[1]
    x, w, b, dy = norm_case(shape, groups, dtype, seed=54)
    check_norm(x, groups, w, b, dy, "silu", u8)
