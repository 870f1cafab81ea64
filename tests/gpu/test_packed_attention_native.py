"""Native packed attention against the formula in 64 bits, with error bounds from the arithmetic."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover - collected on CPU, skipped there
    pytest.skip("needs CUDA", allow_module_level=True)

from mia_train_b200.ops._native import raise_on_device_errors  # noqa: E402
from mia_train_b200.ops.packed_attention import PackedSequences, packed_attention  # noqa: E402

DEV = torch.device("cuda", 0)
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U32 = 2.0**-23  # a step of fp32: the tensor core's sums may be cut instead of rounded


def _inputs(lq, lk, hq, hk, d, dtype, pad=0, seed=0, grad=1.0):
    gen = torch.Generator(device=DEV).manual_seed(seed + d)
    normal = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    tq, tk = sum(lq) + pad, sum(lk) + pad
    if lq is lk:
        proj = normal(tq, hq + 2 * hk, d).to(dtype)
        q, k, v = proj[:, :hq], proj[:, hq:hq + hk], proj[:, hq + hk:]
    else:
        q, k, v = normal(tq, hq, d).to(dtype), normal(tk, hk, d).to(dtype), normal(tk, hk, d).to(dtype)
    return q, k, v, (grad * normal(tq, hq, d)).to(dtype)


def _visible(m, n, causal):
    seen = torch.ones(m, n, dtype=torch.bool, device=DEV)
    return seen.tril(n - m) if causal else seen


def _expected(q, k, v, do, lq, lk, causal, scale, dtype):
    """Outputs and gradients in 64 bits and a bound on each one's error.

    u is half a step of the inputs' type, to which P, dS and the results are rounded; `rho` the relative error of a
    probability: its score (D products and their sum, times the largest score), exp2 of the multi-function unit
    (2^-22), the statistics' own rounding. fp16 adds half a step of its subnormals to every P and dS.
    """
    u = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    half = dtype == F16
    tiny = 2.0**-25 if half else 0.0
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = hq // hk
    outs = [torch.zeros(x.shape, device=DEV, dtype=torch.float64) for x in (q, q, k, v)]
    errs = [torch.zeros_like(x) for x in outs]
    # fp16 dS are scaled by a power of two near the largest |do| of the launch's tiles: at most that of all
    norm = 2 * do.double().norm(dim=-1).max().item() if do.numel() else 1.0
    a = c = 0
    for m, n in zip(lq, lk, strict=True):
        rows, cols = slice(a, a + m), slice(c, c + n)
        a, c = a + m, c + n
        if m == 0 or n == 0:
            continue
        seen = _visible(m, n, causal)
        for h in range(hq):
            x, y, w, dy = q[rows, h].double(), k[cols, h // g].double(), v[cols, h // g].double(), do[rows, h].double()
            s = (x @ y.t()) * scale
            s = torch.where(seen, s, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            o = p @ w
            dp = dy @ w.t()
            delta = (dy * o).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            size = ((x.abs() @ y.abs().t()) * abs(scale)).max().item() if m and n else 0.0
            rho = (d + 16) * U32 * size + 2.0**-18 + n * U32
            pv = p @ w.abs()
            tops = w.abs().sum(0)
            err_o = (u + rho) * pv + u * o.abs() + tiny * tops
            err_delta = (dy.abs() * err_o).sum(-1, keepdim=True) + d * U32 * (dy.abs() * o.abs()).sum(-1, keepdim=True)
            e = u * ds.abs() + rho * (ds.abs() + p * (dp.abs() + delta.abs())) + p * (
                err_delta + (d + 2) * U32 * (dy.abs() @ w.abs().t())) + tiny * 2.0**-8 * norm * seen
            outs[0][rows, h] = o
            errs[0][rows, h] = err_o
            dq = scale * (ds @ y)
            outs[1][rows, h] = dq
            errs[1][rows, h] = abs(scale) * ((e + n * U32 * ds.abs()) @ y.abs()) + u * dq.abs()
            outs[2][cols, h // g] += scale * (ds.t() @ x)
            errs[2][cols, h // g] += abs(scale) * ((e + g * m * U32 * ds.abs()).t() @ x.abs())
            outs[3][cols, h // g] += p.t() @ dy
            errs[3][cols, h // g] += (((u + rho + g * m * U32) * p + tiny * 2.0**-8 * seen).t() @ dy.abs())
    for i in (2, 3):
        errs[i] += u * outs[i].abs()
    # results below fp16's normal range are rounded to its subnormals
    return outs, [x + (2.0**-24 if half else 1e-30) for x in errs]


def _run(q, k, v, do, seq, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    o = packed_attention(*leaves, seq, scale)
    return [o.detach(), *torch.autograd.grad(o, leaves, do)]


def _compare(lq, lk, hq, hk, d, dtype, causal, pad=0, scale=None, seed=0, grad=1.0):
    q, k, v, do = _inputs(lq, lk, hq, hk, d, dtype, pad, seed, grad)
    seq = PackedSequences(lq, None if lq is lk else lk, causal=causal, device=DEV)
    got = _run(q, k, v, do, seq, scale)
    raise_on_device_errors(DEV)
    want, bound = _expected(q, k, v, do, lq, lk, causal, d**-0.5 if scale is None else scale, dtype)
    for name, x, y, b in zip(("o", "dq", "dk", "dv"), got, want, bound, strict=True):
        assert x.dtype == dtype and torch.isfinite(x).all(), name
        err = (x.double() - y).abs()
        assert (err <= b).all(), f"{name}: {(err / b).max().item():.3g} times the bound"
    return got


SAME = [1], [9] * 8, [128], [127, 1, 129], [0, 5, 0, 300, 64, 0], [517, 69, 69, 513], [257, 1, 1, 1, 1, 600]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lengths", SAME, ids=str)
def test_lengths(lengths, dtype, causal):
    _compare(lengths, lengths, 4, 2, 64, dtype, causal)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [8, 16, 24, 32, 40, 64, 72, 80, 96, 120, 128])
def test_head_sizes(d, dtype, causal):
    lengths = [150, 33, 200]
    _compare(lengths, lengths, 3, 3, d, dtype, causal, pad=5)


CROSS = [([1] * 5, [300, 7, 0, 1, 129]), ([200, 5], [30, 400]), ([0, 130, 64], [50, 1, 700]), ([7], [0]), ([3, 300], [0, 0])]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lq,lk", CROSS, ids=str)
def test_query_and_key_lengths(lq, lk, dtype, causal):
    _compare(lq, lk, 4, 1, 64, dtype, causal, pad=3)


@pytest.mark.parametrize("hq,hk", [(1, 1), (8, 1), (6, 3), (5, 5), (16, 4)])
@pytest.mark.parametrize("d", [64, 128])
def test_grouped_heads(hq, hk, d):
    lengths = [140, 260]
    _compare(lengths, lengths, hq, hk, d, BF16, True)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_two_query_tiles_a_block(dtype):
    """Enough tiles for the forward kernel's pairs, which then differ in the keys they see."""
    lengths = [2500, 10, 1100, 300]
    _compare(lengths, lengths, 12, 12, 64, dtype, True)
    _compare(lengths, lengths, 12, 4, 128, dtype, False)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_sequence(dtype):
    lengths = [8200]
    _compare(lengths, lengths, 1, 1, 64, dtype, True)


@pytest.mark.parametrize("scale", [1.0, 3.0, 0.0, -0.5])
def test_scales(scale):
    """Large scores move the running maximum, a scale that is not positive takes the row kernels."""
    lengths = [300, 40]
    _compare(lengths, lengths, 2, 2, 32, BF16, False, scale=scale)


@pytest.mark.parametrize("grad", [1e-4, 200.0])
def test_half_precision_gradients_of_any_size(grad):
    lengths = [400, 700]
    _compare(lengths, lengths, 2, 2, 64, F16, False, grad=grad)


def test_rising_scores_rescale_the_sums():
    q, k, v, do = _inputs([512], [512], 1, 1, 64, BF16, seed=3)
    k = (k * torch.linspace(0.1, 12, 512, device=DEV)[:, None, None]).to(BF16)
    seq = PackedSequences([512], [512], device=DEV)
    got = _run(q, k, v, do, seq)
    want, bound = _expected(q, k, v, do, [512], [512], False, 64**-0.5, BF16)
    for x, y, b in zip(got, want, bound, strict=True):
        assert ((x.double() - y).abs() <= b).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_behind_the_sequences_give_zeros_and_are_not_read(dtype):
    lengths = [70, 60]
    q, k, v, do = _inputs(lengths, lengths, 2, 2, 64, dtype, pad=200)
    seq = PackedSequences(lengths, device=DEV)
    clean = _run(q, k, v, do, seq)
    for x in (q, k, v, do):
        x[130:] = math.nan
    got = _run(q, k, v, do, seq)
    for x, y in zip(got, clean, strict=True):
        assert torch.equal(x, y) and (x[130:] == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("d", [64, 128])
def test_what_one_sequence_holds_reaches_no_other(which, bad, d):
    lengths = [50, 30, 100, 200]
    q, k, v, do = _inputs(lengths, lengths, 4, 2, d, BF16)
    seq = PackedSequences(lengths, device=DEV)
    clean = _run(q, k, v, do, seq)
    dict(q=q, k=k, v=v, do=do)[which][60, :, 5] = bad  # in the second sequence
    got = _run(q, k, v, do, seq)
    want = packed_attention_cpu(q, k, v, do, lengths)
    others = torch.ones(380, dtype=torch.bool, device=DEV)
    others[50:80] = False
    for x, y, z, (w, b) in zip(got, clean, want[0], zip(*want[1], strict=True), strict=True):
        # the tile's rows are computed again by another kernel where the neighbour reached them: within the bounds
        assert torch.isfinite(x[others]).all()
        assert ((x.double() - w).abs() <= b)[others].all()
        if which == "v" and x is got[0]:  # a value reaches its own column only
            assert torch.equal(torch.isfinite(x[50:80]), torch.isfinite(z[50:80]).to(DEV))


def packed_attention_cpu(q, k, v, do, lengths):
    """(the plain forward pass on the CPU, the clean sequences' expected values and bounds)"""
    from mia_train_b200.ops.packed_attention import packed_attention_reference

    seq = PackedSequences(lengths, device="cpu")
    o = packed_attention_reference(q.cpu().float(), k.cpu().float(), v.cpu().float(), seq, q.shape[2] ** -0.5)
    finite = [x.nan_to_num(0.0, 0.0, 0.0) for x in (q, k, v, do)]
    return [o] * 4, _expected(*finite, lengths, lengths, False, q.shape[2] ** -0.5, q.dtype)


def test_infinite_scores_that_are_masked_leave_the_row_alone():
    lengths = [64, 64]
    q, k, v, do = _inputs(lengths, lengths, 1, 1, 64, BF16)
    k[:64] = torch.finfo(BF16).max
    got = _run(q, k, v, do, PackedSequences(lengths, device=DEV))
    want, bound = _expected(q, k, v, do, lengths, lengths, False, 0.125, BF16)
    for x, y, b in zip(got, want, bound, strict=True):
        assert ((x.double() - y).abs() <= b)[64:].all()


def test_the_same_bits_every_time():
    lengths = [300, 700, 20]
    q, k, v, do = _inputs(lengths, lengths, 8, 2, 64, BF16)
    seq = PackedSequences(lengths, causal=True, device=DEV)
    first = _run(q, k, v, do, seq)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(_run(q, k, v, do, seq), first, strict=True))


def test_strides_that_the_kernel_cannot_take_are_copied():
    lengths = [40, 90]
    q, k, v, do = _inputs(lengths, lengths, 2, 2, 32, BF16)
    seq = PackedSequences(lengths, device=DEV)
    want = _run(q, k, v, do, seq)
    wide = [torch.zeros(130, 2, 65, device=DEV, dtype=BF16) for _ in range(4)]
    views = []
    for w, x in zip(wide, (q, k, v, do), strict=True):
        w[:, :, 1:65:2] = x
        views.append(w[:, :, 1:65:2])
    assert all(torch.equal(x, y) for x, y in zip(_run(*views, seq), want, strict=True))
    one = do[:1, :1].expand(130, 2, 32)  # as the gradient of a sum
    got = _run(q, k, v, one, seq)
    assert all(torch.equal(x, y) for x, y in zip(got, _run(q, k, v, one.contiguous(), seq), strict=True))


def test_other_streams_and_captured_graphs():
    lengths = [200, 300]
    q, k, v, do = _inputs(lengths, lengths, 4, 4, 64, BF16)
    want = _run(q, k, v, do, PackedSequences(lengths, device=DEV))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(_run(q, k, v, do, PackedSequences(lengths, device=DEV)))  # the plan goes at once
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(x, y) for x, y in zip(o, want, strict=True))
    seq = PackedSequences(lengths, device=DEV)
    leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
    side = torch.cuda.Stream()
    graphs = []
    with torch.cuda.stream(side):
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                o = packed_attention(*leaves, seq)
                got = [o.detach(), *torch.autograd.grad(o, leaves, do)]
            del o
            graphs.append((graph, got))
    torch.cuda.synchronize()
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        assert all(torch.equal(x, y) for x, y in zip(got, want, strict=True))


def test_changed_operands_and_second_derivatives_are_refused():
    q, k, v, do = _inputs([30], [30], 1, 1, 32, BF16)
    seq = PackedSequences([30], device=DEV)
    leaf = q.detach().clone().requires_grad_(True)
    x = leaf * 1
    o = packed_attention(x, k, v, seq)
    x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
    o = packed_attention(leaf, k, v, seq)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(o, leaf, do, create_graph=True)


def test_refusals():
    q, k, v, _ = _inputs([30], [30], 2, 2, 32, BF16)
    seq = PackedSequences([30], device=DEV)
    for bad in (
        lambda: packed_attention(q[:, :, :12], k[:, :, :12], v[:, :, :12], seq),
        lambda: packed_attention(q.double(), k.double(), v.double(), seq),
        lambda: packed_attention(*(x.repeat(1, 1, 5) for x in (q, k, v)), seq),
        lambda: packed_attention(q[:20], k, v, seq),
        lambda: packed_attention(q, k[:20], v[:20], seq),
        lambda: packed_attention(q, k.half(), v, seq),
        lambda: packed_attention(q, k, v, PackedSequences([30], device="cpu")),
        lambda: packed_attention(q, k, v, seq, scale=math.nan),
    ):
        with pytest.raises(ValueError):
            bad()


FEW = [([1] * 6, [700, 3, 0, 1500, 513, 512]), ([1, 2, 0, 3], [5000, 900, 40, 2100]), ([5], [9000]), ([1] * 40, [300] * 40)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lq,lk", FEW, ids=str)
def test_few_queries_over_many_keys(lq, lk, dtype, causal):
    assert PackedSequences(lq, lk, causal=causal, device=DEV).items is not None
    _compare(lq, lk, 2, 2, 64, dtype, causal, pad=2)


@pytest.mark.parametrize("hq,hk", [(8, 1), (6, 2), (3, 3)])
@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
def test_few_queries_of_grouped_heads(hq, hk, d):
    _compare([1, 3, 1], [2000, 1800, 4000], hq, hk, d, BF16, True)


def test_few_queries_do_not_see_what_is_masked():
    lq, lk = [2, 2], [1500, 1400]
    q, k, v, do = _inputs(lq, lk, 2, 1, 64, BF16, pad=4)
    seq = PackedSequences(lq, lk, causal=True, device=DEV)
    clean = packed_attention(q, k, v, seq)
    k[1499], v[1499] = math.nan, math.nan  # the first sequence's last key: its last query alone sees it
    k[2900:], v[2900:] = math.inf, math.nan
    got = packed_attention(q, k, v, seq)
    assert got[1].isnan().all() and torch.equal(got[0], clean[0]) and torch.equal(got[2:], clean[2:])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lq,lk", [([3, 2], [0, 0]), ([0, 0], [4, 1]), ([], []), ([0], [0])], ids=str)
def test_tensors_without_rows(lq, lk, dtype):
    q, k, v, do = _inputs(lq, list(lk), 2, 1, 32, dtype)
    for x, like in zip(_run(q, k, v, do, PackedSequences(lq, lk, device=DEV)), (q, q, k, v), strict=True):
        assert x.shape == like.shape and (x == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("scale", [1e-13, 1e-8, 1e-4])
def test_tiny_scales(scale, dtype):
    """The row statistics divided by the scale pass the range of the values that the tensor core subtracts."""
    lengths = [200, 60]
    _compare(lengths, lengths, 2, 1, 64, dtype, False, scale=scale)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("size", [40.0, 400.0])
def test_half_precision_scores_beyond_its_range(size, sign):
    """Every score the same and far from 0: q . k is 1e5 and 1e7, P is uniform and its gradients are not 0."""
    lengths = [150]
    q, k, v, do = _inputs(lengths, lengths, 1, 1, 64, F16)
    q, k = torch.full_like(q, size), torch.full_like(k, sign * size)
    got = _run(q, k, v, do, PackedSequences(lengths, device=DEV))
    want = do.double().mean(0, keepdim=True).expand_as(do)  # dv = P^T do with P = 1 / 150
    # the scores are whole numbers below 2^24 and equal: P is off by the statistics' rounding, 2^-24 of 1.4e6 in units
    # of log2 at most, then by half a step of fp16 in P and dv; 150 products of that
    rel = 2.0**-24 * size * size * 64 * 0.125 * 1.45 * 2
    bound = (rel + 2.0**-10) * do.double().abs().mean(0, keepdim=True) + 2.0**-11 * want.abs() + 2.0**-24
    assert ((got[3].double() - want).abs() <= bound).all()
    assert ((got[0].double() - v.double().mean(0, keepdim=True)).abs() <= (2.0**-10) * v.double().abs().mean(0, keepdim=True) * 2 + 2.0**-10).all()


@pytest.mark.parametrize("last", [1, 200])
def test_offsets_beyond_32_bits(last):
    """Keys whose elements lie past 2^31 in a wide buffer give what they give at its start (tiles and few queries)."""
    wide = torch.zeros(270000, 8192, device=DEV, dtype=BF16)
    torch.manual_seed(0)
    small = torch.randn(last + 300, 8192, device=DEV).to(BF16)
    wide[-(last + 300):] = small
    first = wide.shape[0] - small.shape[0]
    views = [wide[:, 64 * i:64 * (i + 2)].view(-1, 2, 64) for i in (10, 40)]
    q = torch.randn(1 + last, 2, 64, device=DEV).to(BF16)
    do = torch.randn(1 + last, 2, 64, device=DEV).to(BF16)
    got = _run(q, *views, do, PackedSequences([1, last], [first, last + 300], device=DEV))
    near = [small[:, 64 * i:64 * (i + 2)].view(-1, 2, 64) for i in (10, 40)]
    want, bound = _expected(q[1:], *near, do[1:], [last], [last + 300], False, 0.125, BF16)
    for x, y, b in zip((got[0][1:], got[1][1:], got[2][first:], got[3][first:]), want, bound, strict=True):
        assert ((x.double() - y).abs() <= b).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_rows_computed_again_leave_the_other_tile_of_their_block_alone(dtype, causal):
    """Wide heads in enough tiles for two a block: a NaN and an infinity in V make neighbours' rows of one tile be computed
    again while the other tile still goes through its keys. The clean sequences stay within the bounds."""
    # 10 pairs of tiles of 16 heads; sequences end inside of tiles, and the second tile of a pair sees other and more keys
    lengths = [100, 60, 900, 40, 1300, 130]
    q, k, v, do = _inputs(lengths, lengths, 16, 4, 128, dtype)
    want, bound = _expected(q, k, v, do, lengths, lengths, causal, 128**-0.5, dtype)
    clean = torch.ones(sum(lengths), dtype=torch.bool, device=DEV)
    for at, bad in ((1, math.nan), (3, math.inf)):  # whole sequences: causal or not, no clean row sees them
        first = sum(lengths[:at])
        v[first:first + lengths[at], :, 7] = bad
        clean[first:first + lengths[at]] = False
    o = packed_attention(q, k, v, PackedSequences(lengths, causal=causal, device=DEV))
    raise_on_device_errors(DEV)
    err = (o.double() - want[0]).abs()
    assert torch.isfinite(o[clean]).all() and (err <= bound[0])[clean].all()
    assert not torch.isfinite(o[~clean][..., 7]).any()


BLIND = [([256], None, 2, 1, 64), ([130, 300], None, 2, 2, 64), ([130, 300], None, 2, 1, 128), ([900, 1300, 300], None, 16, 16, 128),
         ([1, 2, 3], [600, 700, 40], 2, 1, 64), ([2, 1], [300, 200], 3, 1, 32)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("lq,lk,hq,hk,d", BLIND, ids=str)
def test_a_query_whose_scores_are_all_minus_infinity_gives_nan(lq, lk, hq, hk, d, dtype, causal):
    """0 / 0 in every kernel, in blocks with and without a mask; what does not see the query is not touched."""
    lk = lq if lk is None else lk
    q, k, v, do = _inputs(lq, list(lk), hq, hk, d, dtype)
    k[..., 0] = k[..., 0].abs() + 0.25
    bad = lq[0] - 1  # the first sequence's last query sees all of its keys, causal or not
    want, bound = _expected(q, k, v, do, lq, lk, causal, d**-0.5, dtype)
    q[bad, :, 0] = -math.inf
    got = _run(q, k, v, do, PackedSequences(lq, lk, causal=causal, device=DEV))
    raise_on_device_errors(DEV)
    assert got[0][bad].isnan().all() and got[1][bad].isnan().all()
    assert got[2][:lk[0]].isnan().all() and got[3][:lk[0]].isnan().all()
    rows = torch.arange(sum(lq), device=DEV) != bad
    for x, y, b, keep in zip(got, want, bound, (rows, rows, slice(lk[0], None), slice(lk[0], None)), strict=True):
        assert ((x.double() - y).abs() <= b)[keep].all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lengths,hq,hk,d", [([60, 60], 1, 1, 64), ([130, 1, 40, 300], 4, 2, 64), ([100, 700, 90], 2, 1, 128),
                                             ([0, 520, 3, 0, 257], 3, 3, 32)], ids=str)
def test_gradients_do_not_depend_on_other_sequences_gradients(lengths, hq, hk, d, dtype, causal):
    """The first non-empty sequence's incoming gradients are 2^-9, the others' 2^4 (fp16 has 2^-24 to 2^15): its own results
    are within the bounds of its own size, and the same bits whatever the others' are."""
    q, k, v, do = _inputs(lengths, lengths, hq, hk, d, dtype)
    seq = PackedSequences(lengths, causal=causal, device=DEV)
    own = slice(0, next(n for n in lengths if n))
    do[own] *= 2.0**-9
    first = _run(q, k, v, do, seq)
    do[own.stop:] *= 16
    got = _run(q, k, v, do, seq)
    raise_on_device_errors(DEV)
    want, bound = _expected(*(x[own] for x in (q, k, v, do)), [own.stop], [own.stop], causal, d**-0.5, dtype)
    for x, y, z, b in zip(got, first, want, bound, strict=True):
        assert torch.equal(x[own], y[own])
        assert ((x[own].double() - z).abs() <= b).all()


@pytest.mark.parametrize("hq,hk", [(1, 1), (4, 1)])
def test_half_precision_gradients_of_late_queries(hq, hk):
    """Causal, do falls from 2^4 at the first queries to 2^-10 at the last: keys that only small gradients reach keep them."""
    n = 600
    q, k, v, do = _inputs([n], [n], hq, hk, 64, F16)
    do *= torch.exp2(torch.linspace(4, -10, n, device=DEV))[:, None, None].half()
    seq = PackedSequences([n], causal=True, device=DEV)
    got = _run(q, k, v, do, seq)
    # with gradients of the last 200 queries alone, the bounds of whose size hold for the last 200 keys
    late = do.clone()
    late[:400] = 0
    want, bound = _expected(q, k, v, late, [n], [n], True, 0.125, F16)
    for x, y, b in zip(got[1:], want[1:], bound[1:], strict=True):
        assert ((x.double() - y).abs() <= b)[400:].all()
