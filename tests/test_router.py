"""The general router (ops.route_topk) and its gradient against oracle/router.py.

Tolerances: with u = 2^-24 a score takes at most 5 roundings (exponential, add, divide), the sum over k picks k more, the
division and the product with the scale two: (2 * 5 + k + 4) u relative.  A gradient multiplies a slope (two scores), the
scale and twice 1 / P (5 + k each), and subtracts a sum of k products: (6 * 5 + 4 k + 16) u of the magnitudes that the
formula adds, and 5 more per expert-wide sum of a softmax; then the rounding to the logits' type."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import router as oracle

U = 2.0**-24
HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0**-25}

# E, groups, kept, group_top, top_k
SHAPES = [(256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (64, 1, 1, 2, 6), (60, 1, 1, 2, 4), (96, 4, 2, 2, 5), (1, 1, 1, 2, 1),
          (128, 64, 9, 2, 16), (384, 1, 1, 2, 8), (1024, 32, 4, 2, 64), (7, 7, 3, 2, 3), (512, 16, 16, 1, 1),
          (256, 1, 1, 2, 8), (40, 5, 2, 2, 8), (65, 1, 1, 1, 2), (1000, 8, 5, 2, 12), (256, 32, 8, 2, 8)]


def _floor(renormalize, least=2.0**-150):
    """What a weight may be off where fp32 scores run out: a score below 2^-126 by half of the last step, 2^-150.  The
    forward's sigmoid, 1 / (1 + e) with e = exp(-x) in fp32, is 0 from e >= 2^128 on, where it is at most 2^-128: `least`
    for it.  A renormalised weight divides that by a sum of at least 1e-20."""
    return least * 1e20 if renormalize else 2.0**-126


def _logits(T, E, seed, dtype, kind):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, E, generator=g) * 2
    if kind == "masked":
        x[:, torch.rand(E, generator=g) < 0.2] = -torch.inf
        x[torch.rand(T, generator=g) < 0.3] = -torch.inf
        x[torch.rand(T, E, generator=g) < 0.05] = torch.nan
        x[torch.rand(T, E, generator=g) < 0.01] = torch.inf
    elif kind == "ties":
        x = torch.randint(-2, 3, (T, E), generator=g).float()
    elif kind == "far":
        x = x * 40
    return x.to(dtype)


def _bias(E, seed, kind):
    if kind == "none":
        return None
    g = torch.Generator().manual_seed(seed)
    b = torch.randn(E, generator=g) * 0.1
    if kind == "closed":
        b[::3] = -torch.inf
        b[1:2] = torch.nan
    return b


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_matches_the_layers_router():
    from oracle import routing

    x = _logits(64, 256, 3, torch.float32, "plain").numpy()
    b = _bias(256, 4, "plain").numpy()
    w, ids = oracle.route(x, b, 8, "sigmoid", 8, 4, 2, True, 2.5)
    ref = routing.route(x, b, 2.5)
    assert np.array_equal(ids, ref["ids"])
    assert np.abs(w - ref["weights"]).max() < 2.5 * 30 * U


@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_oracle_gradient_against_differences(scoring, renormalize):
    x = _logits(5, 12, 7, torch.float32, "plain").numpy().astype(np.float64)
    x[2, 3:6] = -np.inf
    _, ids = oracle.route(x, None, 3, scoring, renormalize=renormalize)
    ids[4] = -1
    g = np.random.default_rng(1).standard_normal(ids.shape)
    d, _ = oracle.route_backward(g, x, ids, scoring, renormalize, 1.7)
    for e in range(12):
        step = np.zeros_like(x)
        step[:, e] = 1e-5
        f = [(oracle.weights_of(x + s * step, ids, scoring, renormalize, 1.7) * g).sum(1) for s in (1, -1)]
        assert np.abs((f[0] - f[1]) / 2e-5 - d[:, e]).max() < 1e-8


def test_oracle_all_masked_rows_and_few_open_experts():
    x = np.full((2, 8), -np.inf, np.float32)
    x[1, 5] = 1.0
    for scoring in ("sigmoid", "softmax"):
        w, ids = oracle.route(x, None, 3, scoring, 4, 2)
        assert ids.tolist() == [[-1, -1, -1], [5, -1, -1]]
        assert np.allclose(w, [[0, 0, 0], [1, 0, 0]])


FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: validation fails first


def _topk(lib, logits=FAKE, dtype=0, stride=256, bias=None, T=4, E=256, k=8, scoring=0, groups=8, kept=4, top=2,
          weights=FAKE, ids=FAKE):
    return lib.moe_route_topk(logits, dtype, stride, bias, T, E, k, scoring, groups, kept, top, 1, 1.0, weights, ids,
                              None)


@pytest.mark.parametrize("kw,what", [
    (dict(T=-1), "T must be"), (dict(T=(1 << 24) + 1), "T must be"), (dict(E=0), "n_experts"),
    (dict(E=1025), "n_experts"), (dict(k=0), "top_k"), (dict(k=65), "top_k"), (dict(E=4, groups=1, kept=1, k=5), "top_k"),
    (dict(scoring=2), "scoring"), (dict(dtype=3), "dtype"), (dict(groups=7), "n_group"), (dict(groups=0), "n_group"),
    (dict(groups=128), "n_group"), (dict(kept=9), "topk_group"), (dict(kept=0), "topk_group"), (dict(top=3), "group_top"),
    (dict(groups=64, kept=1), "kept groups"), (dict(logits=None), "logits"), (dict(weights=None), "weights"),
    (dict(ids=None), "ids"), (dict(logits=ctypes.c_void_p(0x10002)), "aligned"),
])
def test_route_topk_refusals(lib, capi, kw, what):
    assert _topk(lib, **kw) == capi.MOE_ERR_INVALID_ARG
    assert what in lib.moe_last_error().decode()


def test_route_topk_T0_is_noop(lib, capi):
    assert _topk(lib, T=0, logits=None) == capi.MOE_OK
    assert lib.moe_route_topk_backward(None, None, 0, 256, None, 0, 256, 8, 0, 1, 1.0, None, None) == capi.MOE_OK


def test_route_topk_backward_refusals(lib, capi):
    def call(grad=FAKE, logits=FAKE, ids=FAKE, out=FAKE, T=4, E=256, k=8):
        return lib.moe_route_topk_backward(grad, logits, 0, 256, ids, T, E, k, 0, 1, 1.0, out, None)

    for kw in (dict(grad=None), dict(logits=None), dict(ids=None), dict(out=None), dict(T=-1), dict(E=2000), dict(k=0),
               dict(out=ctypes.c_void_p(0x10008))):
        assert call(**kw) == capi.MOE_ERR_INVALID_ARG, kw


def test_route_topk_has_no_cpu_path(ops):
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.route_topk(torch.zeros(2, 8), None, 2)


# ------------------------------------------------------------------------------------------------ GPU
def _check(ops, x, bias, k, scoring, groups, kept, top, renormalize, scale, dev):
    w, ids = ops.route_topk(x, None if bias is None else bias.to(dev), k, scoring, groups, kept, top, renormalize, scale)
    want_w, want_ids = oracle.route(x.float().cpu().numpy(), None if bias is None else bias.numpy(), k, scoring, groups,
                                    kept, top, renormalize, scale)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    err = np.abs(w.cpu().numpy() - want_w)
    least = 2.0**-128 if scoring == "sigmoid" else 2.0**-150
    assert (err <= (2 * 5 + k + 4) * U * np.abs(want_w) + scale * _floor(renormalize, least) * (k + 1)).all(), err.max()
    return w, ids


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties", "far"])
def test_route_topk(ops, cuda, shape, scoring, kind):
    E, groups, kept, top, k = shape
    for i, (T, dtype) in enumerate([(1, torch.float32), (67, torch.bfloat16), (130, torch.float16), (33, torch.float32)]):
        x = _logits(T, E, 11 * E + i, dtype, kind).to(cuda)
        for bias in ("none", "plain", "closed"):
            _check(ops, x, _bias(E, E + i, bias), k, scoring, groups, kept, top, bool(i & 1), (1.0, 2.5)[i & 1], cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] <= 256 and s[4] <= 8], ids=str)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kind", ["plain", "masked", "ties", "far", "near"])
def test_route_topk_many_tokens(ops, cuda, shape, scoring, kind):
    """From 4096 tokens on a wave takes four; `near`: rows whose best logits are a few units of the last place apart, and
    equal ones, around every place of the border."""
    E, groups, kept, top, k = shape
    T = 4099
    for i, (dtype, biases) in enumerate([(torch.float32, ("none", "plain")), (torch.bfloat16, ("none", "closed")),
                                         (torch.float16, ("plain",))]):
        x = _logits(T, E, 17 * E + i, torch.float32, "plain" if kind == "near" else kind)
        if kind == "near":
            g = torch.Generator().manual_seed(E + i)
            x = x.abs().neg()
            x += 3.0 * (torch.rand(T, E, generator=g) < 1.5 * k / E)
            close = torch.rand(T, E, generator=g) < 2.0 * k / E
            x = torch.where(close, 1.5 + torch.randint(0, 3, (T, 1), generator=g) * 0.7, x)
            x = torch.where(close, x * (1 + torch.randint(-3, 4, (T, E), generator=g) * 2.0**-23), x)
        x = x.to(dtype).to(cuda)
        for bias in biases:
            b = _bias(E, E + i, bias)
            if kind == "near" and b is not None:
                b = (b * 4).round() / 4
            _check(ops, x, b, k, scoring, groups, kept, top, bool(i & 1), (1.0, 2.5)[i & 1], cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [4095, 4096, 4097])
def test_route_topk_many_tokens_large_bias(ops, cuda, T):
    """Biases that dwarf the scores, of both signs: groups' sums cancel, and v keeps few of the score's digits."""
    x = _logits(T, 256, T, torch.float32, "plain").to(cuda)
    for scale in (30.0, 1e4, 1e30):
        b = _bias(256, 3, "plain") * scale
        b[7], b[40] = torch.inf, 3e38
        _check(ops, x, b, 8, "sigmoid", 8, 4, 2, True, 1.0, cuda)
        _check(ops, x, b, 6, "softmax", 1, 1, 2, False, 1.0, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1000, 6000])
def test_route_topk_equals_the_layers_router(ops, cuda, T):
    x = _logits(T, 256, 21, torch.float32, "plain").to(cuda)
    bias = _bias(256, 22, "plain").to(cuda)
    w, ids = ops.route_topk(x, bias, 8, "sigmoid", 8, 4, scale=2.5)
    ref = ops.route(x, bias, 2.5, 0)
    assert torch.equal(ids, ref["topk_ids"]) and torch.equal(w, ref["topk_w"])


@pytest.mark.gpu
def test_route_topk_strided_and_odd_rows(ops, cuda):
    many = _logits(4100, 131, 32, torch.float32, "plain").to(cuda)
    for x in (many[:, :128], many[:, 3:131], many[:, 2:66], many[:1].expand(4100, 131)[:, :64]):
        _check(ops, x, None, 4, "sigmoid", 4, 2, 2, True, 1.0, cuda)
    wide = _logits(50, 301, 31, torch.bfloat16, "plain").to(cuda)
    for x in (wide[:, 7:167], wide[::3, 1:65], wide[:1].expand(9, 301)[:, :96], wide[10:10, :64]):
        assert x.size(0) < 2 or not x.is_contiguous()
        _check(ops, x, None, 4, "softmax", 1, 1, 2, True, 1.0, cuda)
    with pytest.raises(RuntimeError, match="contiguous along"):
        ops.route_topk(wide.t(), None, 4)


@pytest.mark.gpu
def test_route_topk_python_refusals(ops, cuda):
    x = torch.zeros(4, 64, device=cuda)
    for bad, what in ((dict(top_k=0), "top_k"), (dict(top_k=65), "top_k"), (dict(scoring="tanh"), "scoring"),
                      (dict(bias=torch.zeros(63, device=cuda)), "bias"), (dict(bias=torch.zeros(64)), "bias"),
                      (dict(bias=torch.zeros(64, device=cuda, dtype=torch.bfloat16)), "bias"),
                      (dict(n_group=5), "n_group"), (dict(n_group=8, topk_group=9), "topk_group"),
                      (dict(logits=x.double()), "float32"), (dict(logits=x[0]), "two-dimensional"),
                      (dict(logits=torch.zeros(2, 1025, device=cuda)), "experts")):
        kw = {"logits": x, "bias": None, "top_k": 4, **bad}
        with pytest.raises(RuntimeError, match=what):
            ops.route_topk(**kw)
    with pytest.raises(RuntimeError, match="ids"):
        ops.route_topk_backward(torch.zeros(4, 4, device=cuda), x, torch.zeros(4, 4, device=cuda))
    with pytest.raises(RuntimeError, match="grad_weights"):
        ops.route_topk_backward(torch.zeros(4, 3, device=cuda), x, torch.zeros(4, 4, device=cuda, dtype=torch.int32))


def _check_grad(got, g, x, ids, scoring, renormalize, scale):
    want, mag = oracle.route_backward(g.cpu().numpy(), x.float().cpu().numpy(), ids.cpu().numpy(), scoring, renormalize,
                                      scale)
    k, E, dtype = ids.shape[1], x.shape[1], got.dtype
    ops_ = 6 * 5 + 4 * k + 16 + (2 * E + 5 if scoring == "softmax" else 0)
    bound = ops_ * U * mag
    bound += HALF[dtype] * (np.abs(want) + bound) + TINY[dtype] + 10 * scale * np.abs(g.cpu().numpy()).max(initial=0) * _floor(renormalize)
    err = np.abs(got.float().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_topk_backward(ops, cuda, shape, scoring, renormalize):
    E, groups, kept, top, k = shape
    for i, (T, dtype, kind) in enumerate([(1, torch.float32, "plain"), (66, torch.bfloat16, "plain"),
                                          (131, torch.float16, "ties"), (35, torch.float32, "far")]):
        x = _logits(T, E, 13 * E + i, dtype, kind)
        x[:, 2::7] = -torch.inf
        x[3::11] = -torch.inf
        x = x.to(cuda)
        w, ids = ops.route_topk(x, None, k, scoring, groups, kept, top, renormalize, 2.5)
        g = torch.randn(T, k, generator=torch.Generator().manual_seed(i)).to(cuda)
        _check_grad(ops.route_topk_backward(g, x, ids, scoring, renormalize, 2.5), g, x, ids, scoring, renormalize, 2.5)


@pytest.mark.gpu
def test_route_topk_backward_repeated_and_outside_picks(ops, cuda):
    x = _logits(6, 32, 41, torch.float32, "plain").to(cuda)
    ids = torch.tensor([[3, 3, 9, -1], [0, 31, 32, 100], [-1, -1, -1, -1], [5, 5, 5, 5], [1, 2, 3, 4], [31, 0, -7, 2]],
                       dtype=torch.int32, device=cuda)
    g = torch.randn(6, 4, generator=torch.Generator().manual_seed(2)).to(cuda)
    for scoring in ("sigmoid", "softmax"):
        for renormalize in (True, False):
            _check_grad(ops.route_topk_backward(g, x, ids, scoring, renormalize, 1.5), g, x, ids, scoring, renormalize, 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route_topk_autograd(ops, cuda, dtype, scoring):
    base = _logits(40, 200, 51, dtype, "plain").to(cuda).requires_grad_()
    x = base[:, 8:168]  # strided, and part of a larger tensor
    bias = _bias(160, 5, "plain").to(cuda).requires_grad_()
    w, ids = ops.route_topk(x, bias, 6, scoring, 8, 3, scale=2.0)
    assert w.requires_grad and not ids.requires_grad
    g = torch.randn(40, 6, generator=torch.Generator().manual_seed(3)).to(cuda)
    w.backward(g)
    assert bias.grad is None
    assert base.grad[:, :8].count_nonzero() == 0 and base.grad[:, 168:].count_nonzero() == 0
    _check_grad(base.grad[:, 8:168], g, x.detach(), ids, scoring, True, 2.0)
    base.grad = None
    ops.route_topk(x, bias, 6, scoring, 8, 3, scale=2.0)[0].sum(1, keepdim=True).expand(40, 4).sum().backward()
    assert base.grad is not None  # a gradient that is not contiguous
    with torch.no_grad():
        assert not ops.route_topk(x, bias, 6, scoring, 8, 3)[0].requires_grad


@pytest.mark.gpu
def test_route_topk_empty_batch_autograd(ops, cuda):
    x = torch.zeros(0, 64, device=cuda, requires_grad=True)
    w, ids = ops.route_topk(x, None, 4)
    assert w.shape == (0, 4) and ids.shape == (0, 4)
    w.sum().backward()
    assert x.grad.shape == (0, 64)


@pytest.mark.gpu
def test_route_topk_streams_and_graph(ops, cuda):
    x = _logits(513, 256, 61, torch.float32, "plain").to(cuda)
    bias = _bias(256, 62, "plain").to(cuda)
    g = torch.randn(513, 8, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1, ids1 = ops.route_topk(x, bias, 8, "sigmoid", 8, 4)
    torch.cuda.current_stream().wait_stream(side)
    w0, ids0 = ops.route_topk(x, bias, 8, "sigmoid", 8, 4)
    assert torch.equal(w0, w1) and torch.equal(ids0, ids1)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        w, ids = ops.route_topk(x, bias, 8, "sigmoid", 8, 4)
        d = ops.route_topk_backward(g, x, ids)
    for i in range(3):
        x.copy_(_logits(513, 256, 70 + i, torch.float32, "plain"))
        w.fill_(float("nan"))
        d.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        we, idse = ops.route_topk(x, bias, 8, "sigmoid", 8, 4)
        assert torch.equal(w, we) and torch.equal(ids, idse)
        assert torch.equal(d, ops.route_topk_backward(g, x, idse))


@pytest.mark.gpu
@pytest.mark.parametrize("E,k,dtype", [(60, 4, torch.bfloat16), (64, 16, torch.float16), (100, 8, torch.float32),
                                       (129, 16, torch.bfloat16), (256, 8, torch.float32), (64, 17, torch.float32)])
def test_route_topk_backward_many_tokens(ops, cuda, E, k, dtype):
    """Either side of the size from which a token takes 16 lanes, with repeated and empty picks, rows apart."""
    for T in (32 * E - 1, 32 * E, 32 * E + 3):
        rng = np.random.default_rng(T + k)
        x = torch.from_numpy(rng.standard_normal((T, E + 4)).astype(np.float32)).to(cuda, dtype)[:, :E]
        ids = torch.from_numpy(rng.integers(-1, E + 1, size=(T, k)).astype(np.int32)).to(cuda)
        ids[::3] = ids[::3, :1]
        g = torch.from_numpy(rng.standard_normal((T, k)).astype(np.float32)).to(cuda)
        rows = torch.cat([torch.arange(40), torch.arange(T - 40, T)]).to(cuda)
        for renormalize in (False, True):
            got = ops.route_topk_backward(g, x, ids, "softmax", renormalize, 2.5)
            one = ops.route_topk_backward(g[rows], x[rows], ids[rows], "softmax", renormalize, 2.5)
            _check_grad(got[rows], g[rows], x[rows], ids[rows], "softmax", renormalize, 2.5)
            _check_grad(one, g[rows], x[rows], ids[rows], "softmax", renormalize, 2.5)
            assert torch.equal(got, ops.route_topk_backward(g, x, ids, "softmax", renormalize, 2.5))


@pytest.mark.gpu
def test_route_topk_far_rows(ops, cuda):
    """The largest batch: elements past 2^31, and past 2^32 bytes."""
    T, E = 1 << 24, 256
    x = torch.empty(T, E, dtype=torch.bfloat16, device=cuda)
    x[: 1 << 20] = torch.randn(1 << 20, E, device=cuda).to(torch.bfloat16)
    for i in range(1, 16):
        x[i << 20 : (i + 1) << 20] = x[: 1 << 20].roll(i, 0)
    w, ids = ops.route_topk(x, None, 8, "softmax", 8, 4)
    g = torch.randn(1 << 20, 8, device=cuda).repeat(16, 1)
    dx = ops.route_topk_backward(g, x, ids, "softmax")
    for lo in (0, T // 2 - 4500, T - 9000):
        rows = slice(lo, lo + 9000)  # 8192 and more: the same layout, and order of sums, as the whole batch
        want = ops.route_topk(x[rows], None, 8, "softmax", 8, 4)
        assert torch.equal(w[rows], want[0]) and torch.equal(ids[rows], want[1])
        assert torch.equal(dx[rows], ops.route_topk_backward(g[rows], x[rows], ids[rows], "softmax"))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_route_topk_captured_training_step(ops, cuda, scoring):
    """Forward and backward in a graph, replayed over new logits with eager work between."""
    x = _logits(300, 160, 61, torch.float32, "plain").to(cuda).requires_grad_()
    g = torch.randn(300, 6, generator=torch.Generator().manual_seed(8)).to(cuda)

    def step():
        w, ids = ops.route_topk(x, None, 6, scoring, 8, 3)
        return w.detach(), ids, torch.autograd.grad(w, x, g)[0]  # nothing of the autograd graph stays

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            x.copy_(_logits(300, 160, 70 + seed, torch.float32, "plain"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_route_topk_refuses_numbers_past_32_bits(ops, cuda):
    x = torch.zeros(2, 64, device=cuda)
    for kw in ({"n_group": (1 << 32) + 1}, {"n_group": 8, "topk_group": (1 << 32) + 2}, {"n_group": 8, "group_top": (1 << 32) + 1},
               {"topk_group": -1}):
        with pytest.raises(RuntimeError, match="n_group"):
            ops.route_topk(x, None, 2, **kw)
    with pytest.raises(RuntimeError, match="T must be"):
        ops.route_topk(x[:1].expand((1 << 32) + 2, 64), None, 2)
