"""4-bit weights and FP8 activations (ops.quant_act, quantize_w4, pack_w4, linear_w4, experts_w4) against oracle/w4.py,
which derives the bounds beside its formulas."""

from __future__ import annotations

import ctypes
import importlib

import numpy as np
import pytest
import torch

from oracle import router as orouter
from oracle import w4 as oracle
from oracle.numerics import e4m3_encode


F8 = torch.float8_e4m3fn


def _codes(rng, *shape):
    return rng.integers(0, 256, size=shape, dtype=np.uint8)


def _matrix(rng, N, K, spread=6):
    """Random codes with scales around the size of a trained layer's."""
    return _codes(rng, N, K // 2), rng.integers(118 - spread, 119, size=(N, K // 32), dtype=np.uint8)


def _act(rng, T, K):
    x = rng.standard_normal((T, K)).astype(np.float32) * np.where(rng.random(K) < 0.01, 20.0, 1.0).astype(np.float32)
    return oracle.quant_act(x)


def _dev(a, dev, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    return t if dtype is None else t.view(dtype)


# ------------------------------------------------------------------------------------------------ CPU
def test_oracle_quantize_is_the_nearest_element():
    rng = np.random.default_rng(1)
    w = rng.standard_normal((4, 128)).astype(np.float32)
    codes, scales = oracle.quantize(w)
    v = oracle.decode(codes, scales)
    step = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, axis=1)
    a = np.abs(w) / step
    # below 4 the elements are at most 1 apart; above, 4 and 6, and what exceeds 6 saturates
    assert (np.abs(v - w) <= np.where(a < 2, 0.25, np.where(a < 4, 0.5, np.maximum(1.0, a - 6))) * step + 1e-12).all()
    amax = np.abs(w).reshape(4, 4, 32).max(2) / np.ldexp(1.0, scales.astype(int) - 127)
    assert (amax >= 4).all() and (amax < 8).all()


def test_oracle_pack_layout():
    rng = np.random.default_rng(2)
    codes, scales = _matrix(rng, 37, 640)
    p = oracle.pack(codes, scales)
    assert p.shape == (3, 2, 4352)
    for row, kb, g in ((0, 0, 0), (17, 3, 2), (36, 4, 3), (20, 1, 1)):
        at = p[row // 16, kb // 4]
        lane, b = 16 * g + row % 16, kb % 4
        assert np.array_equal(at[b * 1024 + lane * 16:][:16], codes[row, kb * 64 + g * 16:][:16])
        assert at[4096 + lane * 4 + b] == scales[row, kb * 4 + g]
    assert (p[2, 0, 16 * 6:16 * 16] == 0).all() and p[2, 1, 4096 + 4 * 9 + 1] == 127  # padding rows and K-blocks


def test_oracle_experts_is_the_sum_over_picks():
    rng = np.random.default_rng(3)
    xc, xs = _act(rng, 3, 128)
    w13 = rng.standard_normal((2, 256, 128)) * 0.1
    w2 = rng.standard_normal((2, 128, 128)) * 0.1
    ids = np.array([[0, 1], [1, 1], [-1, 5]], np.int32)
    w = np.ones((3, 2), np.float32)
    out, err = oracle.experts(xc, xs, w13, w2, ids, w, 0)
    x = oracle.act_values(xc, xs)
    g = x[1] @ w13[1].T
    c = g[:128] * g[128:] / (1 + np.exp(-g[128:]))
    cc, cs = oracle.quant_act(c[None].astype(np.float32))
    assert np.allclose(out[1], 2 * (oracle.act_values(cc, cs)[0] @ w2[1].T), rtol=1e-6)
    assert (out[2] == 0).all() and (err[2] == 0).all()


FAKE = ctypes.c_void_p(0x10000)
ODD = ctypes.c_void_p(0x10008)


def _refused(lib, capi, rc, what, code=None):
    assert rc == (capi.MOE_ERR_INVALID_ARG if code is None else code)
    assert what in lib.moe_last_error().decode()


def test_w4_sizes(lib):
    assert lib.moe_packed_w4_bytes(4096, 7168) == 256 * 14 * 4352
    assert lib.moe_packed_w4_bytes(1, 128) == 4352
    for N, K in ((0, 128), (1, 0), (1, 130), (-1, 128), (1, 262144 + 128)):
        assert lib.moe_packed_w4_bytes(N, K) == 0
    assert lib.moe_experts_w4_workspace_bytes(0, 128, 128, 1, 1) >= 0
    small, large = (lib.moe_experts_w4_workspace_bytes(T, 7168, 2048, 32, 8) for T in (1, 64))
    assert 0 < small < large
    for bad in ((1, 100, 128, 1, 1), (1, 128, 100, 1, 1), (1, 128, 128, 0, 1), (1, 128, 128, 1025, 1),
                (1, 128, 128, 1, 0), (1, 128, 128, 1, 65), (-1, 128, 128, 1, 1), (262144, 128, 128, 1, 1)):
        assert lib.moe_experts_w4_workspace_bytes(*bad) == 0


def test_w4_refusals(lib, capi):
    f = FAKE
    _refused(lib, capi, lib.moe_quant_act(f, 3, 128, 1, 128, f, f, None), "dtype")
    _refused(lib, capi, lib.moe_quant_act(f, 1, 128, 1, 64, f, f, None), "K must be")
    _refused(lib, capi, lib.moe_quant_act(f, 1, 132, 2, 128, f, f, None), "16 bytes apart")
    _refused(lib, capi, lib.moe_quant_act(f, 1, 128, -1, 128, f, f, None), "T must be")
    _refused(lib, capi, lib.moe_quant_act(ODD, 1, 128, 1, 128, f, f, None), "aligned")
    _refused(lib, capi, lib.moe_quantize_w4(None, 1, 4, f, f, None), "null")
    _refused(lib, capi, lib.moe_quantize_w4(f, 1, (1 << 29) + 1, f, f, None), "groups")
    _refused(lib, capi, lib.moe_pack_w4(f, f, f, -1, 16, 128, None), "n must be")
    _refused(lib, capi, lib.moe_pack_w4(f, f, f, 1, 0, 128, None), "N must be")
    _refused(lib, capi, lib.moe_pack_w4(f, f, f, 1, 16, 100, None), "K must be")
    _refused(lib, capi, lib.moe_pack_w4(f, f, f, 1 << 20, 4096, 7168, None), "2^36")
    _refused(lib, capi, lib.moe_unpack_w4(f, None, f, 1, 16, 128, None), "null")
    _refused(lib, capi, lib.moe_linear_w4(f, f, f, 262144, 16, 128, f, None), "T must be")
    _refused(lib, capi, lib.moe_linear_w4(f, f, f, 1, 0, 128, f, None), "N must be")
    _refused(lib, capi, lib.moe_linear_w4(f, f, ODD, 1, 16, 128, f, None), "aligned")

    def experts(x=f, ids=f, ws=f, ws_bytes=1 << 40, T=4, H=256, I=128, E=4, k=2, off=0):
        return lib.moe_experts_w4(x, f, f, f, ids, f, T, H, I, E, k, off, ws, ws_bytes, f, None)

    for kw, what in ((dict(x=None), "x must"), (dict(ids=ctypes.c_void_p(0x10002)), "ids"), (dict(T=-1), "T must"),
                     (dict(H=200), "hidden"), (dict(I=0), "inter"), (dict(E=0), "e_local"), (dict(k=65), "top_k"),
                     (dict(off=-1), "local_expert_offset"), (dict(off=(1 << 30) + 1), "local_expert_offset"),
                     (dict(ws=None), "workspace")):
        _refused(lib, capi, experts(**kw), what)
    _refused(lib, capi, experts(ws_bytes=64), "workspace", capi.MOE_ERR_WORKSPACE)


def test_w4_empty_calls(lib, capi):
    assert lib.moe_quant_act(None, 1, 128, 0, 128, None, None, None) == capi.MOE_OK
    assert lib.moe_quantize_w4(None, 1, 0, None, None, None) == capi.MOE_OK
    assert lib.moe_pack_w4(None, None, None, 0, 16, 128, None) == capi.MOE_OK
    assert lib.moe_linear_w4(None, None, None, 0, 16, 128, None, None) == capi.MOE_OK
    assert lib.moe_experts_w4(None, None, None, None, None, None, 0, 128, 128, 1, 1, 0, None, 0, None, None) == capi.MOE_OK


def test_w4_has_no_cpu_path(ops):
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.quant_act(torch.zeros(1, 128))
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.quantize_w4(torch.zeros(16, 128))
    with pytest.raises(RuntimeError, match="HIP device"):
        ops.pack_w4(torch.zeros(16, 64, dtype=torch.uint8), torch.zeros(16, 4, dtype=torch.uint8))


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("T,K", [(1, 128), (3, 640), (17, 7168), (130, 2048), (1000, 384)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quant_act(ops, cuda, T, K, dtype):
    g = torch.Generator().manual_seed(T + K)
    x = (torch.randn(T, K, generator=g) * torch.rand(K, generator=g) * 30).to(dtype)
    x[T // 2, :128] = 0
    wide = torch.zeros(T, K + 64, dtype=dtype)
    wide[:, 8:8 + K] = x
    for y in (x.to(cuda), wide.to(cuda)[:, 8:8 + K]):
        codes, scale = ops.quant_act(y)
        want, want_s = oracle.quant_act(x.float().numpy())
        assert codes.dtype == F8 and np.array_equal(scale.cpu().numpy(), want_s)
        assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), want)


@pytest.mark.gpu
def test_quant_act_equals_the_producer(ops, cuda):
    x = torch.randn(65, 7168, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    packed = ops.pack_router(torch.zeros(256, 7168, dtype=torch.bfloat16, device=cuda))
    _, hq, hs = ops.router_quant(x, packed)
    codes, scale = ops.quant_act(x)
    assert torch.equal(codes.view(torch.uint8), hq.view(torch.uint8)) and torch.equal(scale, hs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quant_act_infinities_and_nan(ops, cuda, dtype):
    x = torch.randn(4, 256, generator=torch.Generator().manual_seed(2)).to(dtype)
    x[0, 5], x[1, 7], x[2, 200] = torch.inf, torch.nan, -torch.inf
    codes, scale = (t.cpu() for t in ops.quant_act(x.to(cuda)))
    c = codes.float()
    assert torch.isinf(scale[0, 0]) and torch.isinf(scale[1, 2]) and torch.isfinite(scale[:, [1, 3]]).all()
    assert torch.isnan(c[1, 7]) and torch.isfinite(c[1, :7]).all()  # a NaN stays one and leaves its block's scale
    assert torch.isfinite(c[3]).all() and torch.isfinite(c[0, 128:]).all()


@pytest.mark.gpu
def test_quant_act_refusals(ops, cuda):
    for bad, what in ((torch.zeros(2, 130), "multiple of 128"), (torch.zeros(2, 0), "multiple of 128"),
                      (torch.zeros(2, 128, dtype=torch.float64), "float32"), (torch.zeros(128), "two-dimensional")):
        with pytest.raises(RuntimeError, match=what):
            ops.quant_act(bad.to(cuda))
    wide = torch.zeros(4, 260, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(RuntimeError, match="aligned"):
        ops.quant_act(wide[:, :256])
    with pytest.raises(RuntimeError, match="contiguous along"):
        ops.quant_act(torch.zeros(128, 128, device=cuda).t())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_w4(ops, cuda, dtype):
    g = torch.Generator().manual_seed(4)
    w = torch.randn(9, 256, generator=g) * torch.exp2(torch.randint(-20, 12, (9, 1), generator=g).float())
    w[0, :32] = 0
    w[1, :64] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -2.5, 6.0, 7.9, 4.0, 0.5, 0.0, -5.0, 6.5]).repeat(4)
    w = w.to(dtype)
    if dtype == torch.float32:
        w[2, :32] *= 2.0**-126  # below the smallest scale
        w[3, 0] = 3e38
    codes, scales = ops.quantize_w4(w.to(cuda))
    want, want_s = oracle.quantize(w.float().numpy())
    assert np.array_equal(scales.cpu().numpy(), want_s)
    assert np.array_equal(codes.cpu().numpy(), want)
    w[5, 40], w[6, 3] = torch.nan, -torch.inf
    codes, scales = ops.quantize_w4(w.to(cuda))
    bad = scales.cpu() == 255
    assert bad[5, 1] and bad[6, 0] and bad.sum() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(16, 128), (37, 640), (1, 512), (4096, 7168), (130, 2048)])
def test_pack_w4(ops, cuda, N, K):
    rng = np.random.default_rng(N + K)
    codes, scales = _codes(rng, N, K // 2), _codes(rng, N, K // 32)
    p = ops.pack_w4(_dev(codes, cuda), _dev(scales, cuda))
    assert np.array_equal(p.cpu().numpy(), oracle.pack(codes, scales))
    back = ops.unpack_w4(p, N, K)
    assert np.array_equal(back[0].cpu().numpy(), codes) and np.array_equal(back[1].cpu().numpy(), scales)
    if N * K < 1 << 20:
        three = ops.pack_w4(_dev(np.stack([codes] * 3), cuda), _dev(np.stack([scales] * 3), cuda))
        assert three.shape == (3, *p.shape) and all(torch.equal(q, p) for q in three)
        out = torch.zeros_like(three)
        ops.pack_w4(_dev(codes[None], cuda), _dev(scales[None], cuda), out=out[1:2])
        assert torch.equal(out[1], p) and out[0].count_nonzero() == 0 and out[2].count_nonzero() == 0


@pytest.mark.gpu
def test_pack_w4_refusals(ops, cuda):
    c, s = torch.zeros(16, 64, dtype=torch.uint8, device=cuda), torch.zeros(16, 4, dtype=torch.uint8, device=cuda)
    for args, what in (((c.int(), s), "uint8"), ((c, s[:, :3].contiguous()), "K / 32"), ((c[:, :50].contiguous(), s), "128"),
                       ((c.t(), s), "contiguous"), ((c[0], s[0]), "contiguous"), ((c, s.cpu()), "HIP device"),
                       ((c, s, torch.zeros(2, 1, 4352, dtype=torch.uint8, device=cuda)), "out must be")):
        with pytest.raises(RuntimeError, match=what):
            ops.pack_w4(*args)
    p = ops.pack_w4(c, s)
    with pytest.raises(RuntimeError, match="packed must be"):
        ops.unpack_w4(p, 17, 128)


def _check_linear(ops, dev, rng, T, N, K):
    xc, xs = _act(rng, T, K)
    codes, scales = _matrix(rng, N, K)
    p = ops.pack_w4(_dev(codes, dev), _dev(scales, dev))
    y = ops.linear_w4(_dev(xc, dev, F8), _dev(xs, dev), p, N)
    assert y.dtype == torch.bfloat16 and y.shape == (T, N)
    want, bound = oracle.linear(xc, xs, oracle.decode(codes, scales))
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= bound).all(), (T, N, K, float((err / bound).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 257])
@pytest.mark.parametrize("N,K", [(16, 128), (1, 512), (17, 384), (48, 640), (131, 1152), (64, 1536), (528, 2048)])
def test_linear_w4(ops, cuda, T, N, K):
    _check_linear(ops, cuda, np.random.default_rng(T * N + K), T, N, K)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(1, 4096, 7168), (33, 2064, 7168), (3, 7168, 2048), (1, 16, 16384), (600, 200, 896),
                                   (2050, 96, 256)])
def test_linear_w4_large(ops, cuda, T, N, K):
    _check_linear(ops, cuda, np.random.default_rng(T + N + K), T, N, K)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(65, 7168, 2048), (300, 1301, 384), (700, 530, 1152), (4100, 100, 128), (257, 2064, 640),
                                   (960, 4096, 128), (1200, 4091, 256), (1900, 4096, 128), (1200, 8192, 128)])
def test_linear_w4_tiles(ops, cuda, T, N, K):
    """Sizes that run in tiles: ragged ends of every kind, and of 1 to 5 fragments a wave."""
    _check_linear(ops, cuda, np.random.default_rng(T + N + K), T, N, K)


@pytest.mark.gpu
def test_linear_w4_same_rows_at_any_batch(ops, cuda):
    """A NaN row, and rows behind it, leave the others' values alone."""
    rng = np.random.default_rng(12)
    xc, xs = _act(rng, 700, 640)
    xc[333] = 0x7F
    codes, scales = _matrix(rng, 1040, 640)
    p = ops.pack_w4(_dev(codes, cuda), _dev(scales, cuda))
    y = ops.linear_w4(_dev(xc, cuda, F8), _dev(xs, cuda), p)
    assert torch.isnan(y[333]).all() and torch.isfinite(y[:333]).all() and torch.isfinite(y[334:]).all()
    few = ops.linear_w4(_dev(xc[325:341], cuda, F8), _dev(np.ascontiguousarray(xs[:, 325:341]), cuda), p)
    assert torch.isnan(few[8]).all() and torch.isfinite(few[:8]).all() and torch.isfinite(few[9:]).all()


@pytest.mark.gpu
def test_linear_w4_single_elements(ops, cuda):
    """One-hot activations read single weights: the operand layouts and the place of each scale, exactly."""
    rng = np.random.default_rng(8)
    N, K = 48, 640
    codes, scales = _codes(rng, N, K // 2), rng.integers(120, 135, size=(N, K // 32), dtype=np.uint8)
    w = oracle.decode(codes, scales)
    xc = np.zeros((K, K), np.uint8)
    xc[np.arange(K), np.arange(K)] = 0x38  # 1.0
    xs = np.ones((K // 128, K), np.float32)
    p = ops.pack_w4(_dev(codes, cuda), _dev(scales, cuda))
    for rows in (slice(0, K), slice(0, 16), slice(100, 133)):
        y = ops.linear_w4(_dev(xc[rows], cuda, F8), _dev(np.ascontiguousarray(xs[:, rows]), cuda), p)
        assert np.array_equal(y.double().cpu().numpy(), w.T[rows])


@pytest.mark.gpu
def test_linear_w4_special_scales(ops, cuda):
    """Scales at both ends of e8m0, the NaN scale, and an e4m3 NaN stay where they belong."""
    N, K = 20, 128
    codes = np.full((N, K // 2), 0x22, np.uint8)  # all 1.0
    scales = np.full((N, K // 32), 127, np.uint8)
    scales[0], scales[1], scales[2] = 0, 254, 255
    xc = np.zeros((3, K), np.uint8)
    xc[0, 0], xc[1, 3] = 0x38, 0x7F
    p = ops.pack_w4(_dev(codes, cuda), _dev(scales, cuda))
    y = ops.linear_w4(_dev(xc, cuda, F8), torch.ones(1, 3, device=cuda), p, N).double().cpu().numpy()
    assert y[0, 0] == 2.0**-127 and y[0, 1] == 2.0**127 and np.isnan(y[0, 2]) and (y[0, 3:] == 1).all()
    assert np.isnan(y[1]).all() and (y[2, 3:] == 0).all()


@pytest.mark.gpu
def test_linear_w4_refusals(ops, cuda):
    x, xs = torch.zeros(4, 256, device=cuda).to(F8), torch.ones(2, 4, device=cuda)
    p = torch.zeros(3, 1, 4352, dtype=torch.uint8, device=cuda)
    assert ops.linear_w4(x, xs, p).shape == (4, 48)
    assert ops.linear_w4(x[:0], xs[:, :0].contiguous(), p, 33).shape == (0, 33)
    for args, what in (((x.float(), xs, p), "e4m3"), ((x, xs.t().contiguous(), p), "x_scale"), ((x, xs, p, 32), "n_out"),
                       ((x, xs, p, 49), "n_out"), ((x, xs, p[:, :, :-1]), "pack_w4"), ((x, xs, p.cpu()), "HIP device"),
                       ((x, xs, p[0]), "pack_w4"), ((x[:, :200].contiguous(), xs, p), "128"), ((x, xs.double(), p), "x_scale")):
        with pytest.raises(RuntimeError, match=what):
            ops.linear_w4(*args)


def _experts_case(rng, T, hidden, inter, E, k, picks):
    xc, xs = _act(rng, T, hidden)
    w13 = [_matrix(rng, 2 * inter, hidden) for _ in range(E)]
    w2 = [_matrix(rng, hidden, inter) for _ in range(E)]
    ids = picks(rng, T, k, E).astype(np.int32)
    weights = rng.random((T, k)).astype(np.float32)
    return xc, xs, w13, w2, ids, weights


def _run_experts(ops, dev, case, offset):
    xc, xs, w13, w2, ids, weights = case
    packed = [ops.pack_w4(_dev(np.stack([c for c, _ in w]), dev), _dev(np.stack([s for _, s in w]), dev)) for w in (w13, w2)]
    return ops.experts_w4(_dev(xc, dev, F8), _dev(xs, dev), *packed, _dev(ids, dev), _dev(weights, dev), offset)


def _check_experts(ops, dev, case, offset):
    xc, xs, w13, w2, ids, weights = case
    out = _run_experts(ops, dev, case, offset)
    wide = [np.stack([oracle.decode(c, s) for c, s in w]) for w in (w13, w2)]
    want, bound = oracle.experts(xc, xs, *wide, ids, weights, offset)
    err = np.abs(out.double().cpu().numpy() - want)
    assert out.dtype == torch.bfloat16
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())
    # the bound is not empty: nearly all of the result is where it should be
    assert np.linalg.norm(err) <= 0.01 * np.linalg.norm(want) + 1e-30
    return out


def _even(rng, T, k, E):
    return np.argsort(rng.random((T, 4 * E)), axis=1)[:, :k]


def _one(rng, T, k, E):
    return np.broadcast_to(np.array([E + 1 + i for i in range(k)]), (T, k)).copy()


def _none(rng, T, k, E):
    return np.where(rng.random((T, k)) < 0.5, -1, 100000)


def _repeated(rng, T, k, E):
    ids = _even(rng, T, k, E)
    ids[:, 1:] = ids[:, :1]
    ids[::3] = E
    return ids


def _wild(rng, T, k, E):
    return rng.integers(-(2**31), 2**31, size=(T, k))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 2, 7, 16, 17, 40, 100, 300, 400, 1000])
@pytest.mark.parametrize("hidden,inter,E,k", [(128, 128, 3, 2), (640, 384, 5, 4), (512, 1152, 2, 2)])
def test_experts_w4(ops, cuda, T, hidden, inter, E, k):
    rng = np.random.default_rng(T + hidden)
    for picks in (_even, _one, _none, _repeated, _wild):
        case = _experts_case(rng, T, hidden, inter, E, k, picks)
        out = _check_experts(ops, cuda, case, E)
        local = ((case[4].astype(np.int64) - E >= 0) & (case[4].astype(np.int64) - E < E)).any(1)
        assert out[torch.from_numpy(~local).to(cuda)].count_nonzero() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 19, 130, 450])
def test_experts_w4_layer_size(ops, cuda, T):
    rng = np.random.default_rng(T)
    case = _experts_case(rng, T, 7168, 2048, 2, 8, lambda r, t, k, e: _even(r, t, k, 4))
    _check_experts(ops, cuda, case, 1)


@pytest.mark.gpu
def test_experts_w4_many_experts_and_picks(ops, cuda):
    """More picks than one workgroup sorts (2048), 1024 experts, up to 64 picks a token."""
    rng = np.random.default_rng(5)
    for T, E, k in ((40, 1024, 64), (130, 1024, 64), (2100, 40, 5), (8193, 3, 1)):
        case = _experts_case(rng, T, 128, 128, E, k, lambda r, t, kk, e: np.argsort(r.random((t, e)), axis=1)[:, :kk])
        _check_experts(ops, cuda, case, 0)


@pytest.mark.gpu
def test_experts_w4_same_result_every_time(ops, cuda):
    rng = np.random.default_rng(6)
    for T in (3, 9, 30, 700):
        case = _experts_case(rng, T, 256, 256, 4, 4, lambda r, t, k, e: _even(r, t, k, 2))
        first = _run_experts(ops, cuda, case, 0)
        for _ in range(3):
            assert torch.equal(_run_experts(ops, cuda, case, 0), first)


@pytest.mark.gpu
def test_experts_w4_refusals(ops, cuda):
    rng = np.random.default_rng(7)
    xc, xs, w13, w2, ids, weights = _experts_case(rng, 4, 384, 128, 2, 2, _even)
    p13, p2 = (ops.pack_w4(_dev(np.stack([c for c, _ in w]), cuda), _dev(np.stack([s for _, s in w]), cuda)) for w in (w13, w2))
    good = dict(x=_dev(xc, cuda, F8), x_scale=_dev(xs, cuda), w13=p13, w2=p2, ids=_dev(ids, cuda), weights=_dev(weights, cuda))
    assert ops.experts_w4(**good).shape == (4, 384)
    for bad, what in ((dict(ids=good["ids"].long()), "ids"), (dict(ids=good["ids"][:3]), "ids"),
                      (dict(weights=good["weights"].double()), "weights"), (dict(weights=good["weights"][:, :1].contiguous()), "weights"),
                      (dict(w2=p2[:1]), "same experts"), (dict(w2=p13), "w2"), (dict(w13=p2), "w"), (dict(w13=p13[0]), "w13"),
                      (dict(x=good["x"][:, :128].contiguous()), "x_scale"), (dict(local_offset=-1), "local_expert_offset"),
                      (dict(ids=good["ids"][:, :0].contiguous(), weights=good["weights"][:, :0].contiguous()), "top_k"),
                      (dict(ids=good["ids"].cpu()), "HIP device")):
        with pytest.raises(RuntimeError, match=what):
            ops.experts_w4(**{**good, **bad})
    empty = {**good, "x": good["x"][:0], "x_scale": good["x_scale"][:, :0].contiguous(), "ids": good["ids"][:0], "weights": good["weights"][:0]}
    assert ops.experts_w4(**empty).shape == (0, 384)


@pytest.mark.gpu
def test_w4_rows_behind_the_batch_stay(lib, capi, ops, cuda):
    """Nothing is written past the last token of the caller's buffers."""
    rng = np.random.default_rng(9)
    T, N, K = 19, 37, 256
    xc, xs = _act(rng, T, K)
    codes, scales = _matrix(rng, N, K)
    p = ops.pack_w4(_dev(codes, cuda), _dev(scales, cuda))
    x, s = _dev(xc, cuda, F8), _dev(xs, cuda)
    out = torch.full((T * N + 64,), -7.0, dtype=torch.bfloat16, device=cuda)
    capi.check(lib.moe_linear_w4(x.data_ptr(), s.data_ptr(), p.data_ptr(), T, N, K, out.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream), "linear_w4")
    assert (out[T * N:] == -7.0).all() and torch.equal(out[:T * N].view(T, N), ops.linear_w4(x, s, p, N))
    q = torch.full((T * K + 64,), 1, dtype=torch.uint8, device=cuda)
    sc = torch.full((2 * T + 16,), -7.0, device=cuda)
    y = torch.randn(T, K, device=cuda)
    capi.check(lib.moe_quant_act(y.data_ptr(), 0, K, T, K, q.data_ptr(), sc.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream), "quant_act")
    assert (q[T * K:] == 1).all() and (sc[2 * T:] == -7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 400])
def test_w4_layer_run(ops, cuda, T):
    """The operators together, as a layer with 4-bit experts and a shared expert uses them: bf16 hidden states -> logits
    and FP8 activations -> picks -> routed experts, and the shared expert as dense products; then the same captured into
    a graph and replayed over new states, with eager work between."""
    g = torch.Generator().manual_seed(T)
    inter, E = 256, 8
    router = ops.pack_router((torch.randn(256, 7168, generator=g) * 7168**-0.5).bfloat16().to(cuda))
    bias = (torch.randn(256, generator=g) * 0.1).to(cuda)

    def weight(*shape):
        w = (torch.randn(*shape, generator=g) * shape[-1] ** -0.5).bfloat16().to(cuda)
        codes, scales = ops.quantize_w4(w)
        return ops.pack_w4(codes, scales), oracle.decode(codes.cpu().numpy(), scales.cpu().numpy())

    w13, w13_f = weight(E, 2 * inter, 7168)
    w2, w2_f = weight(E, 7168, inter)
    s13, s13_f = weight(2 * inter, 7168)
    s2, s2_f = weight(7168, inter)

    def layer(hidden):
        logits, hq, hs = ops.router_quant(hidden, router)
        weights, ids = ops.route_topk(logits, bias, 8, "sigmoid", 8, 4, scale=2.5)
        routed = ops.experts_w4(hq, hs, w13, w2, ids, weights, 64)
        u = ops.linear_w4(hq, hs, s13).float()
        c = (u[:, :inter] * torch.nn.functional.silu(u[:, inter:])).bfloat16()
        return logits, ids, weights, hq, hs, routed, c, ops.linear_w4(*ops.quant_act(c), s2)

    hidden = torch.randn(T, 7168, generator=g).bfloat16().to(cuda)
    logits, ids, weights, hq, hs, routed, c, shared = layer(hidden)
    _, want_ids = orouter.route(logits.cpu().numpy(), bias.cpu().numpy(), 8, "sigmoid", 8, 4, 2, True, 2.5)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    n = slice(0, 60)  # the oracle's 64-bit products, on some of the rows
    xc, xs = hq.view(torch.uint8).cpu().numpy()[n], np.ascontiguousarray(hs.cpu().numpy()[:, n])
    want, bound = oracle.experts(xc, xs, w13_f, w2_f, want_ids[n], weights.cpu().numpy()[n], 64)
    assert (np.abs(routed.double().cpu().numpy()[n] - want) <= bound).all()
    u, _ = oracle.linear(xc, xs, s13_f)
    cc, cs = oracle.quant_act(c.float().cpu().numpy()[n])
    want, bound = oracle.linear(cc, cs, s2_f)
    assert (np.abs(shared.double().cpu().numpy()[n] - want) <= bound).all()

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = layer(hidden)
    for i in range(3):
        hidden.copy_(torch.randn(T, 7168, generator=g).bfloat16())
        for t in captured:
            t.view(torch.uint8).fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, layer(hidden)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_w4_two_streams(ops, cuda):
    """Two calls at once, each on its own stream with its own workspace."""
    rng = np.random.default_rng(10)
    cases = [_experts_case(rng, T, 512, 256, 4, 4, lambda r, t, k, e: _even(r, t, k, 2)) for T in (33, 260)]
    want = [_run_experts(ops, cuda, c, 0) for c in cases]
    args = []
    for xc, xs, w13, w2, ids, weights in cases:
        packed = [ops.pack_w4(_dev(np.stack([c for c, _ in w]), cuda), _dev(np.stack([s for _, s in w]), cuda)) for w in (w13, w2)]
        args.append((_dev(xc, cuda, F8), _dev(xs, cuda), *packed, _dev(ids, cuda), _dev(weights, cuda)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(5):
        for s, a in zip(streams, args):
            with torch.cuda.stream(s):
                got.append(ops.experts_w4(*a))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


# ------------------------------------------------------------------------------------------------ the layer and its loader
def test_checkpoint_w4_refusals(tmp_path):
    ck = importlib.import_module("15642_moe_amd.checkpoint")
    with pytest.raises(ValueError, match="0..255"):
        ck.load_moe_layer_w4(tmp_path, 0, 250, 10)
    with pytest.raises(ValueError, match="0..255"):
        ck.load_moe_layer_w4(tmp_path, 0, 0, 0)
    with pytest.raises(RuntimeError, match="HIP device"):
        ck.load_moe_layer_w4(tmp_path, 0, 0, 1, device="cpu")


@pytest.mark.gpu
def test_checkpoint_w4(tmp_path, ops, cuda):
    """A layer's FP8 experts from a checkpoint, in 4 bits: some rows of every part against the oracle's quantisation."""
    from oracle.numerics import E4M3_TABLE

    ck = importlib.import_module("15642_moe_amd.checkpoint")
    rng = np.random.default_rng(20)

    def expert():
        w = [torch.from_numpy(e4m3_encode(rng.standard_normal(s).astype(np.float32))).view(F8) for s in ((4096, 7168), (7168, 2048))]
        s = [torch.from_numpy(rng.uniform(1e-3, 1e-2, n).astype(np.float32)) for n in ((32, 56), (56, 16))]
        return w[0], s[0], w[1], s[1]

    experts = {7: expert(), 8: expert()}
    bias = torch.linspace(-1, 1, 256)
    ck.save_moe_layer(tmp_path, 3, experts, bias)
    layer = ck.load_moe_layer_w4(tmp_path, 3, 7, 2, device=cuda)
    assert layer.router_weight is None and torch.equal(layer.routing_bias.cpu(), bias)
    for e in (0, 1):
        for packed, w, s, N, K in ((layer.w13[e], *experts[7 + e][:2], 4096, 7168), (layer.w2[e], *experts[7 + e][2:], 7168, 2048)):
            codes, scales = (t.cpu().numpy() for t in ops.unpack_w4(packed, N, K))
            for row in (0, 127, 128, 2047, 2048, N - 1):
                wide = E4M3_TABLE[w[row].view(torch.uint8).numpy()].astype(np.float32) * np.repeat(s[row // 128].numpy(), 128)
                want = oracle.quantize(wide[None])
                assert np.array_equal(codes[row], want[0][0]) and np.array_equal(scales[row], want[1][0])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 33, 300])
def test_moe_forward_w4_equals_fp8(ops, cuda, T):
    """4-bit weights whose scales are equal over 128 x 128 blocks are e4m3 weights with those block scales, exactly: both
    layers' results lie within the oracle's bounds of one exact result, so within two of each other."""
    rng = np.random.default_rng(T)
    E, off = 2, 32

    def pair(N, K):
        codes = _codes(rng, E, N, K // 2)
        block = rng.integers(116, 120, size=(E, N // 128, K // 128), dtype=np.uint8)
        scales = np.repeat(np.repeat(block, 128, 1), 4, 2)
        fp8 = e4m3_encode(oracle.E2M1.astype(np.float32))
        w8 = np.stack([fp8[codes & 15], fp8[codes >> 4]], -1).reshape(E, N, K)
        packed = ops.pack_w4(_dev(codes, cuda), _dev(np.ascontiguousarray(scales), cuda))
        return packed, _dev(w8, cuda, F8), _dev(np.ldexp(1.0, block.astype(np.int32) - 127).astype(np.float32), cuda), (codes, scales)

    p13, f13, s13, c13 = pair(4096, 7168)
    p2, f2, s2, c2 = pair(7168, 2048)
    xc, xs = _act(rng, T, 7168)
    x, s = _dev(xc, cuda, F8), _dev(xs, cuda)
    logits = torch.from_numpy(rng.standard_normal((T, 256)).astype(np.float32)).to(cuda)
    bias = torch.zeros(256, device=cuda)
    bias[off] = 2.0
    y4 = ops.moe_forward_w4(x, s, p13, p2, logits, bias, 2.5, off)
    y8 = ops.moe_forward(x, s, ops.pack_w13(f13), s13, ops.pack_w2(f2), s2, logits, bias, 2.5, off)
    n = slice(0, 20)
    weights, ids = orouter.route(logits.cpu().numpy(), bias.cpu().numpy(), 8, "sigmoid", 8, 4, 2, True, 2.5)
    want, bound = oracle.experts(xc[n], np.ascontiguousarray(xs[:, n]), oracle.decode(*c13), oracle.decode(*c2), ids[n],
                                 weights[n], off)
    a, b = (t.double().cpu().numpy() for t in (y4, y8))
    assert (np.abs(a[n] - want) <= bound).all()
    assert (np.abs(a[n] - b[n]) <= 2 * bound).all()
    assert np.linalg.norm(a - b) <= 0.01 * np.linalg.norm(b) and np.linalg.norm(b) > 0


@pytest.mark.gpu
def test_experts_w4_refuses_weights_that_would_lose_their_gradient(ops, cuda):
    rng = np.random.default_rng(30)
    x, s = ops.quant_act(torch.from_numpy(rng.standard_normal((3, 128)).astype(np.float32)).to(cuda))
    w13 = ops.pack_w4(*ops.quantize_w4(torch.from_numpy(rng.standard_normal((2, 256, 128)).astype(np.float32)).to(cuda)))
    w2 = ops.pack_w4(*ops.quantize_w4(torch.from_numpy(rng.standard_normal((2, 128, 128)).astype(np.float32)).to(cuda)))
    logits = torch.from_numpy(rng.standard_normal((3, 2)).astype(np.float32)).to(cuda).requires_grad_()
    weights, ids = ops.route_topk(logits, None, 1)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.experts_w4(x, s, w13, w2, ids, weights)
    want = ops.experts_w4(x, s, w13, w2, ids, weights.detach())
    with torch.no_grad():
        assert torch.equal(ops.experts_w4(x, s, w13, w2, *reversed(ops.route_topk(logits, None, 1))), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantize_w4_every_value(ops, cuda, dtype):
    """Every finite value of a 16-bit type, in groups whose largest element lies up to three binades above it."""
    every = torch.arange(1 << 16).to(torch.int32).to(torch.int16).view(dtype)
    every = every[every.isfinite()]
    for up in (0, 1, 2, 3):
        top = torch.minimum(every.float().abs() * 2.0**up * 1.5, torch.tensor(torch.finfo(dtype).max))
        w = torch.zeros(every.numel(), 32)
        w[:, ::4], w[:, 1] = every.float()[:, None], top
        w = w.to(dtype).view(-1, 128)
        codes, scales = ops.quantize_w4(w.to(cuda))
        want, want_s = oracle.quantize(w.float().numpy())
        assert np.array_equal(scales.cpu().numpy(), want_s)
        assert np.array_equal(codes.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("T,N,K", [(86, 2000, 512), (87, 2000, 512), (33, 7168, 2048), (35, 7168, 1920), (190, 1030, 896)])
def test_linear_w4_streams_and_tiles(ops, cuda, T, N, K):
    """Either side of the sizes from which the product runs in tiles."""
    _check_linear(ops, cuda, np.random.default_rng(T + N + K), T, N, K)


@pytest.mark.gpu
def test_experts_w4_far_weights(ops, cuda):
    """Experts past 2^32 bytes of packed weights: each form on the last ones, against a view of theirs alone."""
    E, hidden, inter = 300, 7168, 2048
    w13 = torch.full((E, 2 * inter // 16, hidden // 512, 4352), 0x71, dtype=torch.uint8, device=cuda)
    w2 = torch.full((E, hidden // 16, inter // 512, 4352), 0x71, dtype=torch.uint8, device=cuda)
    assert w13.numel() > 1 << 32
    w13[-2:, ..., :4096].random_(0, 256)
    w2[-2:, ..., :4096].random_(0, 256)
    rng = np.random.default_rng(31)
    for T in (1, 40, 70):
        xc, xs = _act(rng, T, hidden)
        x, s = _dev(xc, cuda, F8), _dev(xs, cuda)
        ids = _dev(rng.integers(E - 2, E, size=(T, 2)).astype(np.int32), cuda)
        weights = _dev(rng.uniform(0.1, 1, (T, 2)).astype(np.float32), cuda)
        got = ops.experts_w4(x, s, w13, w2, ids, weights)
        # 32 experts, so that the same form is taken
        want = ops.experts_w4(x, s, w13[-32:], w2[-32:], ids, weights, E - 32)
        assert torch.equal(got, want) and got.count_nonzero() > 0


@pytest.mark.gpu
def test_linear_w4_far_rows(ops, cuda):
    """Activations past 2^32 bytes and outputs past 2^31 elements."""
    T, K, N = 200_000, 16_384, 11_008
    x = torch.empty(T, K, dtype=torch.bfloat16, device=cuda)
    x[:20_000] = torch.randn(20_000, K, device=cuda).to(torch.bfloat16)
    for i in range(1, 10):
        x[20_000 * i : 20_000 * (i + 1)] = x[:20_000].roll(i, 0)
    codes, scale = ops.quant_act(x)
    p = torch.full((N // 16, K // 512, 4352), 0x71, dtype=torch.uint8, device=cuda)
    p[..., :4096].random_(0, 256)
    y = ops.linear_w4(codes, scale, p)
    for lo in (0, 97_000, T - 4096):
        rows = slice(lo, lo + 4096)
        c, s = ops.quant_act(x[rows])
        assert torch.equal(c.view(torch.uint8), codes[rows].view(torch.uint8)) and torch.equal(s, scale[:, rows])
        assert torch.equal(ops.linear_w4(c, s, p), y[rows])


@pytest.mark.gpu
def test_w4_two_graphs(ops, cuda):
    """Two captured calls, replayed in turn and over each other on two streams: each has its own workspace."""
    rng = np.random.default_rng(33)
    w13 = ops.pack_w4(_dev(_codes(rng, 4, 1024, 256), cuda), torch.full((4, 1024, 16), 118, dtype=torch.uint8, device=cuda))
    w2 = ops.pack_w4(_dev(_codes(rng, 4, 512, 256), cuda), torch.full((4, 512, 16), 118, dtype=torch.uint8, device=cuda))
    runs, held = [], []
    for T in (390, 400):
        xc, xs = _act(rng, T, 512)
        args = (_dev(xc, cuda, F8), _dev(xs, cuda), w13, w2, _dev(rng.integers(0, 4, (T, 3)).astype(np.int32), cuda),
                _dev(rng.uniform(0.1, 1, (T, 3)).astype(np.float32), cuda))
        want = ops.experts_w4(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.experts_w4(*args)
        runs.append((graph, out, want, torch.cuda.Stream()))
        held.append(args)  # a replay reads them
    for _ in range(3):
        for graph, out, want, _ in runs:
            out.zero_()
            graph.replay()
        for graph, out, want, _ in runs:
            assert torch.equal(out, want)
        torch.cuda.synchronize()
        for graph, _, _, stream in runs:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for _, out, want, _ in runs:
            assert torch.equal(out, want)


@pytest.mark.gpu
def test_experts_w4_refuses_offsets_past_32_bits(ops, cuda):
    x, s = torch.zeros(1, 128, dtype=torch.uint8, device=cuda).view(F8), torch.zeros(1, 1, device=cuda)
    w13, w2 = (torch.zeros(1, n, 1, 4352, dtype=torch.uint8, device=cuda) for n in (16, 8))
    ids, weights = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.ones(1, 1, device=cuda)
    for offset in (-1, 1 << 32, (1 << 30) + 1):
        with pytest.raises(RuntimeError, match="local_expert_offset"):
            ops.experts_w4(x, s, w13, w2, ids, weights, offset)
