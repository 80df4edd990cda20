"""Products with 4-bit weights on the GPU against their definition in 64 bits: every group size,
scale type, tile remainder and token count, values at float32's ends, and the same bits for a token
in whatever batch."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from q4_helpers import quantize, sum_tolerance

pytestmark = pytest.mark.gpu
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def up(dev, a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    return t if dtype is None else t.to(dtype)


def matrix(ie, dev, rng, rows, cols, group, scale="f16", zero=False):
    packed, s, z, w = quantize(rng, rows, cols, group, scale, zero)
    return ie.matrix_q4(up(dev, packed), up(dev, s, DTYPES[scale]), group,
                        zero=None if z is None else up(dev, z)), w


def activations(rng, T, cols):
    x = rng.standard_normal((T, cols), dtype=np.float32)
    x[:, rng.integers(0, cols, max(1, cols // 200))] *= np.float32(25)
    return x


def product(ie, dev, m, x, bias=None, y0=None):
    T = x.shape[0]
    y = torch.full((T, m.rows), float("nan"), device=dev) if y0 is None else up(dev, y0)
    ie.matmul_q4(y, up(dev, x), m, None if bias is None else up(dev, bias),
                 accumulate=y0 is not None, workspace=ie.matmul_q4_workspace(T, m.cols, dev))
    torch.cuda.synchronize()
    return y.cpu().numpy()


SHAPES = [
    # T, rows, cols, group
    (1, 16, 32, 32), (1, 1, 32, 128), (2, 17, 64, 64), (3, 5, 96, 64), (5, 33, 160, 128),
    (16, 130, 896, 128), (17, 1111, 2080, 32), (33, 127, 1056, 64), (1, 1152, 896, 128),
    (64, 96, 4864, 128), (15, 48, 4864, 32), (65, 256, 512, 64), (128, 300, 1024, 128),
    (129, 257, 992, 32), (300, 129, 640, 128), (7, 9000, 128, 32), (4, 20000, 224, 64),
    (48, 40000, 64, 64), (31, 152000, 32, 128), (513, 515, 352, 64), (1000, 80, 128, 128),
]


@pytest.mark.parametrize("T,rows,cols,group", SHAPES)
@pytest.mark.parametrize("scale,zero", [("f16", False), ("bf16", True), ("f32", True)])
def test_matmul(ie, dev, T, rows, cols, group, scale, zero):
    print(f"matmul_q4 {T} x {rows} x {cols}, groups of {group}, {scale}, zero {zero}", flush=True)
    rng = np.random.default_rng(T + rows + cols)
    m, w = matrix(ie, dev, rng, rows, cols, group, scale, zero)
    x = activations(rng, T, cols)
    bias = rng.standard_normal(rows, dtype=np.float32) if zero else None
    y0 = rng.standard_normal((T, rows), dtype=np.float32) if scale == "f32" else None
    got = product(ie, dev, m, x, bias, y0)
    want = x.astype(np.float64) @ w.T
    tol = sum_tolerance(cols, group, w, x)
    if bias is not None:
        want, tol = want + bias, tol + 2.0 ** -22 * np.abs(bias)
    if y0 is not None:
        want, tol = want + y0, tol + 2.0 ** -22 * np.abs(y0)
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("T", [1, 16, 40, 200])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_qkv_is_the_matmul(ie, dev, T, group):
    """Each output in its own buffer, bit for bit the stacked product's columns."""
    rng = np.random.default_rng(T)
    q_dim, kv_dim, cols = 448, 64, 896
    m, _ = matrix(ie, dev, rng, q_dim + 2 * kv_dim, cols, group, zero=group == 64)
    x, bias = activations(rng, T, cols), rng.standard_normal(q_dim + 2 * kv_dim, dtype=np.float32)
    q, k, v = (torch.full((T, d), float("nan"), device=dev) for d in (q_dim, kv_dim, kv_dim))
    ie.qkv_proj_q4(q, k, v, up(dev, x), m, up(dev, bias),
                   workspace=ie.matmul_q4_workspace(T, cols, dev))
    got = torch.cat([q, k, v], 1).cpu().numpy()
    assert np.array_equal(got.view(np.uint32), product(ie, dev, m, x, bias).view(np.uint32))


@pytest.mark.parametrize("T,rows,cols", [(1, 4864, 896), (13, 100, 96), (64, 640, 896),
                                         (150, 333, 480), (2, 70000, 64)])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gate_up(ie, dev, T, rows, cols, group):
    rng = np.random.default_rng(rows)
    mg, wg = matrix(ie, dev, rng, rows, cols, group, "bf16", True)
    mu, wu = matrix(ie, dev, rng, rows, cols, group, "bf16", False)
    x = activations(rng, T, cols)
    out = torch.full((T, rows), float("nan"), device=dev)
    ie.gate_up_silu_q4(out, up(dev, x), mg, mu, workspace=ie.matmul_q4_workspace(T, cols, dev))
    a, b = x.astype(np.float64) @ wg.T, x.astype(np.float64) @ wu.T
    with np.errstate(over="ignore"):
        sig = 1 / (1 + np.exp(-a))
    # |d silu| <= 1.1 |d a|; f32's exp, sum, division and products: 4 ulps of the result.
    tol = (1.1 * sum_tolerance(cols, group, wg, x) * np.abs(b)
           + np.abs(a * sig) * sum_tolerance(cols, group, wu, x) + 2.0 ** -21 * np.abs(a * sig * b))
    # expf of an argument known to 2^-24 |a|: the sigmoid's own relative error.
    tol += 2.0 ** -23 * np.abs(a) * np.abs(a * sig * b) + 1e-35
    err = np.abs(out.cpu().numpy() - a * sig * b)
    assert (err <= tol).all(), float((err / tol).max())


def test_a_token_does_not_depend_on_its_batch(ie, dev):
    """Bit for bit, over every kernel a token count may take, wide and narrow matrices."""
    rng = np.random.default_rng(3)
    for rows, cols, group in ((257, 2080, 32), (64, 896, 128), (20000, 256, 64), (8200, 4864, 128)):
        m, _ = matrix(ie, dev, rng, rows, cols, group, zero=True)
        x = activations(rng, 400, cols)
        want = product(ie, dev, m, x).view(np.uint32)
        for T in (1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 256, 257):
            got = product(ie, dev, m, x[:T]).view(np.uint32)
            assert np.array_equal(got, want[:T]), (rows, cols, T)
        alone = product(ie, dev, m, x[399:]).view(np.uint32)
        assert np.array_equal(alone, want[399:])


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("cols", [32, 992, 1024, 1056])
def test_few_rows_of_many_tokens(ie, dev, cols, group):
    """Matrices of up to a few row tiles, on both sides of the rules that let their products split the
    tokens: bit for bit what the tokens are alone, each kind of product."""
    rng = np.random.default_rng(cols + group)
    for rows, T in ((31, 700), (64, 2041), (65, 700), (250, 250), (256, 256), (257, 257)):
        m, _ = matrix(ie, dev, rng, rows, cols, group, zero=True)
        up_m, _ = matrix(ie, dev, rng, rows, cols, group, zero=True)
        x = activations(rng, T, cols)
        x[T // 2, 0] = np.inf
        x[T - 1] = 0
        got = product(ie, dev, m, x).view(np.uint32)
        out = torch.full((T, rows), float("nan"), device=dev)
        ie.gate_up_silu_q4(out, up(dev, x), m, up_m, workspace=ie.matmul_q4_workspace(T, cols, dev))
        for t in (0, 15, 16, T // 2, T - 1):
            assert np.array_equal(got[t:t + 1], product(ie, dev, m, x[t:t + 1]).view(np.uint32)), (rows, T, t)
            one = torch.empty((1, rows), device=dev)
            ie.gate_up_silu_q4(one, up(dev, x[t:t + 1]), m, up_m)
            assert torch.equal(one.view(torch.int32), out[t:t + 1].view(torch.int32)), (rows, T, t)


@pytest.mark.parametrize("cols", [1952, 2080])
@pytest.mark.parametrize("group", [32, 128])
def test_many_tokens_on_both_sides_of_a_rule(ie, dev, cols, group):
    """108 tiles of 128 x 128, which one count of columns takes as tiles and the other by slots: bit for
    bit what the tokens are eight at a time."""
    rng = np.random.default_rng(cols + group)
    m, _ = matrix(ie, dev, rng, 1501, cols, group, zero=True)
    x = activations(rng, 1030, cols)
    got = product(ie, dev, m, x).view(np.uint32)
    for t in (0, 511, 1022):
        assert np.array_equal(got[t:t + 8], product(ie, dev, m, x[t:t + 8]).view(np.uint32)), t


def test_every_weight_and_zero_point(ie, dev):
    """All 16 values against zero points to 255, one column at a time: exact."""
    q = np.tile(np.arange(16, dtype=np.uint8), 2)[None].repeat(256, 0)
    z = np.arange(256, dtype=np.uint8)[:, None]
    m = ie.matrix_q4(up(dev, q[:, 0::2] | (q[:, 1::2] << 4)), torch.ones((256, 1), device=dev), 32,
                     zero=up(dev, z))
    for T in (32, 128):
        x = np.eye(32, dtype=np.float32)[np.arange(T) % 32] * np.float32(3)
        want = (3.0 * (q.astype(np.float64) - z)).T[np.arange(T) % 32]
        assert np.array_equal(product(ie, dev, m, x).astype(np.float64), want)


@pytest.mark.parametrize("T", [2, 100])
def test_ends_of_float32(ie, dev, T):
    """Blocks of zeros, denormals, and values near both ends of the range keep 23 bits; infinities
    and NaN go the way of the plain product and touch their own token only."""
    rng = np.random.default_rng(9)
    cols, rows = 384, 40
    packed, s, z, w = quantize(rng, rows, cols, 128, "f32", True)
    q = np.stack((packed & 15, packed >> 4), -1).reshape(rows, cols)
    q[q == np.repeat(z, 128, 1)] ^= 1  # no zero weights: infinity times a weight stays infinite
    w = (q.astype(np.float64) - np.repeat(z, 128, 1)) * np.repeat(s.astype(np.float64), 128, 1)
    m = ie.matrix_q4(up(dev, q[:, 0::2] | (q[:, 1::2] << 4)), up(dev, s), 128, zero=up(dev, z))
    base = activations(rng, T, cols)
    for scale in (1e-30, 1e-20, 1e20, 1e34):
        x = base * np.float32(scale)
        err = np.abs(product(ie, dev, m, x) - x.astype(np.float64) @ w.T)
        assert (err <= sum_tolerance(cols, 128, w, x)).all(), scale
    assert not product(ie, dev, m, base * 0).any()
    tiny = np.abs(product(ie, dev, m, (base * np.float32(1e-42)))) # below 2^-126: gone or nearly
    assert (tiny <= 1e-37).all()
    x = base.copy()
    x[0, 200] = np.inf
    x[1, 3], x[1, 4] = np.nan, -np.inf
    got, plain = product(ie, dev, m, x), product(ie, dev, m, base)
    assert np.array_equal(got[0], np.where(w[:, 200] > 0, np.inf, -np.inf))
    assert np.isnan(got[1]).all()
    assert np.array_equal(got[2:], plain[2:])


def test_offsets_past_32_bits(ie, dev):
    """A matrix of more than 4 GiB: its last rows."""
    rows, cols = 140000, 65536
    data = torch.zeros((rows, cols // 2), dtype=torch.uint8, device=dev)
    scale = torch.ones((rows, cols // 128), dtype=torch.float16, device=dev)
    data[-1] = 0x99
    data[-2, -1] = 0xA8
    m = ie.matrix_q4(data, scale, 128)
    for T in (1, 40):
        x = torch.ones((T, cols), device=dev)
        y = torch.empty((T, rows), device=dev)
        ie.matmul_q4(y, x, m, workspace=ie.matmul_q4_workspace(T, cols, dev))
        assert (y[:, -1] == cols).all() and (y[:, -2] == -8 * (cols - 2) + 2).all()
        assert (y[:, 0] == -8 * cols).all()


def test_stream_and_graph(ie, dev):
    """On a side stream, and captured: replays with new inputs between eager calls."""
    rng = np.random.default_rng(5)
    m, _ = matrix(ie, dev, rng, 300, 896, 64)
    for T in (4, 90):
        xs = [up(dev, activations(rng, T, 896)) for _ in range(4)]
        ws, y = ie.matmul_q4_workspace(T, 896, dev), torch.empty((T, 300), device=dev)
        eager = lambda x: (ie.matmul_q4(e := torch.empty_like(y), x, m,
                                        workspace=ie.matmul_q4_workspace(T, 896, dev)), e)[1]
        want = [eager(x) for x in xs]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        ie.matmul_q4(y, xs[0], m, workspace=ws, stream=s)
        s.synchronize()
        assert torch.equal(y, want[0])
        x = xs[0].clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ie.matmul_q4(y, x, m, workspace=ws)
        for xi, wi in zip(xs, want):
            x.copy_(xi)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, wi)
            assert torch.equal(eager(xi), wi)


@pytest.mark.parametrize("T,cols", [(1, 23552), (1, 23584), (1, 16384), (2, 5888), (4, 5888), (3, 5920), (16, 1408),
                                    (9, 1376), (16, 1440), (4, 1024), (12, 1024)])
@pytest.mark.parametrize("group", [32, 128])
def test_room_for_the_activations(ie, dev, T, cols, group):
    """At and past the sizes whose split activations fit beside each stage size: the same bits as the
    same tokens among many."""
    rng = np.random.default_rng(cols)
    m, w = matrix(ie, dev, rng, 75, cols, group, "f16", True)
    x = activations(rng, 20, cols)
    got, many = product(ie, dev, m, x[:T]), product(ie, dev, m, x)
    assert np.array_equal(got.view(np.uint32), many[:T].view(np.uint32))
    assert (np.abs(got - x[:T].astype(np.float64) @ w.T) <= sum_tolerance(cols, group, w, x[:T])).all()
    out = [torch.full((t, 75), float("nan"), device=dev) for t in (T, 20)]
    for o in out:
        t = o.shape[0]
        ie.gate_up_silu_q4(o, up(dev, x[:t]), m, m, workspace=ie.matmul_q4_workspace(t, cols, dev))
    assert torch.equal(out[0], out[1][:T])
