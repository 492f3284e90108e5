"""Rotary positions against the rotation in extended precision.

How far: the angle pos * f is off by |pos f| 2^-52 (its product and its turns) and 2 pi 2^-26 (its fraction of a turn in
fp32); sin and cos by 4 units of 2^-24; gain times them, the two products and their sum by 2^-24 each.  Together at most
(|x0| + |x1|) |gain| (10 * 2^-24 + |pos f| 2^-52), and the result is rounded once: half a step."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops():
    from dsp_amd import ops
    return ops


def check(x, y, freq, pos, layout, inverse=False, gain=1.0):
    """x, y [batch, n, heads, dim]; pos [batch, n] integers."""
    r = 2 * len(freq)
    xs, ys = x.detach().cpu().double().numpy(), y.detach().cpu().double().numpy()
    angle = np.asarray(pos, dtype=np.longdouble)[..., None] * np.asarray(freq, dtype=np.longdouble)
    angle = np.broadcast_to(angle, x.shape[:2] + (r // 2,))
    c, s = np.cos(angle).astype(np.float64)[:, :, None], np.sin(angle).astype(np.float64)[:, :, None]
    far = np.abs(angle.astype(np.float64))[:, :, None] * 2.0 ** -52
    if inverse:
        s = -s
    a, b = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    x0, x1 = xs[..., a], xs[..., b]
    most = (np.abs(x0) + np.abs(x1)) * abs(gain) * (10 * 2.0 ** -24 + far)
    half = torch.finfo(x.dtype).eps / 2
    least = 2.0 ** -25 if x.dtype == torch.float16 else 0.0  # half a step below fp16's normal range
    for got, want in ((ys[..., a], gain * (x0 * c - x1 * s)), (ys[..., b], gain * (x0 * s + x1 * c))):
        assert (np.abs(got - want) <= most + half * (np.abs(want) + most) + least).all()
    assert (ys[..., r:] == xs[..., r:]).all()


SHAPES = [  # batch, n, heads, dim, rotated
    (1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (1, 77, 3, 80, 40), (3, 10, 1, 96, 48), (2, 65, 7, 128, 128), (1, 5, 40, 256, 64),
    (1, 33, 9, 100, 36), (2, 9, 3, 7, 6), (1, 2, 2, 1024, 256), (64, 1, 20, 128, 128), (1, 600, 33, 128, 96),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("kind", TYPES)
def test_rotary(ops, dev, kind, layout, shape):
    from dsp_amd import design
    b, n, h, d, r = shape
    g = torch.Generator().manual_seed(1)
    x = torch.randn(b, n, h, d, generator=g).to(TYPES[kind]).to(dev)
    freq = design.rotary_frequencies(r)
    check(x, ops.rotary(x, freq, layout=layout), freq, np.arange(n), layout)
    pos = torch.randint(-(1 << 20), 1 << 31, (b, n), generator=g)
    y = ops.rotary(x, freq, positions=pos.to(dev), layout=layout, inverse=True, gain=1.25)
    check(x, y, freq, pos.numpy(), layout, inverse=True, gain=1.25)
    z = x.clone()
    assert ops.rotary(z, freq, position=12345, layout=layout, out=z) is z
    check(x, z, freq, 12345 + np.arange(n), layout)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides(ops, dev, layout):
    """Views of a wider buffer, heads in front of tokens, off the 16-byte grid, one position row for all, out a view."""
    g = torch.Generator().manual_seed(2)
    freq = np.array([1.0, 0.1, 0.01, 0.001])
    for kind in TYPES.values():
        for off in (0, 1, 4):
            wide = torch.randn(2, 6, 3, 40, generator=g).to(kind).to(dev)
            x = wide[..., off:off + 24].transpose(1, 2)  # [2, 3 tokens, 6 heads, 24]
            pos = torch.tensor([5, 1 << 20, 0], device=dev)
            into = torch.full((2, 3, 8, 24), 9.0, dtype=kind, device=dev)
            ops.rotary(x, freq, positions=pos, layout=layout, out=into[:, :, 1:7])
            check(x, into[:, :, 1:7], freq, pos.cpu().numpy()[None], layout)
            assert (into[:, :, 0] == 9).all() and (into[:, :, 7] == 9).all()
            check(x, ops.rotary(x, freq, positions=pos.expand(2, 3), layout=layout), freq, pos.cpu().numpy()[None], layout)
    x = torch.randn(1, 1, 4, 24, generator=g).to(dev).expand(3, 5, 4, 24)  # one row for all tokens
    check(x, ops.rotary(x, freq, layout=layout), freq, np.arange(5), layout)
    y = ops.rotary(x[0], freq, layout=layout)  # [n, heads, dim]
    check(x[:1], y[None], freq, np.arange(5), layout)


def test_back_is_the_gradient(ops, dev):
    """<rotate(x), g> = <x, rotate_back(g)>, and a difference along a direction: the call is linear."""
    gen = torch.Generator().manual_seed(3)
    x, g = (torch.randn(2, 9, 3, 64, generator=gen).to(dev) for _ in range(2))
    freq = 0.3 ** np.arange(24)
    for layout in ("half", "interleaved"):
        y, back = ops.rotary(x, freq, layout=layout, gain=1.1), ops.rotary(g, freq, layout=layout, gain=1.1, inverse=True)
        # elements from 48 on pass unscaled both ways; 3456 products, each side 12 * 2^-24 off at most
        left, right = (y.double() * g.double()).sum(), (x.double() * back.double()).sum()
        assert abs(left - right) <= 4 * 12 * 2.0 ** -24 * (x.double().norm() * g.double().norm())
        up, down = ops.rotary(x + g, freq, layout=layout), ops.rotary(x - g, freq, layout=layout)
        assert ((up.double() - down.double()) / 2 - ops.rotary(g, freq, layout=layout).double()).abs().max() <= 32 * 2.0 ** -24 * (x.abs() + g.abs()).max()


def test_empty_stream_and_graph(ops, dev):
    x = torch.randn(4, 50, 6, 64, dtype=torch.float32, device=dev).to(torch.bfloat16)
    freq, pos = 0.5 ** np.arange(32), torch.arange(200, device=dev).view(4, 50)
    assert ops.rotary(x[:, :0], freq).shape == (4, 0, 6, 64) and ops.rotary(x[:0], freq).shape == (0, 50, 6, 64)
    want = ops.rotary(x, freq, positions=pos)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.rotary(x, freq, positions=pos)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.rotary(x, freq, positions=pos)
    for _ in range(3):
        pos += 7
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.rotary(x, freq, positions=pos))


def test_refusals(ops, dev):
    from dsp_amd.capi import DspGpuError
    x = torch.zeros(2, 3, 4, 16, device=dev)
    f, pos = np.ones(4), torch.zeros(2, 3, dtype=torch.int64, device=dev)
    for i, call in enumerate((
            lambda: ops.rotary(x.double(), f), lambda: ops.rotary(x.cpu(), f), lambda: ops.rotary(x[0, 0], f),
            lambda: ops.rotary(x, np.ones(9)), lambda: ops.rotary(x, []), lambda: ops.rotary(x, [math.nan]), lambda: ops.rotary(x, [f]),
            lambda: ops.rotary(x, f, layout="other"), lambda: ops.rotary(x, f, gain=math.inf), lambda: ops.rotary(x.transpose(-1, -2), f),
            lambda: ops.rotary(x, f, positions=pos.int()), lambda: ops.rotary(x, f, positions=pos.cpu()), lambda: ops.rotary(x, f, positions=pos[:, :2]),
            lambda: ops.rotary(x, f, out=x.half()), lambda: ops.rotary(x, f, out=x[:1]), lambda: ops.rotary(x[:, :2], f, out=x[:, 1:]))):
        with pytest.raises(DspGpuError) as e:
            call()
        assert e.value.code == -1, i
