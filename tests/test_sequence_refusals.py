"""What the sequence-layer entry points refuse (CPU: every check comes before any HIP call), the C struct's layout, the
designers, and the 64-bit reference against differences."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import sequence_reference as ref
from dsp_amd import capi, design, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = (C.c_char * (1 << 16))()
BASE = (C.addressof(BUF) + 255) & ~255
Q, K, V, O, S, T = (BASE + 8192 * i for i in range(6))


def shape(batch=1, n=4, rows=0, heads=2, hq=2, hk=2, hv=2, dk=8, dv=8, kind=capi.BF16, offsets=0, lengths=0, o=None, q=None):
    def st(h, d):
        return (n * h * d, h * d, d)
    return capi.ATTENTION_SHAPE.pack(batch, n, rows, heads, hq, hk, hv, dk, dv, kind, *(q or st(hq, dk)), *st(hk, dk), *st(hv, dv),
                                     *(o or st(heads, dv)), offsets, lengths, 0)


def decay(*v):
    return np.array(v, dtype=np.float64).tobytes()


def forward(sh, q=Q, k=K, v=V, o=O, ld=decay(-0.1, -0.1), scale=1.0, s_in=None, s_out=None, ws=None, nws=0):
    return capi.lib().dsp_gpu_linear_attention(q, k, v, o, sh, ld, scale, s_in, s_out, ws, nws, None)


REFUSED = {
    "sample type": dict(kind=capi.F64), "no heads": dict(heads=0), "too many heads": dict(heads=257, hq=1, hk=1, hv=1),
    "heads of q": dict(heads=4, hq=3), "heads of k": dict(heads=4, hk=8), "heads of v": dict(heads=4, hv=0),
    "dim_k": dict(dk=0), "dim_k too large": dict(dk=257), "dim_v": dict(dv=257), "both": dict(offsets=BASE, lengths=BASE),
    "negative stride": dict(q=(64, -16, 8)), "rows of o overlap": dict(o=(64, 8, 8)), "huge batch": dict(batch=1 << 25),
}


@pytest.mark.parametrize("case", REFUSED)
def test_shapes_refused(case):
    assert forward(shape(**REFUSED[case])) == capi.EINVAL
    assert b"dsp_gpu_linear_attention" in capi.lib().dsp_gpu_last_error_string()


def test_arguments_refused():
    sh = shape()
    assert forward(None) == capi.EINVAL
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(o=None), dict(ld=None), dict(ld=decay(0.1, -1.0)),
                dict(ld=decay(math.nan, -1.0)), dict(scale=math.inf), dict(o=Q), dict(o=V), dict(o=Q + 64),
                dict(s_in=O), dict(s_out=O), dict(s_out=Q), dict(s_in=S, s_out=S + 64)):
        assert forward(sh, **bad) == capi.EINVAL, bad
    assert forward(shape(batch=0)) == capi.OK
    L = capi.lib()
    back = lambda dq=S, dk=S + 512, dv=S + 1024, s_in=None, d_out=None, d_in=None: L.dsp_gpu_linear_attention_backward(  # noqa: E731
        Q, K, V, O, dq, dk, dv, sh, decay(-0.1, -0.1), 1.0, s_in, d_out, d_in, None, 0, None)
    for bad in (dict(dq=None), dict(dk=None), dict(dv=None), dict(dq=Q), dict(dk=O), dict(dv=V + 16), dict(dk=S), dict(d_in=S),
                dict(d_out=T, d_in=T), dict(s_in=S)):
        assert back(**bad) == capi.EINVAL, bad
    one = shape(n=1)
    step = lambda sh=one, q=Q, o=O, s=S, slots=None, n=0: L.dsp_gpu_linear_attention_step(  # noqa: E731
        q, K, V, o, sh, decay(-0.1, -0.1), 1.0, s, slots, n, None)
    for bad in (dict(sh=shape(n=2)), dict(sh=shape(n=1, lengths=T)), dict(q=None), dict(o=None), dict(s=None), dict(o=S), dict(s=Q),
                dict(slots=T, n=0), dict(slots=S, n=4)):
        assert step(**bad) == capi.EINVAL, bad
    assert step(sh=shape(batch=0, n=1)) == capi.OK
    need = C.c_size_t(1)
    assert L.dsp_gpu_linear_attention_workspace(sh, 0, C.byref(need)) == capi.OK and need.value == 0
    big = shape(n=4096)
    for backward in (0, 1):
        assert L.dsp_gpu_linear_attention_workspace(big, backward, C.byref(need)) == capi.OK and need.value > 0
    assert L.dsp_gpu_linear_attention_workspace(None, 0, C.byref(need)) == capi.EINVAL
    far = 1 << 40  # buffers far enough apart for the larger shape; the call stops at the workspace
    assert forward(big, q=far, k=2 * far, v=3 * far, o=4 * far, ws=T, nws=16) == capi.EINVAL
    assert b"workspace" in L.dsp_gpu_last_error_string()
    assert forward(big, q=far, k=2 * far, v=3 * far, o=4 * far, ws=T + 8, nws=1 << 40) == capi.EINVAL


def test_rotary_refused():
    st = capi.STRIDES3.pack(64, 16, 8)
    f = np.ones(4).tobytes()
    good = dict(x=Q, y=K, kind=capi.F32, batch=1, n=4, heads=2, dim=8, xs=st, ys=st, f=f, rot=8, layout=0, pos=None, ps=None, at=0,
                gain=1.0, direction=0)

    def call(**bad):
        return capi.lib().dsp_gpu_rotary(*{**good, **bad}.values(), None)

    nan, minus = np.array([1.0, math.nan, 1.0, 1.0]).tobytes(), capi.STRIDES3.pack(64, -16, 8)
    for bad in (dict(x=None), dict(y=None), dict(kind=capi.F64), dict(heads=0), dict(dim=1), dict(dim=1025), dict(xs=None),
                dict(ys=None), dict(f=None), dict(f=nan), dict(rot=7), dict(rot=0), dict(rot=16), dict(dim=512, rot=512),
                dict(layout=2), dict(pos=T), dict(gain=math.inf), dict(direction=2), dict(xs=minus), dict(y=Q + 16),
                dict(y=Q, xs=capi.STRIDES3.pack(64, 32, 8)), dict(ys=capi.STRIDES3.pack(64, 8, 8)), dict(ys=capi.STRIDES3.pack(64, 0, 8)),
                dict(pos=K, ps=capi.STRIDES2.pack(0, 1)), dict(pos=T, ps=capi.STRIDES2.pack(0, -1)), dict(n=1 << 40)):
        assert call(**bad) == capi.EINVAL, bad
    assert call(batch=0) == capi.OK and call(n=0) == capi.OK


def test_python_refusals():
    x = torch.zeros(1, 4, 2, 8)
    for call in (lambda: ops.rotary(x, [1.0]), lambda: ops.rotary(np.zeros((4, 2, 8), np.float32), [1.0]),
                 lambda: ops.linear_attention(x, x, x, [-0.1, -0.1]), lambda: ops.linear_attention_step(x[0], x[0], x[0], [-0.1, -0.1], x),
                 lambda: ops.linear_attention_backward(x, x, x, [-0.1, -0.1], x)):
        with pytest.raises(capi.DspGpuError) as e:
            call()
        assert e.value.code == capi.EINVAL


def test_struct_layout(tmp_path):
    """capi.ATTENTION_SHAPE packs what the compiler lays out."""
    fields = "batch n rows heads heads_q heads_k heads_v dim_k dim_v sample_type q_stride k_stride v_stride o_stride offsets lengths zero_rest"
    src = tmp_path / "layout.cpp"
    src.write_text('#include <cstdio>\n#include <cstddef>\n#include "dsp_gpu.h"\nint main() {\n' + "".join(
        f'    std::printf("%zu ", offsetof(dsp_gpu_linear_attention_shape, {f}));\n' for f in fields.split())
        + '    std::printf("%zu\\n", sizeof(dsp_gpu_linear_attention_shape));\n}\n')
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    packed = capi.ATTENTION_SHAPE.pack(*range(1, 11), *range(11, 23), 23, 24, 25)
    assert got[-1] == capi.ATTENTION_SHAPE.size
    ints = {0: 8, 1: 8, 2: 8, **{i: 4 for i in range(3, 10)}, 10: 8, 11: 8, 12: 8, 13: 8, 14: 8, 15: 8, 16: 4}
    want = [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 14, 17, 20, 23, 24, 25]
    for i, (off, w) in enumerate(zip(got, want)):
        assert int.from_bytes(packed[off:off + ints[i]], "little") == w, i


def test_designers():
    f = design.rotary_frequencies(64)
    assert f.shape == (32,) and f[0] == 1.0 and math.isclose(f[16], 10000.0 ** -0.5)
    assert np.allclose(design.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4.0, rtol=1e-15)
    b = design.rotary_frequencies(64, scaling="base", factor=8.0)
    assert b[0] == f[0] and math.isclose(b[-1], f[-1] / 8.0, rel_tol=1e-12) and (b <= f).all()
    r = design.rotary_frequencies(64, scaling="ramp", factor=8.0, original_length=4096)
    turns = 4096 * f / (2 * math.pi)
    assert (r[turns >= 32] == f[turns >= 32]).all() and np.allclose(r[turns <= 1], f[turns <= 1] / 8.0, rtol=1e-15)
    assert ((r <= f) & (r >= f / 8.0)).all()
    assert design.rotary_frequencies(2, scaling="base", factor=8.0)[0] == 1.0
    for bad in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, base=0.0), dict(rot_dim=8, factor=0.0), dict(rot_dim=8, scaling="x"),
                dict(rot_dim=8, scaling="ramp", fast_turns=1.0, slow_turns=1.0)):
        with pytest.raises(ValueError):
            design.rotary_frequencies(**bad)
    d = design.head_decays(8)
    assert d.shape == (8,) and np.allclose(np.exp(d[[0, -1]]), [1 - 1 / 32, 1 - 1 / 512]) and (np.diff(d) > 0).all()
    assert design.head_decays(1).shape == (1,)
    with pytest.raises(ValueError):
        design.head_decays(0)


def test_reference_gradients_against_differences():
    """The formulas the GPU tests hold the kernels to, against central differences of the forward recurrence in 64 bits."""
    g = torch.Generator().manual_seed(3)
    b, n, h, dk, dv = 2, 5, 2, 3, 4
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    q, k, v, s0, do, d1 = r(b, n, h, dk), r(b, n, h, dk), r(b, n, h, dv), r(b, h, dk, dv), r(b, n, h, dv), r(b, h, dk, dv)
    ld, scale = [-0.3, -1.1], 0.7

    def loss(q, k, v, s0):
        o, end = ref.forward(q, k, v, ld, scale, s0)
        return (o * do).sum() + (end * d1).sum()

    grads = ref.backward(q, k, v, ld, scale, s0, do, d1)
    for i, (x, gx) in enumerate(zip((q, k, v, s0), grads)):
        for _ in range(6):
            at = tuple(int(torch.randint(0, m, (), generator=g)) for m in x.shape)
            args = [t.clone() for t in (q, k, v, s0)]
            args[i][at] += 1e-4
            up = loss(*args)
            args[i][at] -= 2e-4
            assert math.isclose((up - loss(*args)) / 2e-4, gx[at], rel_tol=1e-7, abs_tol=1e-7)
