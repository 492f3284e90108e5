"""What the sequence-layer entry points write must not meet anything else (CPU: refused before any HIP call)."""
import ctypes as C

import numpy as np
import pytest

from dsp_amd import capi
from test_sequence_refusals import BASE, K, O, Q, S, T, V, decay, forward, shape

STATE = 4 * 2 * 8 * 8  # bytes of the states of shape(): one sequence, two heads, 8 x 8
DQ, DK, DV = S, S + 512, S + 1024


def backward(sh, dq=DQ, dk=DK, dv=DV, s_in=None, d_out=None, d_in=None, ws=None, nws=0):
    return capi.lib().dsp_gpu_linear_attention_backward(Q, K, V, O, dq, dk, dv, sh, decay(-0.1, -0.1), 1.0, s_in, d_out, d_in, ws, nws, None)


@pytest.mark.parametrize("at", [DQ, DK, DV, DQ - STATE + 4, DV + 64], ids=["dq", "dk", "dv", "in front of dq", "in dv"])
def test_gradients_over_the_gradient_of_the_state_after(at):
    assert backward(shape(), d_out=at) == capi.EINVAL


@pytest.mark.parametrize("by", [0, 8, -8])
def test_outputs_over_offsets_and_lengths(by):
    if by >= 0:  # one length, 8 bytes; two offsets, 16
        assert forward(shape(lengths=O + by)) == capi.EINVAL
        assert forward(shape(lengths=T + by), s_out=T) == capi.EINVAL
    assert forward(shape(rows=4, offsets=O + by)) == capi.EINVAL
    assert forward(shape(rows=4, offsets=T + by), s_in=T, s_out=T) == capi.EINVAL


@pytest.mark.parametrize("at", [DQ, DK, DV + 16, T, T + STATE - 8], ids=["dq", "dk", "in dv", "dstate", "end of dstate"])
def test_gradients_over_offsets_and_lengths(at):
    assert backward(shape(lengths=at), d_in=T) == capi.EINVAL
    assert backward(shape(rows=4, offsets=at), d_in=T) == capi.EINVAL


def test_workspace_over_anything():
    """Buffers of 1,024 tokens at addresses far apart; the workspace over the first or the last bytes of one after the other."""
    n, L = 1024, capi.lib()
    at = {name: (1 << 40) + (i << 32) for i, name in enumerate(("q", "k", "v", "o", "s_in", "s_out", "index", "dq", "dk", "dv", "d_out", "d_in"))}
    for back in (0, 1):
        for more in (dict(lengths=at["index"]), dict(rows=n, offsets=at["index"])):
            sh = shape(n=n, **more)
            need = C.c_size_t(0)
            assert L.dsp_gpu_linear_attention_workspace(sh, back, C.byref(need)) == capi.OK and need.value > 0
            for name in at:
                if name in (("s_out",) if back else ("dq", "dk", "dv", "d_out", "d_in")):
                    continue
                for ws in (at[name], at[name] - (need.value + 15) // 16 * 16 + 16):
                    if back:
                        rc = L.dsp_gpu_linear_attention_backward(*(at[x] for x in ("q", "k", "v", "o", "dq", "dk", "dv")), sh, decay(-0.1, -0.1),
                                                                 1.0, at["s_in"], at["d_out"], at["d_in"], ws, need.value, None)
                    else:
                        rc = L.dsp_gpu_linear_attention(*(at[x] for x in ("q", "k", "v", "o")), sh, decay(-0.1, -0.1), 1.0, at["s_in"],
                                                        at["s_out"], ws, need.value, None)
                    assert rc == capi.EINVAL and b"workspace" in L.dsp_gpu_last_error_string(), (back, name)


def test_more_than_any_memory():
    """Extents that 64 bits do not hold would come out small, and overlap nothing."""
    huge = 1 << 40
    for bad in (dict(batch=1 << 24, n=4, q=(huge, 16, 8)), dict(batch=2, n=1 << 31, q=(16, huge, 8)), dict(batch=1 << 24, n=4, o=(huge, 16, 8))):
        assert forward(shape(**bad)) == capi.EINVAL, bad
        need = C.c_size_t(0)
        assert capi.lib().dsp_gpu_linear_attention_workspace(shape(**bad), 0, C.byref(need)) == capi.EINVAL, bad
    st, f = capi.STRIDES3, np.ones(4).tobytes()
    good = dict(x=Q, y=BASE + (1 << 42), kind=capi.F32, batch=1 << 24, n=4, heads=2, dim=8, xs=st.pack(64, 16, 8), ys=st.pack(64, 16, 8), f=f,
                rot=8, layout=0, pos=None, ps=None, at=0, gain=1.0, direction=0)
    for bad in (dict(xs=st.pack(huge, 16, 8)), dict(ys=st.pack(huge, 16, 8)), dict(xs=st.pack(0, 0, 0), batch=1 << 31, n=1 << 31, ys=st.pack(huge, 16, 8)),
                dict(pos=T, ps=capi.STRIDES2.pack(1 << 62, 1)), dict(pos=T, ps=capi.STRIDES2.pack(0, 1 << 62))):
        assert capi.lib().dsp_gpu_rotary(*{**good, **bad}.values(), None) == capi.EINVAL, bad
