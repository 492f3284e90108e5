"""What the sequence-layer calls ask for as workspace (CPU: the query makes no HIP call)."""
import ctypes as C

import pytest

from dsp_amd import capi


def workspace(backward, batch, n, rows, heads, dk, dv, kind=capi.BF16, packed=True, shared=1):
    st = lambda h, d: (n * h * d, h * d, d)  # noqa: E731
    hq = heads // shared
    shape = capi.ATTENTION_SHAPE.pack(batch, n, rows, heads, hq, heads, heads, dk, dv, kind, *st(hq, dk), *st(heads, dk), *st(heads, dv),
                                      *st(heads, dv), 256 if packed else 0, 0, 0)
    need = C.c_size_t(0)
    assert capi.lib().dsp_gpu_linear_attention_workspace(shape, backward, C.byref(need)) == capi.OK
    return need.value


@pytest.mark.parametrize("batch,rows", [(16, 20011), (64, 8192), (256, 32768), (1000, 32768), (1024, 131072), (30000, 1000000)])
@pytest.mark.parametrize("heads,dk,dv", [(16, 128, 128), (1, 128, 128), (8, 64, 64), (4, 256, 256)])
@pytest.mark.parametrize("backward", [0, 1])
def test_packed_batches_ask_for_what_their_rows_can_hold(backward, heads, dk, dv, batch, rows):
    """A segment with another one behind it has 128 rows at least: rows / 128 states for each gradient, however many sequences
    there are and whatever max_length is (left out: all rows)."""
    state = 4 * heads * dk * dv
    most = (3 if backward else 1) * (rows // 128) * state + 4096
    for n in (rows, rows // 2):
        assert workspace(backward, batch, n, rows, heads, dk, dv) <= most


@pytest.mark.parametrize("batch,n", [(1, 600), (2, 2048), (8, 2048), (4, 300), (3, 32768)])
def test_dense_batches_ask_for_the_states_between_segments(batch, n):
    """At most n / 128 segments, and a state between each two of them -- none for the one before the first token."""
    heads, d = 2, 64
    assert workspace(0, batch, n, 0, heads, d, d, packed=False) <= (n // 128 - 1) * batch * 4 * heads * d * d + 256
