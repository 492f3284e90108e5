"""Host-side mirror of the reference's hot-path interface, on top of the C ABI.

Names and argument meaning follow the reference (file:line relative to its dsp/include/dsp/):

    fft0(x, inverse)                  fft.h:31-55      complex [.., 2^k] -> complex, unnormalised
    fft(x_real, nf, inverse, shift)   fft.h:57-94      real rows, zero padded to 2^ceil(log2 nf)
    convolve(x, taps, mode)           convolution.h:8-29 / filter.h:123-140
    moving_average(x, npoints)        filter.h:81-101
    iir(x, a, b, c0, d0, state, mode) coefficients.h:88-130,172-195

Sequence layers (no counterpart in the reference; torch CUDA tensors, fp32, fp16 or bf16):

    rotary(x, inv_freq, positions)                    pairs of each head turned by pos * inv_freq, and back
    linear_attention(q, k, v, log_decay)              S_t = w S_{t-1} + k_t v_t^T, o_t = scale q_t S_t, whole sequences
    linear_attention_backward(q, k, v, log_decay, do) its gradients
    linear_attention_step(q, k, v, log_decay, state)  one token a row, states updated in place

Nothing here is recorded by autograd: outputs of inputs that require gradients have none, and the gradients of the sequence
layers are calls of their own (rotary with inverse=True, linear_attention_backward), for a torch.autograd.Function to make.

Inputs are torch CUDA tensors (device pointers, asynchronous on the current torch stream)
or numpy arrays (host pointers, staged by the library).  fp32 unless a name says otherwise.  No CPU fallback.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import capi

try:  # torch is plumbing for device memory / streams only
    import torch
except Exception:  # pragma: no cover
    torch = None


def _is_torch(x) -> bool:
    return torch is not None and isinstance(x, torch.Tensor)


def _stream_of(x) -> int:
    if _is_torch(x) and x.is_cuda:
        return torch.cuda.current_stream(x.device).cuda_stream
    return 0


def _prep(x, dtype_np, dtype_torch_name):
    """-> (contiguous array/tensor, data pointer, mem flag)"""
    if _is_torch(x):
        want = getattr(torch, dtype_torch_name)
        if not x.is_cuda:
            raise capi.DspGpuError(capi.EINVAL, "torch tensors must live on the GPU (pass numpy for host memory)")
        if x.dtype != want:
            raise capi.DspGpuError(capi.EINVAL, f"expected {want}, got {x.dtype}")
        x = x.contiguous()
        return x, x.data_ptr(), capi.MEM_DEVICE
    x = np.ascontiguousarray(x, dtype=dtype_np)
    return x, x.ctypes.data, capi.MEM_HOST


def _empty_like(x, shape, dtype_np, dtype_torch_name):
    if _is_torch(x):
        return torch.empty(shape, dtype=getattr(torch, dtype_torch_name), device=x.device)
    return np.empty(shape, dtype=dtype_np)


def _ptr(a):
    return a.data_ptr() if _is_torch(a) else a.ctypes.data


def _out(out, x, shape, dtype_np, dtype_torch_name):
    """The output buffer: a fresh one, or the caller's after the checks the kernels rely on (they write `count`
    elements through a raw pointer: same kind of container and device as x, dtype, size, contiguity)."""
    if out is None:
        return _empty_like(x, shape, dtype_np, dtype_torch_name)
    count = int(np.prod(shape))
    if _is_torch(out) != _is_torch(x):
        raise capi.DspGpuError(capi.EINVAL, "out must live where x lives (torch tensor with torch, numpy with numpy)")
    if _is_torch(out):
        ok = (out.device == x.device and out.dtype == getattr(torch, dtype_torch_name) and out.numel() == count
              and out.is_contiguous())
    else:
        ok = out.dtype == dtype_np and out.size == count and out.flags.c_contiguous and out.flags.writeable
    if not ok:
        raise capi.DspGpuError(capi.EINVAL, f"out must be a contiguous {dtype_torch_name} buffer of {count} elements on x's device")
    return out


class _on_device:
    """Runs the C call with x's GPU current: the library takes its workspaces and tables from hipGetDevice()."""

    def __init__(self, x):
        self._ctx = torch.cuda.device(x.device) if _is_torch(x) and x.is_cuda else None

    def __enter__(self):
        if self._ctx is not None:
            self._ctx.__enter__()

    def __exit__(self, *exc):
        if self._ctx is not None:
            return self._ctx.__exit__(*exc)
        return False


def fft0(x, inverse: bool = False, out=None):
    """Batched complex FFT over the last axis (length 2^k, k in 1..30).  fft.h:31-55."""
    x, px, mem = _prep(x, np.complex64, "complex64")
    n = x.shape[-1]
    log2n = int(n).bit_length() - 1
    if n < 2 or (1 << log2n) != n:
        raise capi.DspGpuError(capi.EINVAL, f"transform length {n} is not a power of two >= 2")
    batch = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    out = _out(out, x, tuple(x.shape), np.complex64, "complex64")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_fft_batch(px, _ptr(out), log2n, batch, capi.INVERSE if inverse else capi.FORWARD,
                                                mem, _stream_of(x)))
    return out


def fft0_f64(x, inverse: bool = False, out=None):
    """The same in the reference's own sample type, std::complex<double> (fft.h:31-32): complex128 in and out, double
    arithmetic, length 2^k with k in 1..24."""
    x, px, mem = _prep(x, np.complex128, "complex128")
    n = x.shape[-1]
    log2n = int(n).bit_length() - 1
    if n < 2 or (1 << log2n) != n:
        raise capi.DspGpuError(capi.EINVAL, f"transform length {n} is not a power of two >= 2")
    batch = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    out = _out(out, x, tuple(x.shape), np.complex128, "complex128")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_fft_batch_f64(px, _ptr(out), log2n, batch, capi.INVERSE if inverse else capi.FORWARD,
                                                    mem, _stream_of(x)))
    return out


def fft(x, nf: int, inverse: bool = False, shift: bool = False, out=None):
    """Real-input wrapper dsp::fft (fft.h:57-83), optionally followed by dsp::shift (fft.h:85-94)."""
    x, px, mem = _prep(x, np.float32, "float32")
    n_in = x.shape[-1]
    batch = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    log2n = max(1, int(np.ceil(np.log2(nf))))
    out = _out(out, x, tuple(x.shape[:-1]) + (1 << log2n,), np.complex64, "complex64")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_fft_real_batch(px, n_in, n_in, _ptr(out), int(nf), batch,
                                                     capi.INVERSE if inverse else capi.FORWARD, int(shift), mem,
                                                     _stream_of(x)))
    return out


_MODES = {"auto": capi.CONV_AUTO, "direct": capi.CONV_DIRECT, "time": capi.CONV_DIRECT,
          "overlap_save": capi.CONV_OVERLAP_SAVE, "frequency": capi.CONV_OVERLAP_SAVE,
          "direct_valu": capi.CONV_DIRECT_VALU}


def convolve(x, taps, mode: str = "auto", out=None):
    """Causal FIR, first len(taps)-1 outputs zero.  x: [n] or [channels, n] fp32.  filter.h:123-140."""
    x, px, mem = _prep(x, np.float32, "float32")
    taps = np.ascontiguousarray(taps, dtype=np.float32)  # the designers produce double; the device runs fp32
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    y = _out(out, x, tuple(x.shape), np.float32, "float32")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_convolve(px, _ptr(y), channels, n, taps.ctypes.data, taps.size, _MODES[mode], mem,
                                               _stream_of(x)))
    return y


def convolve_f64(x, taps, mode: str = "auto", out=None):
    """The same filter on double samples with double taps: SincFilter<>::apply(SampleBuffer<double>&), filter.h:123-140
    (time domain on the double matrix cores; mode "auto" or "direct")."""
    x, px, mem = _prep(x, np.float64, "float64")
    taps = np.ascontiguousarray(taps, dtype=np.float64)
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    y = _out(out, x, tuple(x.shape), np.float64, "float64")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_convolve_f64(px, _ptr(y), channels, n, taps.ctypes.data, taps.size, _MODES[mode], mem,
                                                   _stream_of(x)))
    return y


def convolve_stream(x, taps, history, position: int, mode: str = "direct", out=None):
    """One chunk of a streamed FIR.  history: [channels, len(taps)-1] fp32 where x lives, updated in place;
    position = samples of the stream consumed so far (0 starts it; the first len(taps)-1 outputs of the
    stream are zero as in the one-shot call)."""
    x, px, mem = _prep(x, np.float32, "float32")
    taps = np.ascontiguousarray(taps, dtype=np.float32)
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    if _is_torch(history) != _is_torch(x):
        raise capi.DspGpuError(capi.EINVAL, "history must live where x lives")
    want = channels * (taps.size - 1)
    ok = (history.is_contiguous() and history.dtype == torch.float32 and history.numel() == want) if _is_torch(history) \
        else (history.flags.c_contiguous and history.dtype == np.float32 and history.size == want)
    if not ok:
        raise capi.DspGpuError(capi.EINVAL, "history must be contiguous fp32 [channels, ntaps-1]")
    y = _out(out, x, tuple(x.shape), np.float32, "float32")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_convolve_stream(px, _ptr(y), channels, n, taps.ctypes.data, taps.size,
                                                      _ptr(history) if want else None, int(position), _MODES[mode], mem,
                                                      _stream_of(x)))
    return y


def moving_average(x, npoints: int, out=None):
    """Centred moving average, zero edges.  filter.h:81-101."""
    x, px, mem = _prep(x, np.float32, "float32")
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    y = _out(out, x, tuple(x.shape), np.float32, "float32")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_moving_average(px, _ptr(y), channels, n, int(npoints), mem, _stream_of(x)))
    return y


def moving_average_f64(x, npoints: int, out=None):
    """MovingAverageFilter::apply on double samples (filter.h:81-101)."""
    x, px, mem = _prep(x, np.float64, "float64")
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    y = _out(out, x, tuple(x.shape), np.float64, "float64")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_moving_average_f64(px, _ptr(y), channels, n, int(npoints), mem, _stream_of(x)))
    return y


_IIR_MODES = {"auto": capi.IIR_AUTO, "batch": capi.IIR_BATCH, "scan": capi.IIR_SCAN, "batch_ref": capi.IIR_BATCH_REF}


def _iir_any(x, f64, a, b, c0, d0, state, mode, out):
    np_t, torch_t = (np.float64, "float64") if f64 else (np.float32, "float32")
    x, px, mem = _prep(x, np_t, torch_t)
    a = np.ascontiguousarray(a, dtype=np.float64)
    b = np.ascontiguousarray(b, dtype=np.float64)
    if a.size != b.size:
        raise capi.DspGpuError(capi.EINVAL, "a and b must have poles+1 entries each")
    poles = a.size - 1
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    y = _out(out, x, tuple(x.shape), np_t, torch_t)
    pstate = None
    if state is not None:
        if _is_torch(state) != _is_torch(x):
            raise capi.DspGpuError(capi.EINVAL, "state must live where x lives")
        if _is_torch(state):
            if not (state.is_contiguous() and state.dtype == torch.float64 and state.numel() == channels * 2 * poles):
                raise capi.DspGpuError(capi.EINVAL, "state must be contiguous float64 [channels, 2*poles]")
        elif not (state.flags.c_contiguous and state.dtype == np.float64 and state.size == channels * 2 * poles):
            raise capi.DspGpuError(capi.EINVAL, "state must be contiguous float64 [channels, 2*poles]")
        pstate = _ptr(state)
    fn = capi.lib().dsp_gpu_iir_f64 if f64 else capi.lib().dsp_gpu_iir
    with _on_device(x):
        capi.check(fn(px, _ptr(y), channels, n, a.ctypes.data, b.ctypes.data, poles, float(c0), float(d0), pstate,
                      _IIR_MODES[mode], mem, _stream_of(x)))
    return y


def iir(x, a, b, c0: float = 1.0, d0: float = 0.0, state=None, mode: str = "auto", out=None):
    """IIR recursion with feedback ADDED (coefficients.h:106-130), fp32 samples.

    state: [channels, 2*poles] float64 {x[t-1..t-poles], v[t-1..t-poles]}, updated in place
    (the reference's x[]/y[] history, coefficients.h:11-12).  mode "batch_ref": the reference's own arithmetic,
    bit for bit (float accumulator for the generic section, the all-double BiQuad for two poles)."""
    return _iir_any(x, False, a, b, c0, d0, state, mode, out)


def iir_f64(x, a, b, c0: float = 1.0, d0: float = 0.0, state=None, mode: str = "auto", out=None):
    """The same on double samples: Coefficients<P>::operator()(const SampleBuffer<double>&), the instantiation every
    in-repo caller of the reference uses (eval/recursive_filters/main.cpp:35).  One lane per channel ("scan" is
    unsupported, "auto" runs "batch")."""
    return _iir_any(x, True, a, b, c0, d0, state, mode, out)


def iir_settle(a, b) -> int:
    """Samples after which the response to any initial state has decayed below 2^-44 of it (dsp_gpu_iir_settle);
    host arithmetic only."""
    import ctypes as C
    a = np.ascontiguousarray(a, dtype=np.float64)
    b = np.ascontiguousarray(b, dtype=np.float64)
    if a.size != b.size:
        raise capi.DspGpuError(capi.EINVAL, "a and b must have poles+1 entries each")
    out = C.c_size_t(0)
    capi.check(capi.lib().dsp_gpu_iir_settle(a.ctypes.data, b.ctypes.data, a.size - 1, C.byref(out)))
    return int(out.value)


def iir_multi(x, a, b, c0=None, d0=None, state=None, out=None, mode: str = "batch", f64: bool = False):
    """Filter bank: channel k runs its own Coefficients (a[k], b[k], c0[k], d0[k]); a, b [channels, poles+1]
    float64, c0/d0 [channels] float64 or None (1 and 0), all living where x lives.  Block-wise form of a
    retuned filter (eval/signals/wind_generator.h:150-167): call per block with new coefficients, carry `state`.
    f64: double samples; mode "batch_ref": the reference's own arithmetic (dsp_gpu_iir_multi_ex)."""
    np_t, torch_t = (np.float64, "float64") if f64 else (np.float32, "float32")
    x, px, mem = _prep(x, np_t, torch_t)
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    poles = a.shape[-1] - 1

    def chk(t, count, what):
        if t is None:
            return None
        if _is_torch(t) != _is_torch(x):
            raise capi.DspGpuError(capi.EINVAL, f"{what} must live where x lives")
        ok = (t.is_contiguous() and t.dtype == torch.float64 and t.numel() == count) if _is_torch(t) \
            else (t.flags.c_contiguous and t.dtype == np.float64 and t.size == count)
        if not ok:
            raise capi.DspGpuError(capi.EINVAL, f"{what} must be contiguous float64 with {count} entries")
        return _ptr(t)

    pa, pb = chk(a, channels * (poles + 1), "a"), chk(b, channels * (poles + 1), "b")
    pc0, pd0 = chk(c0, channels, "c0"), chk(d0, channels, "d0")
    pstate = chk(state, channels * 2 * poles, "state")
    y = _out(out, x, tuple(x.shape), np_t, torch_t)
    with _on_device(x):
        if not f64 and mode == "batch":
            capi.check(capi.lib().dsp_gpu_iir_multi(px, _ptr(y), channels, n, pa, pb, poles, pc0, pd0, pstate, mem,
                                                    _stream_of(x)))
        else:
            capi.check(capi.lib().dsp_gpu_iir_multi_ex(px, _ptr(y), capi.F64 if f64 else capi.F32, channels, n, pa, pb,
                                                       poles, pc0, pd0, pstate, _IIR_MODES[mode], mem, _stream_of(x)))
    return y


_SWEPT_KINDS = {"bandpass": 0, "bandreject": 1}


def biquad_swept(x, fc, bandwidth: float, kind: str = "bandpass", state=None, out=None):
    """A band-pass / band-reject BiQuad retuned at every sample (dsp_gpu_biquad_swept): per sample the design of
    recursive_filters.h:165-209 at centre frequency fc[t], then one BiQuad step (coefficients.h:172-182) -- the
    loop of eval/signals/wind_generator.h:150-167.  x float32 [..., n]; fc float32 of the same shape (a sweep per
    channel) or [n] (one sweep for all channels), living where x lives; state float64 [channels, 4] = {x1, x2, y1,
    y2}, carried across calls."""
    x, px, mem = _prep(x, np.float32, "float32")
    n = x.shape[-1]
    channels = int(np.prod(x.shape[:-1])) if x.ndim > 1 else 1
    if _is_torch(fc) != _is_torch(x):
        raise capi.DspGpuError(capi.EINVAL, "fc must live where x lives")
    if _is_torch(fc) and fc.device != x.device:
        raise capi.DspGpuError(capi.EINVAL, "fc must be on x's device")
    fc, pfc, _ = _prep(fc, np.float32, "float32")
    if tuple(fc.shape) == tuple(x.shape):
        stride = n
    elif tuple(fc.shape) == (n,):
        stride = 0
    else:
        raise capi.DspGpuError(capi.EINVAL, "fc must have x's shape or be one sweep of n samples")
    if kind not in _SWEPT_KINDS:
        raise capi.DspGpuError(capi.EINVAL, f"kind {kind!r}")
    pstate = None
    if state is not None:
        if _is_torch(state) != _is_torch(x):
            raise capi.DspGpuError(capi.EINVAL, "state must live where x lives")
        ok = (state.is_contiguous() and state.dtype == torch.float64 and state.numel() == channels * 4) \
            if _is_torch(state) else (state.flags.c_contiguous and state.dtype == np.float64 and state.size == channels * 4)
        if not ok:
            raise capi.DspGpuError(capi.EINVAL, "state must be contiguous float64 [channels, 4]")
        pstate = _ptr(state)
    y = _out(out, x, tuple(x.shape), np.float32, "float32")
    with _on_device(x):
        capi.check(capi.lib().dsp_gpu_biquad_swept(px, pfc, _ptr(y), channels, n, stride, _SWEPT_KINDS[kind],
                                                   float(bandwidth), pstate, mem, _stream_of(x)))
    return y


# ---- sequence layers -------------------------------------------------------------------------------------------------
# One token of a serving step is a few microseconds on the GPU: these calls keep what they do on the host short, too.  Like
# every call here they are not recorded by autograd: gradients are calls of their own.

_SAMPLE_TYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16} if torch is not None else {}
_LAYOUTS = {"half": capi.ROTARY_HALF, "interleaved": capi.ROTARY_INTERLEAVED}


# the handle of a device's current stream, without the Stream object around it (most of what asking for one costs)
_raw_stream = getattr(getattr(torch, "_C", None), "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _bad(message):
    return capi.DspGpuError(capi.EINVAL, message)


def _sample_type(x, what):
    if not _is_torch(x) or not x.is_cuda:
        raise _bad(f"{what} must be a torch tensor on the GPU")
    kind = _SAMPLE_TYPES.get(x.dtype)
    if kind is None:
        raise _bad(f"{what}: expected float32, float16 or bfloat16, got {x.dtype}")
    return kind


def _strides4(x, what):
    """(batch, token, head) strides of a [batch, n, heads, dim] tensor; packed [rows, heads, dim] and one token a row
    [n, heads, dim]: batch stride 0.  0 for an axis of one."""
    st, sh = x.stride(), x.shape
    if st[-1] != 1 and sh[-1] > 1 and x.numel():
        raise _bad(f"{what}: the last axis must be contiguous")
    if len(sh) == 3:
        return 0, st[0] if sh[0] > 1 else 0, st[1] if sh[1] > 1 else 0
    return st[0] if sh[0] > 1 else 0, st[1] if sh[1] > 1 else 0, st[2] if sh[2] > 1 else 0


def _index(x, like, count, what):
    """A device int64 array of `count` entries."""
    if not (_is_torch(x) and x.device == like.device and x.dtype == torch.int64 and tuple(x.shape) == (count,)
            and x.is_contiguous()):
        raise _bad(f"{what} must be a contiguous int64 tensor of {count} entries on x's device")
    return x.data_ptr()


def _new(like, shape):
    """A contiguous tensor of `like`'s type and device."""
    return torch.empty_like(like) if shape == like.shape and like.is_contiguous() else like.new_empty(shape)


def _same(t, like, shape, what):
    """A sample tensor of `like`'s type and device."""
    if not (_is_torch(t) and t.dtype == like.dtype and t.device == like.device and t.shape == shape):
        raise _bad(f"{what} must be a {like.dtype} tensor {tuple(shape)} on {like.device}")
    return t


def _call(x, fn, *args):
    """fn(*args, stream) with x's GPU current, on its current stream."""
    index = x.device.index
    if torch.cuda.current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(x.device):
            rc = fn(*args, _raw_stream(index))
    if rc != capi.OK:
        capi.check(rc)


def rotary(x, inv_freq, positions=None, position: int = 0, layout: str = "half", inverse: bool = False, gain: float = 1.0,
           out=None):
    """Rotary positions (dsp_gpu_rotary).  x [batch, n, heads, dim] or [n, heads, dim], any strides with a contiguous last
    axis; the first 2 * len(inv_freq) elements of each head are turned by the angle pos * inv_freq (host doubles,
    design.rotary_frequencies), pairs (i, i + half) for layout "half", (2i, 2i + 1) for "interleaved"; the rest is copied.
    positions: int64 [batch, n] or [n] on x's device, or None: position, position + 1, ...  inverse: the other way round --
    the gradient of the forward call, with the same gain (autograd does not record the call).  out may be x (in place) or any
    tensor of its shape."""
    kind = _sample_type(x, "x")
    if x.ndim not in (3, 4):
        raise _bad("x must be [batch, n, heads, dim] or [n, heads, dim]")
    if layout not in _LAYOUTS:
        raise _bad(f"layout {layout!r}")
    freq = np.ascontiguousarray(inv_freq, dtype=np.float64)
    if freq.ndim != 1:
        raise _bad("inv_freq must be one-dimensional")
    y = _new(x, x.shape) if out is None else _same(out, x, x.shape, "out")
    batch, n, heads, dim = x.shape if x.ndim == 4 else (1, *x.shape)
    ppos, pstride = None, None
    if positions is not None:
        if not (_is_torch(positions) and positions.device == x.device and positions.dtype == torch.int64
                and tuple(positions.shape) in ((batch, n), (n,))):
            raise _bad("positions must be int64 [batch, n] or [n] on x's device")
        st = positions.stride()
        pstride = capi.STRIDES2.pack(st[0] if len(st) == 2 and batch > 1 else 0, st[-1] if n > 1 else 0)
        ppos = positions.data_ptr()
    _call(x, capi.lib().dsp_gpu_rotary, x.data_ptr(), y.data_ptr(), kind, batch, n, heads, dim,
          capi.STRIDES3.pack(*_strides4(x, "x")), capi.STRIDES3.pack(*_strides4(y, "out")), freq.tobytes(), 2 * freq.size,
          _LAYOUTS[layout], ppos, pstride, position, gain, capi.INVERSE if inverse else capi.FORWARD)
    return y


class _Attention:
    """The checked arguments of a linear-attention call, and the C struct of them as bytes."""
    __slots__ = ("heads", "batch", "out_shape", "state_shape", "log_decay", "lead", "tail", "device")

    def __init__(self, q, k, v, log_decay, lengths, offsets, max_length, axes):
        kind = _sample_type(q, "q")
        if not (_is_torch(k) and _is_torch(v) and k.dtype == q.dtype == v.dtype and k.device == q.device == v.device):
            raise _bad("k and v must have q's type and device")
        qs, ks, vs = q.shape, k.shape, v.shape
        if offsets is not None:
            axes = 3
        if not len(qs) == len(ks) == len(vs) == axes or qs[:-2] != ks[:-2] or qs[:-2] != vs[:-2] or qs[-1] != ks[-1]:
            raise _bad(f"shapes of q {tuple(qs)}, k {tuple(ks)}, v {tuple(vs)} do not belong together")
        self.log_decay = np.ascontiguousarray(log_decay, dtype=np.float64)
        if self.log_decay.ndim != 1:
            raise _bad("log_decay must be one-dimensional: one value a head")
        self.heads = self.log_decay.size
        batch, n, rows, poffsets, plengths = qs[0], 1, 0, 0, 0
        if offsets is not None:
            if lengths is not None:
                raise _bad("offsets and lengths exclude each other")
            if not _is_torch(offsets) or offsets.ndim != 1 or offsets.numel() < 1:
                raise _bad("offsets must have batch + 1 entries")
            batch, rows = offsets.numel() - 1, qs[0]
            n = rows if max_length is None else int(max_length)
            if n < 0:
                raise _bad(f"max_length {n}")
            poffsets = _index(offsets, q, batch + 1, "offsets")
        elif max_length is not None:
            raise _bad("max_length goes with offsets")
        elif axes == 4:
            n = qs[1]
            if lengths is not None:
                plengths = _index(lengths, q, batch, "lengths")
        sq, sk, sv = _strides4(q, "q"), _strides4(k, "k"), _strides4(v, "v")
        if axes == 3 and offsets is None:  # one token a row: the rows are the sequences
            sq, sk, sv = ((s[1], 0, s[2]) for s in (sq, sk, sv))
        self.batch = batch
        self.out_shape = (*qs[:-2], self.heads, vs[-1])
        self.state_shape = (batch, self.heads, qs[-1], vs[-1])
        self.lead = (batch, n, rows, self.heads, qs[-2], ks[-2], vs[-2], qs[-1], vs[-1], kind, *sq, *sk, *sv)
        self.tail = (poffsets, plengths)
        self.device = q.device

    def shape(self, o, what, zero_rest, step=False):
        so = _strides4(o, what)
        return capi.ATTENTION_SHAPE.pack(*self.lead, *((so[1], 0, so[2]) if step else so), *self.tail, zero_rest)

    def state(self, t, what, shape=None):
        if t is None:
            return None
        if not (_is_torch(t) and t.dtype == torch.float32 and t.device == self.device and t.is_contiguous()
                and t.shape == (shape or self.state_shape)):
            raise _bad(f"{what} must be a contiguous float32 tensor {shape or self.state_shape} on q's device")
        return t.data_ptr()

    def workspace(self, shape, backward):
        """(tensor, pointer, bytes) of what the call needs: torch's allocator keeps calls, streams and captured graphs apart."""
        need = C.c_size_t(0)
        capi.check(capi.lib().dsp_gpu_linear_attention_workspace(shape, backward, C.byref(need)))
        if not need.value:
            return None, None, 0
        t = torch.empty(need.value, dtype=torch.uint8, device=self.device)
        return t, t.data_ptr(), need.value


def linear_attention(q, k, v, log_decay, scale: float = 1.0, state=None, new_state=None, lengths=None, offsets=None,
                     max_length=None, out=None):
    """Linear attention with a decay for each head (dsp_gpu_linear_attention): S_t = w S_{t-1} + k_t v_t^T and
    o_t = scale * q_t S_t with w = exp(log_decay[head]).  q, k [batch, n, heads, dim_k], v [batch, n, heads, dim_v], heads
    of each a divisor of len(log_decay); any strides with a contiguous last axis.  A packed batch: [rows, heads, dim] with
    offsets int64 [batch + 1] on the device, not decreasing (max_length: the longest sequence, else all rows; the memory that
    the call takes is the same); a padded one: lengths int64 [batch].  state / new_state: float32 [batch, heads, dim_k, dim_v]
    before the first and after the last token (may be the same tensor).  Returns o [batch, n, heads, dim_v] (rows of no
    sequence: zeros, or what `out` held).  Autograd does not record the call: its gradients are linear_attention_backward."""
    a = _Attention(q, k, v, log_decay, lengths, offsets, max_length, 4)
    o = _new(v, a.out_shape) if out is None else _same(out, q, a.out_shape, "out")
    shape = a.shape(o, "out", out is None)
    s_in, s_out = a.state(state, "state"), a.state(new_state, "new_state")
    ws, pws, nws = a.workspace(shape, 0)
    _call(q, capi.lib().dsp_gpu_linear_attention, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), shape,
          a.log_decay.tobytes(), scale, s_in, s_out, pws, nws)
    return o


def linear_attention_backward(q, k, v, log_decay, dout, scale: float = 1.0, state=None, dnew_state=None, dstate=None,
                              lengths=None, offsets=None, max_length=None):
    """The gradients (dq, dk, dv) of linear_attention from dout and, where given, dnew_state, that of the state after the
    last token.  `state`: as in the forward call.  dstate: a float32 tensor that receives the gradient of `state`.  Gradients
    of heads that several share are summed in order; rows of no sequence get zeros.  log_decay has none."""
    a = _Attention(q, k, v, log_decay, lengths, offsets, max_length, 4)
    shape = a.shape(_same(dout, q, a.out_shape, "dout"), "dout", True)
    s_in, ds_out, ds_in = a.state(state, "state"), a.state(dnew_state, "dnew_state"), a.state(dstate, "dstate")
    dq, dk, dv = _new(q, q.shape), _new(k, k.shape), _new(v, v.shape)
    ws, pws, nws = a.workspace(shape, 1)
    _call(q, capi.lib().dsp_gpu_linear_attention_backward, q.data_ptr(), k.data_ptr(), v.data_ptr(), dout.data_ptr(),
          dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), shape, a.log_decay.tobytes(), scale, s_in, ds_out, ds_in, pws, nws)
    return dq, dk, dv


def linear_attention_step(q, k, v, log_decay, state, scale: float = 1.0, slots=None, out=None):
    """One token a row (dsp_gpu_linear_attention_step): q, k [batch, heads, dim_k], v [batch, heads, dim_v]; `state` float32
    [batch, heads, dim_k, dim_v], updated in place -- or [n_slots, ...] with slots int64 [batch] on the device, row b working
    on state[slots[b]] (a slot outside the pool: the row is skipped; the same slot twice: in the order of the rows).
    Returns o [batch, heads, dim_v] (skipped rows: zeros)."""
    a = _Attention(q, k, v, log_decay, None, None, None, 3)
    if state is None:
        raise _bad("state must be given: it is what the step updates")
    o = _new(v, a.out_shape) if out is None else _same(out, q, a.out_shape, "out")
    if slots is None:
        pslots, n_slots, ps = None, 0, a.state(state, "state")
    else:
        n_slots = state.shape[0] if _is_torch(state) and state.ndim else 0
        pslots, ps = _index(slots, q, a.batch, "slots"), a.state(state, "state", (n_slots, *a.state_shape[1:]))
    _call(q, capi.lib().dsp_gpu_linear_attention_step, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
          a.shape(o, "out", False, True), a.log_decay.tobytes(), scale, ps, pslots, n_slots)
    return o


def fft_kernel_ms(x, out, inverse: bool, iters: int) -> float:
    """Average milliseconds per batched-FFT launch, timed with HIP events on x's stream."""
    n = x.shape[-1]
    log2n = int(n).bit_length() - 1
    batch = x.numel() // n
    ms = C.c_float(0.0)
    capi.check(capi.lib().dsp_gpu_fft_batch_timed(x.data_ptr(), out.data_ptr(), log2n, batch,
                                                  capi.INVERSE if inverse else capi.FORWARD, int(iters), C.byref(ms),
                                                  _stream_of(x)))
    return float(ms.value)
