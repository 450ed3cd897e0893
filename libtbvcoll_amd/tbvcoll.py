"""tbvcoll -- ctypes binding of libtbvcoll.so (MI355X build).

The module keeps the surface of the reference binding (step4/tbvcoll.py:14-111): `init`,
`all_reduce`, `is_async`, `err`, `rails`, `hist`, `raw_fn`, `cap`, `stats`, `stats3`,
`stats4`, `stats5`, with the same guards and return conventions, so a caller written
against the reference (a vLLM `GroupCoordinator.all_reduce` intercept, code that uses the
C function through `raw_fn`) binds without changes.  On one GPU the peer is emulated: a
two-rank exact/stress driver additionally has to hand over the peer's payload with
`stage_peer` before each call (without one the peer echoes this rank's own payload).

    import tbvcoll
    tbvcoll.init(rank, "rail0,rail1", "", cap_bytes=8 << 20)
    tbvcoll.stage_peer(peer_tensor)    # this build only: what the other rank would have sent
    tbvcoll.all_reduce(t)              # in-place SUM; False -> caller falls back

Additions (no counterpart in the reference): the emulated peer (`stage_peer`,
`stage_peer_repeat`, `peer_resident`, `arrival_script`, `hold_rail`, `withhold`,
`arrival_log`), measurement (`latency_probe`, `latencies`, `kernel_timing`, `kernel_times`,
`hbm_probe`, `launch_floor`), `all_reduce_chunked`, `shutdown`, `lib`, and the operators of the layer
around the all-reduce, which need no `init`: `quantize_int8`, `matmul_int8`, `linear_int8_all_reduce`,
`rotary`, `rotary_frequencies`.

There is no CPU fallback: if the shared library is missing, `init` raises.
"""
import ctypes
import math
import os
import struct

import torch
from torch.autograd import forward_ad as _forward

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_lib = None
_cap = 0
_DEFAULT_SO = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libtbvcoll.so")

_VP, _SZ, _I, _U64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_ulonglong
_PD, _PU, _PI, _PSZ = (ctypes.POINTER(t) for t in (ctypes.c_double, ctypes.c_ulonglong, ctypes.c_int, ctypes.c_size_t))

# symbol -> (restype, argtypes): everything include/tbvcoll.h and include/tbvcoll_emu.h declare
_SIGNATURES = {
    "tbv_ar_init": (_I, [_I, ctypes.c_char_p, ctypes.c_char_p, _I, _SZ]),
    "tbv_ar_allreduce": (_I, [_VP, _VP, _SZ, _I, _VP]),
    "tbv_ar_stats": (None, [_PD, _PU]),
    "tbv_ar_stats4": (None, [_PD] * 4 + [_PU]),
    "tbv_ar_stats5": (None, [_PD] * 5 + [_PU]),
    "tbv_ar_cap": (_I, []), "tbv_ar_async": (_I, []), "tbv_ar_err": (_I, []),
    "tbv_ar_rails": (None, []), "tbv_ar_hist": (None, []), "tbv_ar_fini": (None, []),
    "tbv_emu_shutdown": (None, []),
    "tbv_emu_stage_peer": (_I, [_VP, _SZ]), "tbv_emu_stage_peer_repeat": (_I, [_VP, _SZ]), "tbv_emu_peer_resident": (_I, [_VP, _SZ]),
    "tbv_emu_arrival_script": (_I, [_PI, _SZ]), "tbv_emu_withhold": (_I, [_U64, _I]), "tbv_emu_hold_rail": (_I, [_I, _I]),
    "tbv_emu_seq": (_U64, []), "tbv_emu_plan": (_I, [_SZ, _PSZ, _PSZ]), "tbv_emu_configure": (_I, [ctypes.c_char_p, _SZ]),
    "tbv_emu_rendezvous": (_I, [_I, ctypes.c_char_p, _I, ctypes.c_double]),
    "tbv_emu_nslot": (_I, []), "tbv_emu_stride": (_SZ, []), "tbv_emu_send_slot": (_VP, [_I]), "tbv_emu_recv_slot": (_VP, [_I]),
    "tbv_emu_arrival_log": (_SZ, [_PU, _PI, _SZ]),
    "tbv_emu_latency_probe": (_I, [_I]), "tbv_emu_latencies": (_SZ, [_PD, _SZ]),
    "tbv_emu_kernel_timing": (_I, [_I]), "tbv_emu_kernel_times": (_SZ, [_I, _PD, _PD]),
    "tbv_emu_kernel_timeline": (_SZ, [_I, _PD, _PD, _SZ]),
    "tbv_emu_footprints": (None, [_PU]), "tbv_emu_tag_counts": (None, [_PU, _PU, _PU]),
    "tbv_ar_allreduce_chunked": (_I, [_VP, _VP, _SZ, _I, _VP]),
    "tbv_emu_run_pack": (_I, [_VP, _SZ, _I, _VP]), "tbv_emu_run_sum": (_I, [_VP, _VP, _VP, _SZ, _I, _VP]),
    "tbv_step_noalloc": (_I, [_VP, _VP, _VP, _VP, _I, _SZ, _I, _VP, _VP, _U64, _VP]),
    "tbv_emu_hbm_probe": (_I, [_I, _SZ, _SZ, _I, _PD, _PD]), "tbv_emu_launch_floor": (_I, [_I, _PD]),
    "tbv_emu_step_floor": (_I, [_SZ, _I, _PD]),
    "tbv_ar_allreduce_rmsnorm": (_I, [_VP, _VP, _VP, _VP, ctypes.c_float, _SZ, _SZ, _I, _VP]),
    "tbv_emu_run_sum_norm": (_I, [_I, _VP, _VP, _VP, _VP, _VP, ctypes.c_float, _SZ, _SZ, _I, _VP]),
    "tbv_step_quantize_i8": (_I, [ctypes.c_char_p, _VP]),
    "tbv_step_matmul_i8": (_I, [ctypes.c_char_p, _VP]), "tbv_step_rotary": (_I, [ctypes.c_char_p, _VP]),
    "tbv_emu_codec_image_bytes": (_SZ, [_SZ, _I]),
    "tbv_emu_run_quant": (_I, [_VP, _VP, _SZ, _I, _VP]), "tbv_emu_run_sum_quant": (_I, [_VP, _VP, _VP, _SZ, _I, _VP]),
}


def _bind(so):
    l = ctypes.CDLL(so)
    for name, (res, args) in _SIGNATURES.items():
        f = getattr(l, name)                   # AttributeError names the missing symbol
        f.restype, f.argtypes = res, args
    return l


def load(so=_DEFAULT_SO):
    """Load and bind the shared library without initialising it (no GPU needed)."""
    if not os.path.exists(so):
        raise RuntimeError(f"{so} is missing: build it with `make -C libtbvcoll_amd/csrc` "
                           "(there is no fallback path)")
    return _bind(so)


def init(rank, devs, peer_ip, port=18995, cap_bytes=8 << 20, so=_DEFAULT_SO):
    global _lib, _cap
    if _lib is not None:
        return
    l = load(so)
    rc = l.tbv_ar_init(rank, devs.encode(), (peer_ip or "").encode(), port, cap_bytes)
    if rc != 0:
        raise RuntimeError(f"tbv_ar_init failed rc={rc}")
    _lib, _cap = l, l.tbv_ar_cap()


def _call_args(t, out):
    """(in_ptr, out_ptr, nbytes, dtype code) of a tensor pair the library can take, or None: not initialised,
    not on the GPU, not contiguous, mismatched output, unsupported dtype (the guards of step4/tbvcoll.py:38-47)."""
    if _lib is None or not t.is_cuda or not t.is_contiguous():
        return None
    if out is not None and (not out.is_contiguous() or out.dtype is not t.dtype or out.numel() != t.numel()):
        return None
    code = _DT.get(t.dtype)
    if code is None:
        return None
    return _VP(t.data_ptr()), (_VP(out.data_ptr()) if out is not None else None), t.numel() * t.element_size(), code


def _stream():
    # read on every call: a cached handle goes stale when the caller switches streams
    return _VP(torch.cuda.current_stream().cuda_stream)


def all_reduce(t: torch.Tensor, out: torch.Tensor = None) -> bool:
    """SUM with the peer.  out=None means in place.  False means "not handled
    here, use your own collective" (step4/tbvcoll.py:35-58)."""
    a = _call_args(t, out)
    if a is None:
        return False
    pin, pout, nb, code = a
    if nb == 0:
        return True
    if nb > _cap:
        return False
    rc = _lib.tbv_ar_allreduce(pin, pout, nb, code, _stream())
    if rc == -2:
        return False
    if rc != 0:
        raise RuntimeError(f"tbv_ar_allreduce failed rc={rc}")
    return True


def is_async():
    return bool(_lib.tbv_ar_async())


def err():
    return bool(_lib.tbv_ar_err())


def rails():
    """Dump per-rail post / arrival averages to stderr (resets them)."""
    _lib.tbv_ar_rails()


def hist():
    """Dump the transfer histogram by size to stderr (resets it)."""
    _lib.tbv_ar_hist()


def raw_fn():
    """The bound C function for hot callers: (in_ptr, out_ptr, nbytes, dtype, stream) -> rc.
    The caller checks dtype, size and contiguity itself."""
    return _lib.tbv_ar_allreduce


def cap():
    return _cap


def _read_stats(fn, ndoubles):
    vals = [ctypes.c_double() for _ in range(ndoubles)]
    n = ctypes.c_ulonglong()
    fn(*[ctypes.byref(v) for v in vals], ctypes.byref(n))
    return tuple(v.value for v in vals) + (n.value,)


def stats5():
    """(pre, xfer, post, enq, drain, count), microseconds per call; reading resets."""
    return _read_stats(_lib.tbv_ar_stats5, 5)


def stats4():
    """(pre_us, xfer_us, post_us, enq_us, count)."""
    return _read_stats(_lib.tbv_ar_stats4, 4)


def stats3():
    pre, xf, post, _, n = stats4()
    return pre, xf, post, n


def stats():
    """(mean transfer us, calls); reading resets."""
    return _read_stats(_lib.tbv_ar_stats, 1)


# ------------------------------------------------------------------ emulated peer (additive)

def lib():
    """The bound library after `init` (None before)."""
    return _lib


def _nbytes(t):
    return t.numel() * t.element_size()


def _check(rc, what):
    if rc != 0:
        raise RuntimeError(f"{what} failed rc={rc}")


def stage_peer(t: torch.Tensor):
    """Queue `t` as the peer's payload of the next call that has none.  Keep `t`
    alive until that call's result is complete."""
    assert t.is_contiguous()
    _check(_lib.tbv_emu_stage_peer(_VP(t.data_ptr()), _nbytes(t)), "tbv_emu_stage_peer")


def stage_peer_repeat(t):
    if t is None:
        _lib.tbv_emu_stage_peer_repeat(None, 0)
    else:
        assert t.is_contiguous()
        _lib.tbv_emu_stage_peer_repeat(_VP(t.data_ptr()), _nbytes(t))


def peer_resident(t):
    _check(_lib.tbv_emu_peer_resident(None, 0) if t is None else _lib.tbv_emu_peer_resident(_VP(t.data_ptr()), _nbytes(t)),
           "tbv_emu_peer_resident")


def arrival_script(rails_list):
    n = len(rails_list)
    _check(_lib.tbv_emu_arrival_script((ctypes.c_int * max(n, 1))(*rails_list), n), "tbv_emu_arrival_script")


def withhold(seq, rail=0):
    _lib.tbv_emu_withhold(seq, rail)


def hold_rail(rail, hold=True):
    _check(_lib.tbv_emu_hold_rail(rail, 1 if hold else 0), "tbv_emu_hold_rail")


def seq():
    return _lib.tbv_emu_seq()


def latency_probe(on=True):
    _check(_lib.tbv_emu_latency_probe(1 if on else 0), "tbv_emu_latency_probe")


def latencies(max_n=1 << 20):
    buf = (ctypes.c_double * max_n)()
    n = _lib.tbv_emu_latencies(buf, max_n)
    return list(buf[:n])


def arrival_log(max_n=1 << 16):
    s = (ctypes.c_ulonglong * max_n)()
    r = (ctypes.c_int * max_n)()
    n = _lib.tbv_emu_arrival_log(s, r, max_n)
    return [(s[i], r[i]) for i in range(n)]


def kernel_timing(on=True):
    _lib.tbv_emu_kernel_timing(1 if on else 0)


def kernel_times(which):
    """(count, mean_us, min_us) of the recorded pack (0) or sum (1) launches; clears them."""
    m, mn = ctypes.c_double(), ctypes.c_double()
    n = _lib.tbv_emu_kernel_times(which, ctypes.byref(m), ctypes.byref(mn))
    return n, m.value, mn.value


def kernel_timeline(which, max_n=4096):
    """[(start_us, stop_us)] of the recorded launches, relative to the start of the first; keeps the samples."""
    a, b = (ctypes.c_double * max_n)(), (ctypes.c_double * max_n)()
    n = _lib.tbv_emu_kernel_timeline(which, a, b, max_n)
    return [(a[i], b[i]) for i in range(n)]


def hbm_probe(kind, nbytes, pool_bytes, reps, so=_DEFAULT_SO):
    """(mean_us, min_us) of a plain streaming kernel: kind 0 read, 1 write, 2 non-temporal copy, 3 plain copy."""
    l = _lib or load(so)
    m, mn = ctypes.c_double(), ctypes.c_double()
    _check(l.tbv_emu_hbm_probe(kind, nbytes, pool_bytes, reps, ctypes.byref(m), ctypes.byref(mn)), "tbv_emu_hbm_probe")
    return m.value, mn.value


def launch_floor(reps=2000, so=_DEFAULT_SO):
    """Launch-to-launch microseconds of an empty kernel in one stream."""
    l = _lib or load(so)
    v = ctypes.c_double()
    _check(l.tbv_emu_launch_floor(reps, ctypes.byref(v)), "tbv_emu_launch_floor")
    return v.value


def step_floor(nbytes, reps=480, so=_DEFAULT_SO):
    """Microseconds per launch of a kernel that only moves the four streams of one bf16 step of `nbytes`
    (no counting, no signal, no gate) over rotating cache-cold buffers: the floor under every form of the step."""
    l = _lib or load(so)
    v = ctypes.c_double()
    _check(l.tbv_emu_step_floor(nbytes, reps, ctypes.byref(v)), "tbv_emu_step_floor")
    return v.value


def footprints():
    """[wait entered, wait passed, pack started, sum done, wait timed out] sequence numbers (TBV_KWAIT=1)."""
    buf = (ctypes.c_ulonglong * 5)()
    _lib.tbv_emu_footprints(buf)
    return list(buf)


def tag_counts():
    a, b, c = (ctypes.c_ulonglong() for _ in range(3))
    _lib.tbv_emu_tag_counts(ctypes.byref(a), ctypes.byref(b), ctypes.byref(c))
    return a.value, b.value, c.value


def all_reduce_chunked(t: torch.Tensor, out: torch.Tensor = None) -> bool:
    """Pipelined SUM of a tensor of any size as cap-sized chunks."""
    a = _call_args(t, out)
    if a is None:
        return False
    pin, pout, nb, code = a
    _check(_lib.tbv_ar_allreduce_chunked(pin, pout, nb, code, _stream()), "tbv_ar_allreduce_chunked")
    return True


def all_reduce_rmsnorm(t: torch.Tensor, weight: torch.Tensor, eps: float, out: torch.Tensor = None, normed: torch.Tensor = None):
    """SUM with the peer fused with the RMSNorm of the result over the last dimension:
    out = t + peer (in place when out is None), normed = rmsnorm(out) * weight.  Returns `normed`
    (allocated when not given), or None when the library does not take the call (not initialised,
    unsupported layout, over the cap): the caller then runs its own all-reduce and norm."""
    a = _call_args(t, out)
    if a is None or t.dim() < 1 or weight.dtype is not t.dtype or not weight.is_contiguous() or weight.numel() != t.shape[-1]:
        return None
    pin, pout, nb, code = a
    if nb == 0 or nb > _cap:
        return None
    hidden = t.shape[-1]
    # what the row kernel takes: rows of whole 16-byte vectors, at most 64 KiB each, every buffer 16-byte aligned.
    # Anything else is declined here (the caller falls back) rather than turned into an error by the library.
    row_bytes = hidden * t.element_size()
    if row_bytes % 16 or row_bytes > 65536:
        return None
    if normed is not None and (not normed.is_contiguous() or normed.dtype is not t.dtype or normed.numel() != t.numel()):
        return None
    ptrs = [t.data_ptr(), weight.data_ptr()] + [x.data_ptr() for x in (out, normed) if x is not None]
    if any(p % 16 for p in ptrs):
        return None
    if normed is None:
        normed = torch.empty_like(t)
    rc = _lib.tbv_ar_allreduce_rmsnorm(pin, pout, _VP(normed.data_ptr()), _VP(weight.data_ptr()), eps,
                                       t.numel() // hidden, hidden, code, _stream())
    if rc == -2:
        return None
    _check(rc, "tbv_ar_allreduce_rmsnorm")
    return normed



# ------------------------------------------------------------------ the layer around the all-reduce (additive)
#
# These need no `init` and have nothing to fall back to: a call they cannot take raises ValueError.  They run on the
# current stream of the tensors' device and record no gradient.  They write through raw pointers, so they tell autograd
# which of the caller's tensors they wrote (`_wrote`: a backward pass that had saved one then raises, as after any other
# in-place operation).  A decode step makes hundreds of these calls, each on
# the GPU for a few microseconds, so they look at every attribute once and hand the library one packed structure.

_step_lib = None
_QUANTIZE = struct.Struct("3P5q")          # tbv_quantize_i8
_MATMUL = struct.Struct("6P9q")            # tbv_matmul_i8
_ROTARY = struct.Struct("2P7q2P7q2P10qf4x")  # tbv_rotary
_WIDE = {torch.int64: 1, torch.int32: 0}    # positions
_NO_HEADS = (0,) * 9
_wrote = torch._C._increment_version         # (of each tensor in a sequence; 0.4 us, the public wrapper 0.6)


def _steps():
    global _step_lib
    if _step_lib is None:
        _step_lib = _lib or load()
    return _step_lib


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _launch(fn, device, call):
    """Call a step function on the raw current stream of device `device` (an index), that device being current."""
    if device == torch._C._cuda_getDevice():
        rc = fn(call, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(call, torch._C._cuda_getCurrentRawStream(device))
    if rc != 0:
        raise RuntimeError(f"{fn.__name__} failed rc={rc}")


def _frozen():
    """A tensor, read or written, that requires a gradient: the kernels record none, so the call is for code that asks for none."""
    if torch.is_grad_enabled():
        raise ValueError("records no gradient: call it under torch.no_grad(), or in the forward and backward of a torch.autograd.Function")


def _no_tangent(*tensors):
    """The same for forward mode (called inside a dual level only): the kernels carry no tangent along.  In the forward of
    a torch.autograd.Function there is none to carry, its jvp does that."""
    for t in tensors:
        if t is not None and _forward.unpack_dual(t).tangent is not None:
            raise ValueError("carries no forward-mode gradient along: call it in the forward of a torch.autograd.Function that has a jvp")


def _rows(t, shape, what):
    """(rows, columns, row stride) of a tensor of this shape as a matrix of contiguous rows; leading dimensions are taken
    together where their rows are evenly spaced (part of the columns of a larger tensor)."""
    if len(shape) == 2:
        r, c = shape
        s, e = t.stride()
    elif shape:
        c, e = shape[-1], t.stride(-1)
        r, s = math.prod(shape[:-1]), c
        if len(shape) > 1 and r * c and not t.is_contiguous():
            s, n = c, 1                          # rows are s apart: every leading dimension has to step over the ones within it
            for size, step in zip(shape[-2::-1], t.stride()[-2::-1]):
                if size == 1:
                    continue
                if n == 1:
                    s = step
                elif step != s * n:
                    raise ValueError(what + ": the rows have to be evenly spaced")
                n *= size
    else:
        raise ValueError(what + " needs at least one dimension")
    if (e != 1 and c > 1) or (s < c and r > 1):
        raise ValueError(what + ": the last dimension has to be contiguous and rows must not overlap")
    return r, c, s if r > 1 else c


def quantize_int8(x: torch.Tensor, codes: torch.Tensor = None, scale: torch.Tensor = None):
    """Rows of `x` (last dimension; fp32, fp16 or bf16) as int8 codes with one fp32 scale a row:
    scale = max(f32(max|x| / 127), 2^-126), code = x / scale to the nearest integer, ties to even.  Returns
    (codes, scale) of shapes x.shape and x.shape[:-1], allocated when not given.  A row that holds an infinity or a
    NaN gets scale NaN and codes 0, so that every product with it is NaN."""
    code, dev, shape = _DT.get(x.dtype), x.get_device(), x.shape
    if code is None or dev < 0:
        raise ValueError("x has to be a fp32, fp16 or bf16 tensor on the GPU")
    if x.requires_grad:
        _frozen()
    if _forward._current_level >= 0:
        _no_tangent(x, scale)
    rows, cols, xs = _rows(x, shape, "x")
    given = () if codes is None else (codes,)
    if codes is None:
        codes = torch.empty_like(x, dtype=torch.int8) if x.is_contiguous() else x.new_empty(shape, dtype=torch.int8)
        cs = cols
    else:
        if codes.dtype is not torch.int8 or codes.shape != shape or codes.get_device() != dev:
            raise ValueError("codes has to be int8, of x's shape and device")
        cs = _rows(codes, shape, "codes")[2]
    if scale is None:
        scale = x.new_empty(shape[:-1], dtype=torch.float32)
    else:
        if scale.dtype is not torch.float32 or scale.shape != shape[:-1] or scale.get_device() != dev or not scale.is_contiguous():
            raise ValueError("scale has to be contiguous fp32, of x's shape without its last dimension, on its device")
        if scale.requires_grad:
            _frozen()
        given += (scale,)
    if rows:
        _launch((_step_lib or _steps()).tbv_step_quantize_i8, dev, _QUANTIZE.pack(codes.data_ptr(), scale.data_ptr(), x.data_ptr(), cs, xs, rows, cols, code))
        if given:
            _wrote(given)
    return codes, scale


def matmul_int8(x: torch.Tensor, x_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor = None,
                out: torch.Tensor = None, dtype: torch.dtype = torch.bfloat16):
    """x [..., k] int8 times w [n, k] int8 (a linear layer's weight as stored), a scale for each token and each channel:
    out = dtype(float(sum) * x_scale * w_scale + bias), the sum exact in int32.  x_scale: fp32, one per row of x (any
    shape of that many elements) or a single one; w_scale: fp32, n or one; bias: n elements of the result's type.
    Returns `out` [..., n] (its type counts when given).  k up to 131071; fastest where k and the row strides are
    multiples of 16 and the tensors 16-byte aligned."""
    dev, shape, channels = x.get_device(), x.shape, w.shape
    if dev < 0 or x.dtype is not torch.int8 or w.dtype is not torch.int8 or w.get_device() != dev or len(channels) != 2:
        raise ValueError("x and w have to be int8 on one GPU, w a matrix")
    m, k, xs = _rows(x, shape, "x")
    n, wk, ws = _rows(w, channels, "w")
    if k != wk or k > 131071:
        raise ValueError(f"x has rows of {k} and w of {wk}: they have to be equal, and at most 131071 (beyond, the int32 sum can overflow)")
    if x_scale.requires_grad or w_scale.requires_grad or (bias is not None and bias.requires_grad):
        _frozen()
    if _forward._current_level >= 0:
        _no_tangent(x_scale, w_scale, bias, out)
    sx, sw = x_scale.numel(), w_scale.numel()
    if x_scale.dtype is not torch.float32 or x_scale.get_device() != dev or not x_scale.is_contiguous() or (sx != m and sx != 1):
        raise ValueError("x_scale has to be contiguous fp32 on x's device, one for each row of x or one for all")
    if w_scale.dtype is not torch.float32 or w_scale.get_device() != dev or not w_scale.is_contiguous() or (sw != n and sw != 1):
        raise ValueError("w_scale has to be contiguous fp32 on x's device, one for each row of w or one for all")
    if out is None:
        code, os_ = _DT.get(dtype), n
        if code is None:
            raise ValueError("the result is fp32, fp16 or bf16")
        given = False
        out = x_scale.new_empty((m, n) if len(shape) == 2 else shape[:-1] + (n,), dtype=dtype)
    else:
        dtype, given = out.dtype, True
        code = _DT.get(dtype)
        if code is None:
            raise ValueError("the result is fp32, fp16 or bf16")
        wide = shape[:-1] + (n,)
        if out.get_device() != dev or out.shape != wide:
            raise ValueError("out has to be on x's device, of x's shape with n columns")
        if out.requires_grad:
            _frozen()
        os_ = _rows(out, wide, "out")[2]
    if bias is None:
        b = 0
    else:
        if bias.dtype is not dtype or bias.get_device() != dev or not bias.is_contiguous() or bias.numel() != n:
            raise ValueError("bias has to be n contiguous elements of the result's type on x's device")
        b = bias.data_ptr()
    if m and n:
        _launch((_step_lib or _steps()).tbv_step_matmul_i8, dev, _MATMUL.pack(
            out.data_ptr(), x.data_ptr(), x_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), b, os_, xs, ws, m, n, k, sx, sw, code))
        if given:
            _wrote((out,))
    return out


def linear_int8_all_reduce(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor, bias: torch.Tensor = None, out: torch.Tensor = None):
    """The row-parallel linear layer of a tensor-parallel pair with int8 weights: this rank's columns of the activations
    `x` (fp32, fp16 or bf16) as int8 rows, times this rank's columns of the weight, SUM with the peer's partial result
    (bias: on one rank only).  Returns the sum in x's type, or None when the library does not take the all-reduce (not
    initialised, over the cap): `out` is then as it was, and the caller runs its own layer.  Tensors that no call could
    take are refused whether the library takes the all-reduce or not."""
    dev = x.get_device()
    _need(dev >= 0 and x.dim() >= 1 and x.dtype in _DT, "x has to be a fp32, fp16 or bf16 tensor on the GPU")
    _need(w.dim() == 2 and w.dtype is torch.int8 and w.get_device() == dev and w.shape[1] == x.shape[-1],
          "w has to be an int8 matrix on x's device with as many columns as x")
    n = w.shape[0]
    _need(out is None or (out.dtype is x.dtype and out.get_device() == dev and out.shape == x.shape[:-1] + (n,) and out.is_contiguous()),
          "out has to be contiguous, of x's type and device and of x's shape with a column for each row of w")
    # (all that makes `all_reduce` decline is decided here, before anything is written)
    if _lib is None or math.prod(x.shape[:-1]) * n * x.element_size() > _cap:
        return None
    if dev != torch._C._cuda_getDevice():        # `all_reduce` takes the current device's stream: it has to be the product's
        with torch.cuda.device(dev):
            return linear_int8_all_reduce(x, w, w_scale, bias=bias, out=out)
    codes, scale = quantize_int8(x)
    out = matmul_int8(codes, scale, w, w_scale, bias=bias, out=out, dtype=x.dtype)
    return out if all_reduce(out) else None


def rotary_frequencies(rot: int, base: float = 10000.0, factor: float = 1.0, method: str = "linear", context: int = 0,
                       low: float = 1.0, high: float = 32.0, device="cuda"):
    """(freqs, scale) for `rotary`: freqs[i] = base^(-2i/rot), fp64, rot/2 of them, stretched by `factor` for contexts
    longer than the `context` positions a model was trained on:

      "linear"   every frequency divided by factor (positions interpolated);
      "base"     the base raised to base * factor^(rot / (rot - 2)): the slowest frequency is divided by factor, the
                 fastest kept;
      "bands"    a frequency that turns at least `high` times within `context` is kept, one that turns at most `low`
                 times is divided by factor, in between the two are mixed linearly in the number of turns;
      "ramp"     as "bands", but mixed linearly in the frequency's index between the indices that turn `high` and `low`
                 times (rounded outwards), and scale = 0.1 ln(factor) + 1 for the longer softmax.

    scale is 1 except for "ramp"."""
    _need(rot >= 2 and rot % 2 == 0, "rot has to be even and at least 2")
    _need(base > 1.0 and factor >= 1.0, "base has to be above 1 and factor at least 1")
    i = torch.arange(rot // 2, dtype=torch.float64)
    scale = 1.0
    if method == "base":
        if rot > 2:
            base = base * factor ** (rot / (rot - 2))
        freqs = base ** (-2.0 * i / rot)
    else:
        freqs = base ** (-2.0 * i / rot)
        if method == "linear":
            freqs = freqs / factor
        elif method in ("bands", "ramp"):
            _need(context > 0 and 0 < low < high, "bands and ramp need the trained context and 0 < low < high")
            if method == "bands":
                keep = ((context * freqs / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
            else:
                def index(turns):
                    return rot * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(base))
                first, last = max(math.floor(index(high)), 0), min(math.ceil(index(low)), rot - 1)
                keep = 1 - ((i - first) / max(last - first, 1e-3)).clamp(0, 1)
                scale = 0.1 * math.log(factor) + 1.0
            freqs = freqs * keep + freqs / factor * (1 - keep)
        else:
            raise ValueError(f"unknown method {method!r}: linear, base, bands or ramp")
    return freqs.to(device), scale


def _heads(t, shape, o, dtype, dev, what):
    """The nine fields of tbv_rotary_heads for t ([tokens, heads, head] or [batch, tokens, heads, head], of this type and
    device) turned into o."""
    s = t.stride()
    if o is None or o is t:
        at = to = t.data_ptr()
        u = s
    else:
        if o.dtype is not dtype or o.get_device() != dev or o.shape != shape:
            raise ValueError(what + "_out has to be of its input's type, device and shape")
        if o.requires_grad:
            _frozen()
        u, at, to = o.stride(), t.data_ptr(), o.data_ptr()
    if (s[-1] != 1 or u[-1] != 1) and shape[-1] > 1:
        raise ValueError(what + ": the elements of a head have to be contiguous")
    if len(s) == 3:
        return to, at, shape[1], 0, s[0], s[1], 0, u[0], u[1]
    return to, at, shape[2], s[0], s[1], s[2], u[0], u[1], u[2]


def rotary(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, scale: float = 1.0,
           interleaved: bool = False, inverse: bool = False, q_out: torch.Tensor = None, k_out: torch.Tensor = None):
    """Turn the heads of q and k (k may be None) by their positions, in place where no output is given.

    q, k: [tokens, heads, head] or [batch, tokens, heads, head] of one type (fp32, fp16, bf16), any strides (views of a
    packed projection, heads before tokens) with contiguous heads.  positions: int64 or int32, [tokens] or
    [batch, tokens].  freqs: fp64, rot/2 of them (`rotary_frequencies`): the first rot elements of a head turn, the rest
    is copied.  Pairs are (i, i + rot/2), or (2i, 2i + 1) with `interleaved`; cos and sin are multiplied by `scale`.
    `inverse` turns back: with the outputs' gradients for q and k it is the backward pass.  Returns (q_out, k_out)."""
    dev, shape, dtype = q.get_device(), q.shape, q.dtype
    d, code = len(shape), _DT.get(dtype)
    if dev < 0 or code is None or (d != 3 and d != 4):
        raise ValueError("q has to be fp32, fp16 or bf16 on the GPU, [tokens, heads, head] or [batch, tokens, heads, head]")
    if q.requires_grad or (k is not None and k.requires_grad):
        _frozen()
    if _forward._current_level >= 0:
        _no_tangent(q, k, freqs, q_out, k_out)
    batch, tokens, head = 1 if d == 3 else shape[0], shape[-3], shape[-1]
    hq = _heads(q, shape, q_out, dtype, dev, "q")
    if k is None:
        if k_out is not None:
            raise ValueError("k_out without k")
        hk = _NO_HEADS
    else:
        ks = k.shape
        if k.dtype is not dtype or k.get_device() != dev or len(ks) != d or ks[0] != shape[0] or ks[-3] != tokens or ks[-1] != head:
            raise ValueError("k has to be of q's type and device and differ in its heads only")
        hk = _heads(k, ks, k_out, dtype, dev, "k")
    wide, ps = _WIDE.get(positions.dtype), positions.shape
    if positions.get_device() != dev or wide is None:
        raise ValueError("positions have to be int64 or int32 on q's device")
    if len(ps) == 1 and ps[0] == tokens:
        p0, p1 = 0, positions.stride(0)
    elif d == 4 and ps == shape[:2]:
        p0, p1 = positions.stride()
    else:
        raise ValueError("positions have to be [tokens] or [batch, tokens]")
    rot = 2 * freqs.numel()
    if freqs.dtype is not torch.float64 or freqs.get_device() != dev or freqs.dim() != 1 or not freqs.is_contiguous() or rot > head or rot > 8192:
        raise ValueError("freqs has to be contiguous fp64 on q's device, at most half a head and 4096 long")
    if freqs.requires_grad:
        _frozen()
    _launch((_step_lib or _steps()).tbv_step_rotary, dev, _ROTARY.pack(
        *hq, *hk, positions.data_ptr(), freqs.data_ptr(), p0, p1, batch, tokens, head, rot, code, wide, interleaved, inverse, scale))
    if q_out is None:
        q_out = q
    if k is None:
        _wrote((q_out,))
        return q_out, None
    if k_out is None:
        k_out = k
    _wrote((q_out, k_out))
    return q_out, k_out


def shutdown():
    """Tear the library down so that `init` can run again with other settings."""
    global _lib, _cap
    if _lib is not None:
        _lib.tbv_emu_shutdown()
    _lib, _cap = None, 0
