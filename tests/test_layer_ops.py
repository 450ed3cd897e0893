"""The operators of the layer around the all-reduce: int8 rows, the scaled int8 product, rotary positions.

Each is compared with its definition in 64 bits.  Tolerances, derived from the operators' arithmetic (u = 2^-24 is half a
step of fp32, relative; h = finfo(T).eps / 2 half a step of the result's type):

  codes and scales   none: the scale is one correctly rounded division, the code is decided exactly.
  product            the int32 sum is exact; its conversion and the two multiplications are off by u each, the bias'
                     addition by u of the result, the rounding to T by h of it (or half the least subnormal).
  rotary             the angle's fraction of a turn is formed in fp64 (error below 1e-9 rad for angles to 2^22) and rounded
                     to fp32: at most pi u rad; cos and sin are within 2 ulp (4 u); times `scale` 1 u; each product 1 u and
                     their sum 1 u of at most |x1| + |x2|: (pi + 4 + 1 + 2) u scale (|x1| + |x2|) < 10.2 u ..., then h.
"""
import itertools
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from gpu_util import dev, say, session
from libtbvcoll_amd import synth, tbvcoll

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
U = 2.0 ** -24
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu


def half(dt):
    return torch.finfo(dt).eps / 2


# ------------------------------------------------------------------ definitions in 64 bits (CPU)

def want_rows(x):
    """(codes, scale) of the definition; the code by comparing the remainder with half a scale, exact in fp64: the scale
    has 24 bits and the code at most 8, so every product and difference below is exact."""
    x = x.cpu().double()
    top = x.abs().amax(-1) if x.shape[-1] else torch.zeros(x.shape[:-1], dtype=torch.float64)
    bad = ~torch.isfinite(x).all(-1)
    scale = (top / 127).float().clamp_min(2.0 ** -126)
    s = scale.double().unsqueeze(-1)
    low = torch.floor(x / s)
    low = torch.where(low * s > x, low - 1, low)
    rest = x - low * s
    up = (2 * rest > s) | ((2 * rest == s) & (low % 2 != 0))
    codes = torch.where(bad.unsqueeze(-1), torch.zeros_like(low), low + up)
    return codes.to(torch.int8), torch.where(bad, torch.full_like(scale, float("nan")), scale)


def want_product(x, xs, w, ws, bias):
    """(result, tolerance before the rounding to T) of the definition."""
    total = x.cpu().double() @ w.cpu().double().t()
    p = total * xs.cpu().double().reshape(-1, 1) * ws.cpu().double().reshape(1, -1)
    r = p if bias is None else p + bias.cpu().double()
    return r, 3.01 * U * p.abs() + 1.01 * U * r.abs()


def check(got, want, before, dt, what):
    got = got.cpu().double()
    assert got.shape == want.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    tol = before + (0 if dt == torch.float32 else 1) * half(dt) * (want.abs() + before) + LEAST[dt]
    off = (got - want).abs()
    over = off > tol
    over &= ~(torch.isinf(want) & (got == want))
    over |= torch.isinf(got) & (want.abs() + tol < torch.finfo(dt).max)
    assert not bool(over.any()), (what, int(over.sum()), torch.nonzero(over)[:3].tolist(), float(torch.nan_to_num(off).max()))


def want_rotary(x, positions, freqs, scale, interleaved, inverse):
    """(result, tolerance before the rounding) for x [batch, tokens, heads, head]; positions [batch, tokens]."""
    x, positions, freqs = x.cpu().double(), positions.cpu().double(), freqs.cpu().double()
    half_ = freqs.shape[0]
    a = positions[..., None] * freqs
    c, s = (a.cos() * scale)[:, :, None], (a.sin() * scale)[:, :, None] * (-1 if inverse else 1)
    y, tol = x.clone(), torch.zeros_like(x)
    one = slice(0, 2 * half_, 2) if interleaved else slice(0, half_)
    two = slice(1, 2 * half_, 2) if interleaved else slice(half_, 2 * half_)
    x1, x2 = x[..., one], x[..., two]
    y[..., one], y[..., two] = x1 * c - x2 * s, x2 * c + x1 * s
    tol[..., one] = tol[..., two] = 10.2 * U * abs(scale) * (x1.abs() + x2.abs())
    return y, tol


def codes_of(seed, *shape):
    n = int(np.prod(shape))
    return torch.from_numpy((synth.bits32(seed, n) % np.uint64(255)).astype(np.int64) - 127).to(torch.int8).reshape(shape)


def scales_of(seed, n, size=0.01):
    return torch.from_numpy(synth.uniform(seed, n, 0.5 * size, 1.5 * size))


# ------------------------------------------------------------------ on the CPU: refusals, frequencies, the definition itself

def test_definition_of_the_codes_on_hand_made_rows():
    # scale 2^-3 exactly: ties go to even, the largest element to 127
    x = torch.tensor([[127 / 8, 0.5 / 8, 1.5 / 8, 2.5 / 8, -0.5 / 8, -1.5 / 8, -127 / 8, 0.0]])
    codes, scale = want_rows(x)
    assert scale.tolist() == [0.125] and codes.tolist() == [[127, 0, 2, 2, 0, -2, -127, 0]]
    codes, scale = want_rows(torch.tensor([[0.0, 0.0], [float("inf"), 1.0], [float("nan"), 1.0], [1e-45, 0.0]]))
    assert codes.tolist() == [[0, 0]] * 4 and scale[0] == 2.0 ** -126 and torch.isnan(scale[1:3]).all() and scale[3] == 2.0 ** -126


def test_rotary_frequencies():
    f, s = tbvcoll.rotary_frequencies(8, device="cpu")
    assert f.dtype == torch.float64 and s == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    f4, _ = tbvcoll.rotary_frequencies(8, factor=4.0, device="cpu")
    assert torch.equal(f4, f / 4)
    b, _ = tbvcoll.rotary_frequencies(8, factor=4.0, method="base", device="cpu")
    assert abs(float(b[0]) - 1) < 1e-15 and abs(float(b[-1] / (f[-1] / 4)) - 1) < 1e-12    # fastest kept, slowest divided by factor
    plain, _ = tbvcoll.rotary_frequencies(128, base=5e5, device="cpu")
    turns = 8192 * plain / (2 * np.pi)
    d, s = tbvcoll.rotary_frequencies(128, base=5e5, factor=8.0, method="bands", context=8192, low=1.0, high=4.0, device="cpu")
    assert s == 1.0 and torch.equal(d[turns >= 4], plain[turns >= 4]) and torch.allclose(d[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (d[mid] < plain[mid]).all() and (d[mid] > plain[mid] / 8).all()
    r, s = tbvcoll.rotary_frequencies(128, factor=8.0, method="ramp", context=4096, device="cpu")
    base, _ = tbvcoll.rotary_frequencies(128, device="cpu")
    assert abs(s - (0.1 * np.log(8.0) + 1)) < 1e-15 and r[0] == base[0] and abs(float(r[-1] / base[-1]) - 1 / 8) < 1e-12
    assert (r[1:] < r[:-1]).all() and (r <= base * (1 + 1e-15)).all() and (r >= base / 8 * (1 - 1e-15)).all()
    assert tbvcoll.rotary_frequencies(2, factor=2.0, method="base", device="cpu")[0].tolist() == [1.0]
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, base=1.0), dict(rot=8, factor=0.5), dict(rot=8, method="other"),
                dict(rot=8, method="bands"), dict(rot=8, method="ramp", context=16, low=4.0, high=2.0)):
        with pytest.raises(ValueError):
            tbvcoll.rotary_frequencies(device="cpu", **bad)


def test_tensors_on_the_cpu_are_refused():
    x8, s, x = torch.zeros(2, 16, dtype=torch.int8), torch.ones(2), torch.zeros(2, 16)
    with pytest.raises(ValueError):
        tbvcoll.quantize_int8(x)
    with pytest.raises(ValueError):
        tbvcoll.matmul_int8(x8, s, x8, s)
    with pytest.raises(ValueError):
        tbvcoll.rotary(torch.zeros(2, 1, 8), None, torch.arange(2), torch.ones(4, dtype=torch.float64))
    with pytest.raises(ValueError):
        tbvcoll.linear_int8_all_reduce(x, x8, s)


# (call by call: what the C entries refuse before any launch; the pointers are never followed)
P = 1 << 20


def quant(**kw):
    a = dict(codes=P, scale=2 * P, x=3 * P, code_stride=64, x_stride=64, rows=4, hidden=64, dtype=2) | kw
    return tbvcoll.load().tbv_step_quantize_i8(tbvcoll._QUANTIZE.pack(*a.values()), None)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(codes=0), dict(scale=0), dict(x=0), dict(x=3 * P + 1), dict(rows=-1), dict(hidden=-1),
                                dict(scale=2 * P + 2), dict(code_stride=63), dict(x_stride=63), dict(rows=1 << 31),
                                dict(hidden=1 << 31), dict(codes=3 * P + 8), dict(scale=3 * P + 500), dict(scale=P + 16)])
def test_refused_quantize_calls(kw, capfd):
    assert quant(**kw) == -1
    assert "[tbvcoll] int8 rows:" in capfd.readouterr().err


MAT = dict(out=P, x=2 * P, x_scale=3 * P, w=4 * P, w_scale=5 * P, bias=6 * P, out_stride=32, x_stride=64, w_stride=64,
           m=16, n=32, k=64, x_scales=16, w_scales=32, dtype=2)


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(dtype=-1), dict(out=0), dict(x=0), dict(x_scale=0), dict(w=0), dict(w_scale=0),
                                dict(m=-1), dict(n=-1), dict(k=-1), dict(k=131072, x_stride=1 << 20, w_stride=1 << 20), dict(m=1 << 31),
                                dict(x_scales=15), dict(w_scales=33), dict(out_stride=31), dict(x_stride=63), dict(w_stride=63),
                                dict(out=P + 1), dict(bias=6 * P + 1), dict(x_scale=3 * P + 2), dict(w_scale=5 * P + 1),
                                dict(out=2 * P + 16), dict(out=4 * P - 16), dict(out=3 * P + 60), dict(out=5 * P), dict(out=6 * P + 62),
                                dict(x_stride=1 << 41), dict(m=0x7fffffff, n=0x7fffffff, x_scales=1, w_scales=1, out_stride=0x7fffffff)])
def test_refused_matmul_calls(kw, capfd):
    a = MAT | kw
    assert tbvcoll.load().tbv_step_matmul_i8(tbvcoll._MATMUL.pack(*a.values()), None) == -1
    assert "[tbvcoll] int8 product:" in capfd.readouterr().err


def test_empty_calls_launch_nothing():
    lib = tbvcoll.load()
    assert quant(rows=0) == 0
    for kw in (dict(m=0), dict(n=0)):
        assert lib.tbv_step_matmul_i8(tbvcoll._MATMUL.pack(*(MAT | kw).values()), None) == 0
    assert lib.tbv_step_matmul_i8(None, None) == -1 and lib.tbv_step_quantize_i8(None, None) == -1 and lib.tbv_step_rotary(None, None) == -1


HEADS = ("out", "in", "heads", "in_batch", "in_token", "in_head", "out_batch", "out_token", "out_head")


def rot_call(q=(), k=(), **kw):
    """tbv_step_rotary with 2 x 8 tokens, 4 + 2 heads of 64 fp16, dense and apart unless said otherwise."""
    dq = dict(zip(HEADS, (P, 2 * P, 4, 8 * 256, 256, 64, 8 * 256, 256, 64))) | dict(q)
    dk = dict(zip(HEADS, (3 * P, 4 * P, 2, 8 * 128, 128, 64, 8 * 128, 128, 64))) | dict(k)
    a = dict(positions=5 * P, freqs=6 * P, pos_batch=8, pos_token=1, batch=2, tokens=8, head=64, rot=64, dtype=1, pos64=1,
             interleaved=0, inverse=0, scale=1.0) | kw
    return tbvcoll.load().tbv_step_rotary(tbvcoll._ROTARY.pack(*dq.values(), *dk.values(), *a.values()), None)


PACKED = dict(in_batch=8 * 512, in_token=512, in_head=64, out_batch=8 * 512, out_token=512, out_head=64)


@pytest.mark.parametrize("q,k,kw", [
    ({}, {}, dict(dtype=3)), ({}, {}, dict(batch=-1)), ({}, {}, dict(tokens=-1)), ({}, {}, dict(rot=63)), ({}, {}, dict(rot=66)), ({}, {}, dict(rot=8194, head=8194, batch=1, tokens=1)),
    ({}, {}, dict(rot=-2)), ({}, {}, dict(head=-1)), ({}, {}, dict(head=1 << 21)), ({}, {}, dict(positions=0)), ({}, {}, dict(freqs=0)),
    ({}, {}, dict(freqs=6 * P + 4)), ({}, {}, dict(positions=5 * P + 4)), ({}, {}, dict(batch=1 << 20, tokens=1 << 20)),
    (dict(heads=-1), {}, {}), (dict(out=0), {}, {}), ({"in": 0}, {}, {}), (dict(out=P + 1), {}, {}), ({}, {"in": 4 * P + 1}, {}),
    (dict(out_head=32), {}, {}),                                        # heads of the output share elements
    (dict(out_token=0), {}, {}), (dict(in_token=1 << 57), {}, {}),
    (dict(out=2 * P + 128), {}, {}),                                    # shifted by a head: neither apart nor in place
    (dict(out=2 * P, out_token=512, out_batch=4096), {}, {}),           # same start, other strides
    (dict(out=4 * P), {}, {}), ({}, dict(out=2 * P + 64), {}),          # an output on the other input
    (dict(out=3 * P), {}, {}),                                          # both outputs at one place
    (dict(PACKED, out=P, **{"in": P}), dict(PACKED, out=P + 3 * 128, **{"in": P + 3 * 128}), {}),   # packed views that share a head
    (dict(PACKED, out=P, **{"in": P}), dict(PACKED, out=P + 7 * 128, **{"in": P + 7 * 128}), {}),   # k's second head is the next token's q
])
def test_refused_rotary_calls(q, k, kw, capfd):
    assert rot_call(q, k, **kw) == -1
    assert "[tbvcoll] rotary:" in capfd.readouterr().err


@pytest.mark.parametrize("kw", [dict(positions=P), dict(positions=P + 8 * 256 * 4 - 8), dict(positions=3 * P - 8), dict(freqs=3 * P + 8), dict(freqs=P - 248),
                                dict(positions=P + 16384, pos_batch=-8), dict(pos_token=1 << 55), dict(pos_batch=-(1 << 57))])
def test_rotary_outputs_stay_off_positions_and_freqs(kw, capfd):
    assert rot_call(**kw) == -1
    assert "[tbvcoll] rotary:" in capfd.readouterr().err


def test_empty_rotary_calls_launch_nothing():
    assert rot_call(batch=0) == 0 and rot_call(tokens=0) == 0 and rot_call(head=0, rot=0) == 0
    assert rot_call(dict(heads=0, out=0), dict(heads=0, out=0)) == 0


# ------------------------------------------------------------------ int8 rows

@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 17), (8, 4096), (7, 1000), (65, 64), (5, 9472), (2, 16384), (3, 32776),
                                       (2, 100003), (2047, 520), (1, 16), (300, 8), (9, 4104)])
def test_rows_match_the_definition(name, rows, cols):
    x = dev(synth.normal(rows * 7 + cols, rows * cols, 0.02), DT[name]).view(rows, cols)
    x[:, cols // 2] = 8.0 if rows % 2 else -8.0
    say("quantize", name, rows, cols)
    codes, scale = tbvcoll.quantize_int8(x)
    c, s = want_rows(x)
    assert torch.equal(scale.cpu(), s) and torch.equal(codes.cpu(), c)


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("cols,stride,offset", [(64, 80, 0), (64, 64, 1), (61, 67, 3), (4096, 4099, 0), (4096, 4112, 8), (5000, 5008, 5)])
def test_rows_with_strides_and_offsets(name, cols, stride, offset):
    rows = 5
    x = dev(synth.normal(cols, rows * stride + 16), DT[name])[offset:offset + rows * stride].view(rows, stride)[:, :cols]
    store = torch.full((rows, stride + 5), 77, dtype=torch.int8, device="cuda")
    codes, scale = tbvcoll.quantize_int8(x, codes=store[:, 1:1 + cols])
    c, s = want_rows(x)
    assert torch.equal(scale.cpu(), s) and torch.equal(codes.cpu(), c)
    assert bool((store[:, 0] == 77).all()) and bool((store[:, 1 + cols:] == 77).all())       # nothing outside the rows


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("cols", [40, 4096, 20000])
def test_rows_special_values(name, cols):
    dt = DT[name]
    big, tiny = torch.finfo(dt).max, torch.finfo(dt).tiny
    base = torch.from_numpy(synth.uniform(3, cols, -1, 1))
    ties = (torch.arange(cols) % 253 - 126).float() / 2                          # scale 1/2: codes and ties of it
    ties[7] = 63.5
    rows = [torch.zeros(cols), base, ties, base * tiny, torch.full((cols,), tiny / 64), base.sign() * big, base.clone(), base.clone(), base.clone(),
            -torch.ones(cols), torch.zeros(cols)]
    rows[6][cols - 1], rows[7][3], rows[8][cols // 2] = float("inf"), float("-inf"), float("nan")
    rows[10][cols - 1] = -tiny / 4
    x = torch.stack(rows).to(dt).cuda()
    codes, scale = tbvcoll.quantize_int8(x)
    c, s = want_rows(x)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(s)) and torch.equal(torch.nan_to_num(scale.cpu()), torch.nan_to_num(s))
    assert torch.equal(codes.cpu(), c)


@gpu
def test_rows_of_any_shape_and_none():
    x = dev(synth.normal(1, 2 * 3 * 64), torch.bfloat16).view(2, 3, 64)
    codes, scale = tbvcoll.quantize_int8(x)
    assert codes.shape == (2, 3, 64) and scale.shape == (2, 3)
    c1, s1 = tbvcoll.quantize_int8(x[1, 2])
    assert s1.shape == () and torch.equal(c1, codes[1, 2]) and torch.equal(s1, scale[1, 2])
    codes, scale = tbvcoll.quantize_int8(torch.empty(0, 64, device="cuda"))
    assert codes.shape == (0, 64) and scale.shape == (0,)
    codes, scale = tbvcoll.quantize_int8(torch.empty(3, 0, device="cuda"))
    assert codes.shape == (3, 0) and scale.tolist() == [2.0 ** -126] * 3


@gpu
def test_rows_refusals():
    x = torch.zeros(4, 64, device="cuda")
    for bad in (dict(x=x.double()), dict(x=x.t()), dict(x=x[:, None].expand(4, 2, 64)), dict(x=x, codes=torch.empty(4, 63, dtype=torch.int8, device="cuda")),
                dict(x=x, codes=torch.empty(4, 64, device="cuda")), dict(x=x, scale=torch.empty(5, device="cuda")),
                dict(x=x, scale=torch.empty(8, device="cuda")[::2]), dict(x=x[0].expand(4, 64)), dict(x=x.cpu()),
                dict(x=torch.zeros((), device="cuda"))):
        with pytest.raises(ValueError):
            tbvcoll.quantize_int8(**bad)


# ------------------------------------------------------------------ the int8 product

SHAPES = [(1, 1, 1), (1, 4096, 4096), (2, 16, 16), (3, 5, 7), (4, 1000, 512), (7, 33, 4096), (8, 2560, 1024), (16, 64, 64), (17, 129, 272),
          (31, 2048, 528), (32, 31, 16), (33, 4096, 96), (48, 300, 4112), (63, 65, 63), (64, 64, 128), (65, 80, 131), (77, 2741, 1111), (100, 16, 9472),
          (128, 128, 128), (129, 1024, 2048), (200, 136, 48), (256, 256, 256), (257, 511, 400), (300, 640, 4096), (333, 1040, 8192), (512, 2048, 144),
          (600, 72, 1000), (1000, 1024, 1040), (1025, 2049, 640), (2048, 1536, 512), (2049, 768, 320), (64, 4096, 131071), (5, 8, 131056)]


@gpu
@pytest.mark.parametrize("m,n,k", SHAPES, ids=lambda v: str(v))
def test_product_matches_the_definition(m, n, k):
    name = list(DT)[(m + n + k) % 3]
    dt = DT[name]
    x, w = codes_of(m + k, m, k), codes_of(n + 3 * k, n, k)
    xs, ws = scales_of(1, m), scales_of(2, n, 0.0005)
    bias = torch.from_numpy(synth.normal(3, n)).to(dt) if (m + n) % 2 else None
    say("product", m, n, k, name, "bias" if bias is not None else "")
    got = tbvcoll.matmul_int8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), bias=None if bias is None else bias.cuda(), dtype=dt)
    want, before = want_product(x, xs, w, ws, bias)
    check(got, want, before, dt, (m, n, k, name))


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("m", [1, 5, 16, 40, 100, 300, 1100])
@pytest.mark.parametrize("pads", [(0, 0, 0), (16, 16, 16), (0, 0, 1), (32, 48, 8), (1, 0, 0), (0, 3, 3)])
def test_product_with_strides_and_guards(name, m, pads):
    """Row strides beyond the row, offsets, an output inside a larger buffer whose rest stays as it was."""
    n, k, dt = 200, 224, DT[name]
    px, pw, po = pads
    x = codes_of(1, m + 1, k + px).cuda()[1:, px // 2:px // 2 + k]
    w = codes_of(2, n + 1, k + pw).cuda()[:n, pw // 2:pw // 2 + k]
    xs, ws = scales_of(3, m), scales_of(4, n)
    store = torch.full((m + 2, n + 2 * po), 5.0, dtype=dt, device="cuda")
    out = store[1:m + 1, po:po + n]
    got = tbvcoll.matmul_int8(x, xs.cuda(), w, ws.cuda(), out=out)
    assert got is out
    want, before = want_product(x, xs, w, ws, None)
    check(out, want, before, dt, (m, pads, name))
    rest = torch.ones_like(store, dtype=torch.bool)
    rest[1:m + 1, po:po + n] = False
    assert bool((store[rest] == 5.0).all())


@gpu
@pytest.mark.parametrize("m", [1, 30, 70, 256])
def test_product_extremes(m):
    """Largest codes at the largest k, one scale for all, infinite and NaN scales, k = 0, a result beyond fp16."""
    n, k = 48, 131071
    x = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    w = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    one, few = torch.ones(1, device="cuda"), torch.full((1,), 2.0 ** -20, device="cuda")
    got = tbvcoll.matmul_int8(x, one, w, few, dtype=torch.float32)
    assert bool((got == float(np.float32(131071 * 16384)) * 2.0 ** -20).all())
    x, w = codes_of(5, m, 64).cuda(), codes_of(6, n, 64).cuda()
    xs, ws = scales_of(7, m).cuda(), scales_of(8, n).cuda()
    xs[0], ws[3] = float("nan"), float("inf")
    got = tbvcoll.matmul_int8(x, xs, w, ws, dtype=torch.bfloat16).cpu()
    want, before = want_product(x, xs, w, ws, None)
    check(got, want, torch.nan_to_num(before, posinf=0.0), torch.bfloat16, m)
    assert torch.isnan(got[0]).all()
    bias = torch.arange(n, dtype=torch.float16, device="cuda")
    got = tbvcoll.matmul_int8(x[:, :0], xs[1:2] if m > 1 else torch.ones(1, device="cuda"), w[:, :0], torch.ones(1, device="cuda"), bias=bias, dtype=torch.float16)
    assert torch.equal(got, bias.expand(m, n))
    got = tbvcoll.matmul_int8(x, one, w, one, dtype=torch.float16).cpu()
    total = (x.cpu().double() @ w.cpu().double().t())
    assert torch.equal(got, total.float().half())           # exact sums, some beyond fp16: infinities of their sign


@gpu
def test_product_of_any_leading_shape():
    x, w = codes_of(1, 2 * 3 * 4, 96).cuda(), codes_of(2, 40, 96).cuda()
    xs, ws = scales_of(3, 24).cuda(), scales_of(4, 40).cuda()
    flat = tbvcoll.matmul_int8(x, xs, w, ws)
    assert torch.equal(tbvcoll.matmul_int8(x.view(2, 3, 4, 96), xs.view(2, 3, 4), w, ws).view(24, 40), flat)
    assert torch.equal(tbvcoll.matmul_int8(x[5], xs[5], w, ws), flat[5])
    assert tbvcoll.matmul_int8(x[:0], xs[:0], w, ws).shape == (0, 40)
    assert tbvcoll.matmul_int8(x, xs, w[:0], ws[:0]).shape == (24, 0)


@gpu
def test_product_refusals():
    x, w = codes_of(1, 8, 64).cuda(), codes_of(2, 32, 64).cuda()
    xs, ws = scales_of(3, 8).cuda(), scales_of(4, 32).cuda()
    good = dict(x=x, x_scale=xs, w=w, w_scale=ws)
    for bad in (dict(x=x.float()), dict(w=w.float()), dict(w=w[:, :63]), dict(x_scale=xs[:7]), dict(w_scale=ws[:31]), dict(x_scale=xs.double()),
                dict(x_scale=xs.cpu()), dict(w=w.cpu()), dict(bias=torch.zeros(32, device="cuda")), dict(bias=torch.zeros(31, device="cuda", dtype=torch.bfloat16)),
                dict(out=torch.empty(8, 31, device="cuda")), dict(out=torch.empty(8, 32, device="cuda", dtype=torch.float64)), dict(dtype=torch.int32),
                dict(out=torch.empty(32, 8, device="cuda").t()), dict(w=w.view(2, 16, 64)), dict(x=x.t(), w=codes_of(1, 4, 8).cuda(), x_scale=torch.ones(64, device="cuda"), w_scale=ws[:4]),
                dict(w_scale=torch.ones(64, device="cuda")[::2]), dict(out=torch.empty(1, 32, device="cuda").expand(8, 32))):
        with pytest.raises(ValueError):
            tbvcoll.matmul_int8(**(good | bad))
    # an output on top of an operand: refused by the library
    buf = torch.zeros(8 * 64, dtype=torch.int8, device="cuda")
    with pytest.raises(RuntimeError):
        tbvcoll.matmul_int8(buf.view(8, 64), xs, w, ws, out=buf.view(torch.bfloat16)[:8 * 32].view(8, 32))


# ------------------------------------------------------------------ rotary positions

def turn_back_and_forth(q, k, positions, freqs, scale, interleaved, inverse, q_out=None, k_out=None):
    shape4 = (lambda t: t if t.dim() == 4 else t[None])
    p = positions if positions.dim() == 2 else positions[None].expand(shape4(q).shape[0], -1)
    wants = [None if t is None else want_rotary(shape4(t), p, freqs, scale, interleaved, inverse) for t in (q, k)]
    wants = [None if w is None else (w[0].view_as(t) if t.dim() == 4 else w[0][0], w[1] if t.dim() == 4 else w[1][0]) for w, t in zip(wants, (q, k))]
    got = tbvcoll.rotary(q, k, positions, freqs, scale=scale, interleaved=interleaved, inverse=inverse, q_out=q_out, k_out=k_out)
    for g, w in zip(got, wants):
        if w is None:
            assert g is None
            continue
        check(g, w[0], w[1], g.dtype, (tuple(g.shape), interleaved, inverse))
    return got


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,head,rot", [(1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (8, 16, 4, 128, 64), (5, 3, 1, 80, 80), (7, 2, 2, 96, 46),
                                                   (13, 15, 5, 64, 64), (3, 1, 1, 256, 32), (4, 2, 1, 33, 18), (130, 4, 4, 192, 192), (2, 70, 3, 576, 64),
                                                   (1, 1, 0, 64, 0), (6, 5, 2, 100, 100), (3, 2, 1, 4096, 4096), (515, 2, 1, 72, 72)])
def test_rotary_matches_the_definition(name, interleaved, tokens, hq, hk, head, rot):
    dt = DT[name]
    q = dev(synth.normal(tokens + hq, tokens * hq * head), dt).view(tokens, hq, head)
    k = dev(synth.normal(tokens + 3 * head, tokens * hk * head), dt).view(tokens, hk, head) if hk else None
    positions = torch.from_numpy((synth.bits32(5, tokens) % np.uint64(1 << 20)).astype(np.int64)).cuda()
    positions[0] = 0 if tokens > 1 else 131071
    freqs = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / max(rot, 1))
    inverse = bool((tokens + head) % 2)
    say("rotary", name, interleaved, tokens, hq, hk, head, rot, inverse)
    q0 = q.clone()
    out = turn_back_and_forth(q, k, positions, freqs, 1.25, interleaved, inverse, torch.empty_like(q), None if k is None else torch.empty_like(k))
    assert torch.equal(q, q0)                                             # the input stays
    assert torch.equal(out[0][..., rot:], q[..., rot:])                   # the rest of the head is copied bit for bit
    # in place, with int32 positions: the same bits
    q1, k1 = q.clone(), None if k is None else k.clone()
    same = tbvcoll.rotary(q1, k1, positions.int(), freqs, scale=1.25, interleaved=interleaved, inverse=inverse)
    assert same[0] is q1 and same[1] is k1
    assert torch.equal(q1, out[0]) and (k is None or torch.equal(k1, out[1]))


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_layouts(name, interleaved):
    """Views of a packed projection in place (the values and what lies between stay), heads before tokens, batches with
    positions of their own and shared, reversed strides of an input, unaligned starts."""
    dt, b, t, hq, hk, d = DT[name], 2, 9, 6, 2, 64
    freqs, _ = tbvcoll.rotary_frequencies(d)
    pos = torch.tensor([[0, 1, 2, 3, 4, 5, 6, 7, 8], [100000, 5, 70, 1, 1, 0, 131071, 3, 1 << 20]], device="cuda")
    packed = dev(synth.normal(1, b * t * (hq + 2 * hk) * d), dt).view(b, t, hq + 2 * hk, d)
    before = packed.clone()
    turn_back_and_forth(packed[:, :, :hq], packed[:, :, hq:hq + hk], pos, freqs, 1.0, interleaved, False)
    assert torch.equal(packed[:, :, hq + hk:], before[:, :, hq + hk:]) and not torch.equal(packed, before)
    # heads before tokens, shared positions
    packed = before.clone().transpose(1, 2).contiguous().transpose(1, 2)
    turn_back_and_forth(packed[:, :, :hq], packed[:, :, hq:hq + hk], pos[0], freqs, 1.0, interleaved, True)
    # part of a wider, oddly placed buffer, tokens every other row
    wide = dev(synth.normal(2, 2 * t * (hq * d + 3) + 8), dt)[5:5 + 2 * t * (hq * d + 3)].view(2 * t, hq * d + 3)
    q = wide[::2, 1:1 + hq * d].unflatten(1, (hq, d))
    turn_back_and_forth(q, None, pos[1], freqs, 1.0, interleaved, False, torch.empty(t, hq, d, dtype=dt, device="cuda"))
    rest = wide.clone()
    turn_back_and_forth(q, None, pos[1], freqs, 1.0, interleaved, False)
    keep = torch.ones_like(wide, dtype=torch.bool)
    keep[::2, 1:1 + hq * d] = False
    assert torch.equal(wide[keep], rest[keep])
    # one key head shared by all (stride 0) into an output of its own; positions of every other element
    k = before[:, :, :1].expand(b, t, hk, d)
    turn_back_and_forth(before[:, :, :hq], k, pos.repeat_interleave(2, 1)[:, ::2], freqs, 1.0, interleaved, False,
                        torch.empty(b, t, hq, d, dtype=dt, device="cuda"), torch.empty(b, t, hk, d, dtype=dt, device="cuda"))


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_far_and_negative_positions(interleaved):
    """Positions up to 2^40 (beyond 2^22 rad the fp64 angle itself is off by 2^-53 of it on either side: bounded below)."""
    q = dev(synth.normal(1, 6 * 2 * 64), torch.float32).view(6, 2, 64)
    pos = torch.tensor([0, -1, -131072, (1 << 22) - 1, (1 << 31) + 5, 1 << 40], device="cuda")
    freqs, _ = tbvcoll.rotary_frequencies(64)
    got, _ = tbvcoll.rotary(q, None, pos, freqs, interleaved=interleaved, q_out=torch.empty_like(q))
    want, tol = want_rotary(q[None], pos[None], freqs, 1.0, interleaved, False)
    # the angle on either side: one rounded product, and here two more (times 1 / 2 pi, itself rounded): 4 * 2^-53 relative
    tol = tol + (pos.abs().double().cpu()[None, :, None, None] * 4 * 2.0 ** -53) * q[None].abs().double().cpu().amax(-1, keepdim=True) * 2
    check(got, want[0], tol[0], torch.float32, interleaved)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_inverse_is_the_gradient(interleaved):
    """Against the transpose (sum of y * g = sum of q * inverse(g)) and against differences of the forward call, which is
    linear: f(q + e) - f(q - e) over 2 for unit steps is the Jacobian's column up to its own rounding."""
    t, h, d, scale = 3, 2, 16, 1.5
    q, g = (dev(synth.normal(i, t * h * d), torch.float32).view(t, h, d) for i in (1, 2))
    pos = torch.tensor([3, 0, 90001], device="cuda")
    freqs, _ = tbvcoll.rotary_frequencies(12)
    fwd = lambda v: tbvcoll.rotary(v, None, pos, freqs, scale=scale, interleaved=interleaved, q_out=torch.empty_like(v))[0]  # noqa: E731
    back, _ = tbvcoll.rotary(g, None, pos, freqs, scale=scale, interleaved=interleaved, inverse=True, q_out=torch.empty_like(g))
    # each term of either sum is off by at most 10.2 u scale (|a| + |b|) of its partner
    bound = 2 * 10.2 * U * scale * 2 * float(q.abs().double().sum() * g.abs().double().max())
    assert abs(float((fwd(q).double() * g.double()).sum() - (q.double() * back.double()).sum())) <= bound
    diff = torch.zeros_like(g, dtype=torch.float64)
    for i in range(q.numel()):
        e = torch.zeros_like(q)
        e.view(-1)[i] = 1.0
        col = (fwd(q + e).double() - fwd(q - e).double()) / 2
        diff.view(-1)[i] = (col * g.double()).sum()
    size = float((q.abs().max() + 1) * 2 * scale)
    # two outputs depend on an input, each off by 11 u of its size on either side of the difference; then the call's own error
    assert float((diff - back.double()).abs().max()) <= 4 * 11 * U * size * float(g.abs().max()) * 2


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_in_an_autograd_function(interleaved):
    in_a_process_of_its_own("autograd_function", interleaved)


def autograd_function(interleaved):
    """The backward pass as a training program has it, a shared (expanded) key head among the inputs, against autograd
    through the plain formula in 64 bits on the CPU; captured into a graph with leaves of its own."""
    t, hq, hk, d, scale = 5, 4, 2, 32, 1.25
    pos = torch.tensor([0, 7, 70000, 3, 3], device="cuda")
    freqs, _ = tbvcoll.rotary_frequencies(24)

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k):
            return tbvcoll.rotary(q, k, pos, freqs, scale=scale, interleaved=interleaved, q_out=torch.empty_like(q), k_out=k.new_empty(k.shape))

        @staticmethod
        def backward(ctx, gq, gk):
            return tbvcoll.rotary(gq, gk, pos, freqs, scale=scale, interleaved=interleaved, inverse=True, q_out=gq.new_empty(gq.shape), k_out=gk.new_empty(gk.shape))

    q, k = (dev(synth.normal(i, t * h * d), torch.float32).view(t, h, d) for i, h in ((1, hq), (2, 1)))
    gq, gk = (dev(synth.normal(i, t * h * d), torch.float32).view(t, h, d) for i, h in ((3, hq), (4, hk)))
    q.requires_grad_(), k.requires_grad_()

    def grads():
        yq, yk = Rotary.apply(q, k.expand(t, hk, d))
        return torch.autograd.grad((yq, yk), (q, k), (gq, gk), retain_graph=True)

    eager = grads()
    wq, tq = want_rotary(gq[None], pos[None], freqs, scale, interleaved, True)
    wk, tk = want_rotary(gk[None], pos[None], freqs, scale, interleaved, True)
    check(eager[0], wq[0], tq[0], torch.float32, "dq")
    # the shared head's gradient is the sum over its heads: one more rounding of each of the hk - 1 additions
    check(eager[1], wk[0].sum(1, keepdim=True), tk[0].sum(1, keepdim=True) + U * wk[0].abs().sum(1, keepdim=True), torch.float32, "dk")
    q2, k2 = q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = Rotary.apply(q2, k2.expand(t, hk, d))
        caught = torch.autograd.grad(out, (q2, k2), (gq, gk))
    for _ in range(3):
        gq.mul_(1)                                                        # the program's own work between replays
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(caught[0], eager[0]) and torch.equal(caught[1], eager[1])


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("apart", [(3 << 30) + 4096, (4 << 30) - 16 * 512, (4 << 30) - 8 * 512, 5 << 30])
def test_rotary_outputs_far_apart(interleaved, apart):
    """Outputs of q and k at two places of one buffer, below and beyond what a 32-bit offset reaches; what is around them
    stays as it was."""
    t, hq, hk, d = 8, 4, 2, 128
    q, k = (dev(synth.normal(i, t * h * d), torch.bfloat16).view(t, h, d) for i, h in ((1, hq), (2, hk)))
    buf = torch.zeros(apart // 2 + 16384, dtype=torch.bfloat16, device="cuda")
    for first, second in (("q", "k"), ("k", "q")):
        buf.zero_()
        at = {first: 4096, second: apart // 2 + 4096}
        q_out, k_out = (buf[at[n]:at[n] + t * h * d].view(t, h, d) for n, h in (("q", hq), ("k", hk)))
        pos, (freqs, _) = torch.arange(t, device="cuda") * 1000, tbvcoll.rotary_frequencies(d)
        say("rotary", apart, first)
        tbvcoll.rotary(q, k, pos, freqs, interleaved=interleaved, q_out=q_out, k_out=k_out)
        for x, o in ((q, q_out), (k, k_out)):
            want, tol = want_rotary(x[None], pos[None], freqs, 1.0, interleaved, False)
            check(o, want[0], tol[0], torch.bfloat16, (apart, first))
        q_out.zero_(), k_out.zero_()
        assert int(torch.count_nonzero(buf)) == 0


@gpu
def test_rotary_refusals():
    q, k = torch.zeros(4, 3, 64, device="cuda"), torch.zeros(4, 1, 64, device="cuda")
    pos, freqs = torch.arange(4, device="cuda"), torch.ones(32, dtype=torch.float64, device="cuda")
    good = dict(q=q, k=k, positions=pos, freqs=freqs)
    for bad in (dict(q=q.double()), dict(k=k.half()), dict(positions=pos[:3]), dict(positions=pos.float()), dict(freqs=freqs.float()),
                dict(freqs=torch.ones(33, dtype=torch.float64, device="cuda")), dict(freqs=torch.ones(64, dtype=torch.float64, device="cuda")[::2]),
                dict(q=q[0]), dict(k=k[:3]), dict(k=torch.zeros(4, 1, 32, device="cuda")), dict(q_out=torch.zeros(4, 3, 63, device="cuda")),
                dict(q_out=q.half()), dict(k=None, k_out=k), dict(q=torch.zeros(4, 3, 128, device="cuda")[..., ::2]), dict(positions=pos.cpu()),
                dict(positions=pos[None]), dict(freqs=freqs.cpu())):
        with pytest.raises(ValueError):
            tbvcoll.rotary(**(good | bad))
    for bad in (dict(q_out=k.expand(4, 3, 64)), dict(k=q[:, :1]), dict(q_out=q[:, [0]].expand(4, 3, 64))):     # overlaps, found by the library
        with pytest.raises(RuntimeError):
            tbvcoll.rotary(**(good | bad))


# ------------------------------------------------------------------ together

def layer_weights(hidden, heads, kv, head, seed):
    n = (heads + 2 * kv) * head
    return (codes_of(seed, n, hidden).cuda(), scales_of(seed + 1, n, 0.0004).cuda(), codes_of(seed + 2, hidden, heads * head).cuda(),
            scales_of(seed + 3, hidden, 0.0004).cuda())


@gpu
@pytest.mark.parametrize("tokens", [1, 8, 77])
def test_half_a_decoder_layer(orc, tokens):
    """all-reduce + RMSNorm -> int8 rows -> packed projection -> rotary in place -> (values as attention's output) ->
    row-parallel projection -> all-reduce, each stage against its definition on the stage's own input."""
    hidden, heads, kv, head = 512, 6, 2, 64
    w1, s1, w2, s2 = layer_weights(hidden, heads, kv, head, 40)
    freqs, mult = tbvcoll.rotary_frequencies(head, factor=4.0, method="ramp", context=2048)
    with session(rails=2, cap=4 << 20, TBV_NSLOT=4) as tbv:
        part, peer = (dev(synth.normal(i, tokens * hidden), torch.bfloat16).view(tokens, hidden) for i in (50, 51))
        weight = dev(1.0 + 0.25 * synth.normal(52, hidden), torch.bfloat16)
        out = torch.empty_like(part)
        tbv.stage_peer(peer)
        normed = tbv.all_reduce_rmsnorm(part, weight, 1e-6, out=out)
        codes, scale = tbv.quantize_int8(normed)
        qkv = tbv.matmul_int8(codes, scale, w1, s1)
        turned = qkv.clone().view(tokens, heads + 2 * kv, head)
        pos = torch.arange(tokens, device="cuda") + 5000
        tbv.rotary(turned[:, :heads], turned[:, heads:heads + kv], pos, freqs, scale=mult)
        attended = turned[:, :heads].reshape(tokens, heads * head)
        peer2 = dev(synth.normal(53, tokens * hidden), torch.bfloat16).view(tokens, hidden)
        tbv.stage_peer(peer2)
        total = tbv.linear_int8_all_reduce(attended, w2, s2)
        torch.cuda.synchronize()
        want = orc.sum_rmsnorm(orc.DT_BF16, orc.torch_bits(part), orc.torch_bits(peer), orc.torch_bits(weight), hidden, 1e-6)[1]
        assert np.array_equal(orc.torch_bits(normed).reshape(-1), want)
        c, s = want_rows(normed)
        assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu(), s)
        r, before = want_product(c, s, w1, s1, None)
        check(qkv, r, before, torch.bfloat16, "qkv")
        r, before = want_rotary(qkv.view(1, tokens, -1, head)[:, :, :heads + kv], pos[None], freqs, mult, False, False)
        check(turned[:, :heads + kv], r[0], before[0], torch.bfloat16, "rotary")
        assert torch.equal(turned[:, heads + kv:], qkv.view(tokens, -1, head)[:, heads + kv:])
        c2, sc2 = tbv.quantize_int8(attended)
        partial = tbv.matmul_int8(c2, sc2, w2, s2)
        assert np.array_equal(orc.torch_bits(total), orc.torch_bits(orc.sum_torch(partial.cpu(), peer2.cpu())))
        r, before = want_product(*want_rows(attended), w2, s2, None)
        check(partial, r, before, torch.bfloat16, "row-parallel product")
        assert not tbv.err()


@gpu
def test_row_parallel_linear_declines_like_all_reduce():
    x, (w, s) = dev(synth.normal(1, 4 * 64), torch.bfloat16).view(4, 64), (codes_of(1, 32, 64).cuda(), scales_of(2, 32).cuda())
    tbvcoll.shutdown()
    assert tbvcoll.linear_int8_all_reduce(x, w, s) is None                      # not initialised
    with session(rails=1, cap=4096) as tbv:
        assert tbv.linear_int8_all_reduce(x.repeat(33, 1), w, s) is None        # 132 x 32 bf16 are over the cap
        y = tbv.linear_int8_all_reduce(x, w, s)                                 # no staged peer: it echoes this rank
        one = tbv.matmul_int8(*tbv.quantize_int8(x), w, s)
        torch.cuda.synchronize()
        assert torch.equal(y, one + one)


@gpu
def test_intercept_row_linear():
    from types import SimpleNamespace
    from libtbvcoll_amd import vllm_intercept

    class Group:
        def __init__(self, name, world_size):
            self.unique_name, self.world_size = name, world_size

        def all_reduce(self, t):
            return t * 3

    ps = SimpleNamespace(GroupCoordinator=Group, get_tp_group=lambda: SimpleNamespace(unique_name="tp:0"))
    x, (w, s) = dev(synth.normal(1, 4 * 64), torch.bfloat16).view(4, 64), (codes_of(1, 32, 64).cuda(), scales_of(2, 32).cuda())
    tbvcoll.shutdown()
    one = tbvcoll.matmul_int8(*tbvcoll.quantize_int8(x), w, s)
    ic = vllm_intercept.install(ps, 0, "rail0", cap_bytes=4096)
    try:
        assert torch.equal(ic.row_linear_int8(Group("tp:0", 2), x, w, s), one + one)     # through the library (echoing peer)
        assert torch.equal(ic.row_linear_int8(Group("pp:0", 2), x, w, s), one * 3)       # another group: the original
        assert torch.equal(ic.row_linear_int8(Group("tp:0", 1), x, w, s), one)           # alone
        torch.cuda.synchronize()
        assert ic.counters["n"] == 1
    finally:
        ic.uninstall()
        tbvcoll.shutdown()


def in_a_process_of_its_own(name, *args):
    """Streams, once made, stay for the life of a process, which multiplexes them onto a few hardware queues: work on streams
    of its own runs in a child, so that the tests of the all-reduce's streams find the process as it was without it."""
    say(name, *args, "in a process of its own")
    code = f"import sys; sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]; import test_layer_ops as t; t.{name}(*{args!r}); print('DONE', flush=True)"
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=240)
    assert "DONE" in p.stdout, (p.returncode, p.stdout[-1000:], p.stderr[-3000:])


@gpu
@pytest.mark.parametrize("work", ["graph_and_two_streams", "two_threads"])
def test_layer_ops_on_streams(work):
    in_a_process_of_its_own(work)


def graph_and_two_streams():
    """Captured once and replayed with new inputs and the program's own work in between; the same calls on two streams at
    once, eagerly and as two graphs replayed side by side (nothing is shared between calls)."""
    tokens, heads, kv, head, hidden = 40, 4, 2, 64, 256
    w1, s1, w2, s2 = layer_weights(hidden, heads, kv, head, 60)
    freqs, _ = tbvcoll.rotary_frequencies(head)
    pos = torch.arange(tokens, device="cuda")

    def steps(x):
        qkv = tbvcoll.matmul_int8(*tbvcoll.quantize_int8(x), w1, s1)
        h = qkv.view(tokens, -1, head)
        tbvcoll.rotary(h[:, :heads], h[:, heads:heads + kv], pos, freqs)
        return tbvcoll.matmul_int8(*tbvcoll.quantize_int8(h[:, :heads].reshape(tokens, heads * head)), w2, s2), qkv

    xs = [dev(synth.normal(70 + i, tokens * hidden), torch.float16).view(tokens, hidden) for i in range(8)]
    eager = [[t.clone() for t in steps(x)] for x in xs]
    ins = [torch.empty_like(xs[0]) for _ in range(2)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[i]):
            outs.append(steps(ins[i]))
        graphs.append(g)
    for r in range(4):
        for i in range(2):
            ins[i].copy_(xs[2 * r + i])
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], eager[2 * r + i])), (r, i)
        assert torch.equal(steps(xs[r])[0], eager[r][0])                        # eager work between replays
    got = []
    for i, x in enumerate(xs):
        streams[i % 2].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[i % 2]):
            got.append(steps(x))
    torch.cuda.synchronize()
    for a, b in zip(got, eager):
        assert all(torch.equal(u, v) for u, v in zip(a, b))


def two_threads():
    """Two threads at once, each on a stream of its own: every result is that of the calls made alone."""
    tokens, heads, head, hidden = 24, 4, 64, 512
    w, ws = codes_of(80, heads * head, hidden).cuda(), scales_of(81, heads * head, 0.0004).cuda()
    freqs, _ = tbvcoll.rotary_frequencies(head)
    pos = torch.arange(tokens, device="cuda")
    xs = [dev(synth.normal(82 + i, tokens * hidden), torch.bfloat16).view(tokens, hidden) for i in range(2)]

    def steps(x):
        y = tbvcoll.matmul_int8(*tbvcoll.quantize_int8(x), w, ws).view(tokens, heads, head)
        return tbvcoll.rotary(y, None, pos, freqs, q_out=torch.empty_like(y))[0]

    want = [steps(x) for x in xs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                got = [steps(xs[i]) for _ in range(60)]
            stream.synchronize()
            bad.extend(r for r, y in enumerate(got) if not torch.equal(y, want[i]))
        except Exception as e:                                                  # a failure in a thread is the test's
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


FIRST_CALL_IN_A_CAPTURE = r"""
import sys
sys.path.insert(0, {root!r})
import torch
from libtbvcoll_amd import tbvcoll
x = torch.randn(40, 256, device="cuda"); w = torch.randint(-127, 128, (64, 256), device="cuda").to(torch.int8)
ws = torch.ones(64, device="cuda"); freqs, _ = tbvcoll.rotary_frequencies(16); pos = torch.arange(40, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    c, s = tbvcoll.quantize_int8(x)
    y = tbvcoll.matmul_int8(c, s, w, ws, dtype=torch.float32)
    h, _ = tbvcoll.rotary(y.view(40, 4, 16), None, pos, freqs, q_out=torch.empty(40, 4, 16, device="cuda"))
for k in range(3):
    x.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    c1, s1 = tbvcoll.quantize_int8(x)
    y1 = tbvcoll.matmul_int8(c1, s1, w, ws, dtype=torch.float32)
    h1, _ = tbvcoll.rotary(y1.view(40, 4, 16), None, pos, freqs, q_out=torch.empty_like(h))
    print("REPLAY", k, torch.equal(c, c1) and torch.equal(y, y1) and torch.equal(h, h1), flush=True)
"""


@gpu
def test_first_calls_inside_a_capture():
    say("first calls of the layer operators inside a capture, in a fresh process")
    p = subprocess.run([sys.executable, "-c", FIRST_CALL_IN_A_CAPTURE.format(root=ROOT)], capture_output=True, text=True, timeout=240)
    for k in range(3):
        assert f"REPLAY {k} True" in p.stdout, (p.stdout, p.stderr[-2000:])


@gpu
@pytest.mark.parametrize("m,n,k", [(1 << 21, 16, 16), (1100000, 3, 5), (2, (1 << 24) + 17, 16), (70000, 40, 33)])
def test_product_of_very_many_rows(m, n, k):
    """Rows beyond a grid's y, columns beyond its x: every result against the definition in int64."""
    x, w = codes_of(1, 4096, k).cuda().repeat((m + 4095) // 4096, 1)[:m], codes_of(2, 4096, k).cuda().repeat((n + 4095) // 4096, 1)[:n]
    one = torch.ones(1, device="cuda")
    say("product", m, n, k)
    got = tbvcoll.matmul_int8(x, one, w, one, dtype=torch.float32)
    if m > n:
        want = torch.matmul(x.float(), w.float().t().contiguous())              # below 2^24: exact in fp32
    else:
        want = torch.matmul(w.float(), x.float().t().contiguous()).t()
    assert torch.equal(got, want)


@gpu
def test_more_threads_than_a_launch_dimension_holds():
    """16.9 million rows of a block each: 2^32 threads and more in one launch."""
    rows, cols = 16_900_000, 1025
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tail = dev(synth.normal(4, 3 * cols), torch.bfloat16).view(3, cols)
    x[-3:] = tail
    x[1 << 20] = tail[0]
    say("quantize", rows, cols)
    codes, scale = tbvcoll.quantize_int8(x)
    c, s = want_rows(tail)
    assert torch.equal(codes[-3:].cpu(), c) and torch.equal(scale[-3:].cpu(), s)
    assert torch.equal(codes[1 << 20].cpu(), c[0]) and int((scale != 2.0 ** -126).sum()) == 4


# Ragged products that reach each of the product's kernels: few rows 16x16 .. 64x32, tiles 64x64 .. 256x256 (128x128 in its two
# depths), few rows with a weight of 32 MB and more, and the five for rows that start anywhere.
KERNELS = [(17, 40, 4096), (70, 33, 4000), (17, 40, 1040), (39, 1000, 1040), (7, 40, 144), (500, 8200, 16), (97, 2741, 1040), (333, 1000, 1040),
           (300, 2741, 272), (130, 4100, 1040), (333, 2741, 272), (1030, 1000, 144), (130, 8200, 1040), (500, 4100, 1040), (777, 2741, 1040),
           (777, 2741, 16), (2100, 1000, 16), (777, 8200, 144), (2100, 2741, 272), (1030, 8200, 144), (2100, 4100, 1040),
           (3, 8200, 4112), (16, 4100, 8208), (30, 8200, 8208), (1, 28700, 4096), (17, 40, 1041), (17, 40, 143), (300, 4100, 17), (777, 1000, 143), (300, 2741, 143), (500, 4100, 1041), (777, 4100, 143)]


@gpu
@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", KERNELS, ids=lambda v: str(v))
def test_every_kernel_of_the_product(m, n, k, name):
    dt = DT[name]
    x, w = codes_of(m + k, m, k), codes_of(n + 3 * k, n, k)
    xs, ws = scales_of(1, m), scales_of(2, n, 0.0005)
    bias = torch.from_numpy(synth.normal(3, n)).to(dt)
    say("product", m, n, k, name)
    out = torch.full((m, n + 8), 7.0, dtype=dt, device="cuda")
    tbvcoll.matmul_int8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), bias=bias.cuda(), out=out[:, :n])
    want, before = want_product(x, xs, w, ws, bias)
    check(out[:, :n], want, before, dt, (m, n, k, name))
    assert bool((out[:, n:] == 7.0).all())


@gpu
@pytest.mark.parametrize("m,n,k", [(4100, 4112, 1040), (5001, 7000, 1008)])
def test_product_with_a_large_result(m, n, k):
    """A result that is stored past the caches: every element, and the guards beside the rows."""
    x, w = codes_of(1, m, k).cuda(), codes_of(2, n, k).cuda()
    one = torch.ones(1, device="cuda")
    out = torch.full((m, n + 4), 7.0, device="cuda")
    say("product", m, n, k)
    tbvcoll.matmul_int8(x, one, w, one, out=out[:, :n])
    assert torch.equal(out[:, :n], torch.matmul(x.float(), w.float().t().contiguous())) and bool((out[:, n:] == 7.0).all())     # 1040 * 127^2 < 2^24: exact


@gpu
@pytest.mark.parametrize("m,n", [(1, 1), (2, 1), (1, 3), (17, 1), (40, 2), (130, 1), (300, 300)])
@pytest.mark.parametrize("k", [16, 32, 144])
def test_product_of_a_few_bytes(m, n, k):
    """Operands that end long before the loads that run ahead would: the buffers' range is what stops those."""
    x, w = codes_of(1, m, k).cuda(), codes_of(2, n, k).cuda()
    xs, ws = scales_of(3, m).cuda(), scales_of(4, n).cuda()
    say("product", m, n, k)
    got = tbvcoll.matmul_int8(x, xs, w, ws, dtype=torch.float32)
    sums = x.cpu().long() @ w.cpu().long().t()
    assert torch.equal(got.cpu(), sums.float() * xs.cpu()[:, None] * ws.cpu()[None])


@gpu
def test_tensors_that_ask_for_a_gradient_are_refused():
    """The kernels record no gradient: silently dropping one is an error, unless nobody asked for it."""
    x = torch.ones(4, 64, device="cuda", requires_grad=True)
    codes, scale = torch.ones(4, 64, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    learned = torch.ones(4, device="cuda", requires_grad=True)
    pos, freqs = torch.arange(4, device="cuda"), torch.ones(8, dtype=torch.float64, device="cuda")
    calls = [lambda: tbvcoll.quantize_int8(x), lambda: tbvcoll.matmul_int8(codes, learned, codes, scale), lambda: tbvcoll.matmul_int8(codes, scale, codes, learned),
             lambda: tbvcoll.matmul_int8(codes, scale, codes, scale, bias=learned, dtype=torch.float32),
             lambda: tbvcoll.rotary(x.view(4, 4, 16), None, pos, freqs), lambda: tbvcoll.rotary(x.detach().clone().view(4, 4, 16), x.view(4, 4, 16), pos, freqs)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call()
    assert bool((x == 1).all())
    with torch.no_grad():
        for call in calls:
            call()
    with torch.inference_mode():
        calls[1]()


@gpu
@pytest.mark.parametrize("stride", [1 << 22, (1 << 22) + 16, (1 << 23) + 3])
@pytest.mark.parametrize("m,n,k", [(3, 40, 272), (300, 2741, 272), (500, 4100, 1040)])
def test_product_of_rows_far_apart(m, n, k, stride):
    """Row strides at and beyond what a tile's 32-bit offsets hold, of x, and for few rows of w too."""
    x, w = codes_of(1, m, k), codes_of(2, n, k)
    xs, ws = scales_of(3, m), scales_of(4, n)
    far = torch.zeros((m - 1) * stride + k, dtype=torch.int8, device="cuda").as_strided((m, k), (stride, 1))
    far.copy_(x)
    wf = w.cuda()
    if n < 100:
        wf = torch.zeros((n - 1) * stride + k, dtype=torch.int8, device="cuda").as_strided((n, k), (stride, 1))
        wf.copy_(w)
    say("product", m, n, k, stride)
    got = tbvcoll.matmul_int8(far, xs.cuda(), wf, ws.cuda(), dtype=torch.float32)
    want, before = want_product(x, xs, w, ws, None)
    check(got, want, before, torch.float32, (m, n, k, stride))


@gpu
def test_offsets_beyond_32_bits():
    """Rows beyond 4 GiB of codes, inputs and outputs: the last rows' results are those of the rows alone."""
    k, m = 131056, 33000                                                       # 4.3e9 codes
    x = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    w, ws, xs = codes_of(1, 16, k).cuda(), scales_of(2, 16).cuda(), torch.ones(m, device="cuda")
    x[-3:] = codes_of(3, 3, k).cuda()
    got = tbvcoll.matmul_int8(x, xs, w, ws, dtype=torch.float32)
    assert torch.equal(got[-3:], tbvcoll.matmul_int8(x[-3:].clone(), xs[-3:], w, ws, dtype=torch.float32)) and not bool(got[:-3].any())
    del x, got
    rows, cols = 36000, 65536                                                  # 2.4e9 elements of bf16: 4.7 GB
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-2:] = dev(synth.normal(4, 2 * cols), torch.bfloat16).view(2, cols)
    codes, scale = tbvcoll.quantize_int8(x)
    c, s = want_rows(x[-2:])
    assert torch.equal(codes[-2:].cpu(), c) and torch.equal(scale[-2:].cpu(), s) and not bool(codes[:-2].any())
    del codes
    h = x.view(rows, 512, 128)
    freqs, _ = tbvcoll.rotary_frequencies(128)
    pos = torch.arange(rows, device="cuda")
    want, tol = want_rotary(h[None, -2:], pos[None, -2:], freqs, 1.0, False, False)
    tbvcoll.rotary(h, None, pos, freqs)
    check(h[-2:], want[0], tol[0], torch.bfloat16, "far tokens")
    assert not bool(h[:1000].any())


def test_the_shapes_cover_every_side_of_the_tiles():
    """The list above holds sizes below, at and above each tile edge, and k inside, at and across a step."""
    ms, ks = {s[0] for s in SHAPES}, {s[2] for s in SHAPES}
    for edge in (16, 32, 64, 128, 256):
        assert any(m < edge for m in ms) and edge in ms and any(edge < m < 2 * edge for m in ms)
    assert any(k % 16 for k in ks) and any(k % 16 == 0 and k % 128 for k in ks) and any(k % 128 == 0 for k in ks)
    assert len(list(itertools.chain(SHAPES))) == len(set(SHAPES))
