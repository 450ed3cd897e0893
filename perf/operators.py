"""The int8 and rotary operators around the tensor-parallel all-reduce, as a serving or training program runs them.

`run` computes a case in plain torch, or, with `own` set, by the calls a user makes of `libtbvcoll_amd.tbvcoll`:

  quantize  rows of 32/16-bit values -> int8 codes and one scale a row.  What is returned are the values the codes stand
            for (codes * scale, one elementwise multiply on either side) and the scales.
            scale = max(f32(max|x| / 127), 2^-126);  code = x / scale to the nearest integer, ties to even.
  matmul    int8 activations [M, K] x int8 weights [N, K], a scale for each token and each output channel:
            out = T(float(sum_k x w) * x_scale * w_scale + bias).
  rotary    query and key heads rotated by their positions: pairs (i, i + rot/2) or (2i, 2i + 1) of the first `rot`
            elements of a head, the rest copied; `inverse` is the backward pass.
"""
import math

import torch

own = False

_T = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_MAX_MACS = 1 << 38            # multiply-adds of the largest listed product
_MAX_VALUES = 1 << 25          # elements of the largest quantised or rotated tensors


def _quantize(name, rows, k, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "k": k, "dtype": dtype}


def _matmul(name, m, n, k, dtype, bias):
    return {"name": name, "op": "matmul", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _rotary(name, tokens, heads, kv_heads, head, rot, dtype, interleaved, inverse, packed, far, stretch):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head": head, "rot": rot,
            "dtype": dtype, "interleaved": interleaved, "inverse": inverse, "packed": packed, "far": far, "stretch": stretch}


def listed():
    return [
        # eight decode tokens of hidden 4096, between the fused all-reduce + RMSNorm and the next product: latency
        _quantize("quantize-decode-8x4096", 8, 4096, "bf16"),
        # a prefill payload of the all-reduce's benchmark, 2048 tokens of hidden 4096
        _quantize("quantize-prefill-2048x4096", 2048, 4096, "bf16"),
        # one decode token through a square projection of hidden 4096: the weights' bytes are the work
        _matmul("matmul-decode-1", 1, 4096, 4096, "bf16", False),
        # sixteen sequences decoding together, a wide projection with a bias
        _matmul("matmul-decode-16", 16, 8192, 4096, "fp16", True),
        # a ragged batch and odd layer widths; the sums are kept in fp32
        _matmul("matmul-odd-77", 77, 2741, 1111, "fp32", True),
        # a prefill chunk mixed into a decode batch, the row-parallel product of a feed-forward layer
        _matmul("matmul-chunk-333", 333, 4096, 8192, "bf16", False),
        # the prefill payload through a wide projection
        _matmul("matmul-prefill-2048", 2048, 8192, 4096, "bf16", False),
        # a long prompt or a large offline batch
        _matmul("matmul-prefill-8192", 8192, 8192, 4096, "bf16", True),
        # eight decode tokens far into long contexts, the heads of one of two ranks, views of the packed projection
        _rotary("rotary-decode-8", 8, 16, 4, 128, 128, "bf16", False, False, True, 131072, 1.0),
        # a prefill of 2048 tokens, half layout, packed projection
        _rotary("rotary-prefill-2048", 2048, 32, 8, 128, 128, "bf16", False, False, True, 4096, 1.0),
        # 8191 tokens, interleaved pairs in half of each head, frequencies stretched for a long context
        _rotary("rotary-partial-8191", 8191, 16, 4, 128, 64, "fp16", True, False, False, 131072, 8.0),
        # gradients of a training step in fp32: an odd number of tokens and heads, heads of 80
        _rotary("rotary-backward-1021", 1021, 15, 5, 80, 80, "fp32", False, True, False, 8192, 1.0),
    ]


def _between(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("quantize", "matmul", "matmul", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "quantize":
        k = _between(rng, 64, 16384)
        k = max(16, k // 16 * 16) if rng.random() < 0.6 else k
        rows = _between(rng, 1, max(1, min(16384, _MAX_VALUES // k)))
        return {key: v for key, v in _quantize("", rows, k, dtype).items() if key != "name"}
    if op == "matmul":
        n, k = _between(rng, 256, 16384), _between(rng, 256, 16384)
        n = n // 16 * 16 if rng.random() < 0.7 else n
        k = k // 16 * 16 if rng.random() < 0.8 else k
        m = _between(rng, 1, max(1, min(8192, _MAX_MACS // (n * k))))
        return {key: v for key, v in _matmul("", m, n, k, dtype, rng.random() < 0.5).items() if key != "name"}
    heads = rng.randint(1, 48)
    kv_heads = rng.randint(1, min(heads, 12))
    head = rng.choice((64, 80, 96, 128, 192, 256))
    rot = rng.choice((head, head, head // 2, head // 4 * 2 - 2))
    tokens = _between(rng, 1, max(1, min(16384, _MAX_VALUES // ((heads + kv_heads) * head))))
    case = _rotary("", tokens, heads, kv_heads, head, rot, dtype, rng.random() < 0.5, rng.random() < 0.35, rng.random() < 0.5,
                   _between(rng, 2048, 1 << 20), rng.choice((1.0, 1.0, 4.0, 16.0)))
    return {key: v for key, v in case.items() if key != "name"}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = _T[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] == "quantize":
        # hidden states: N(0, 0.02^2) with one element in a thousand at +-8
        x = normal(case["rows"], case["k"]) * 0.02
        u = torch.rand(x.shape, generator=g, device="cuda")
        x = torch.where(u < 5e-4, 8.0, torch.where(u > 1 - 5e-4, -8.0, x)).to(t)
        return {"case": case, "x": x}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"case": case,
                "x": (normal(m, k) * 32).round().clamp(-127, 127).to(torch.int8),
                "x_scale": (normal(m).abs() + 0.5) * 0.02,
                "w": (normal(n, k) * 40).round().clamp(-127, 127).to(torch.int8),
                "w_scale": (normal(n).abs() + 0.5) * 0.0005,
                "bias": normal(n).to(t) if case["bias"] else None}
    n, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["head"]
    if case["packed"]:                      # the projection's output: query, key and value heads side by side
        qkv = normal(n, h + 2 * hk, d).to(t)
        q, k = qkv[:, :h], qkv[:, h:h + hk]
        out = torch.empty_like(qkv)
        q_out, k_out = out[:, :h], out[:, h:h + hk]
    else:
        q, k = normal(n, h, d).to(t), normal(n, hk, d).to(t)
        q_out, k_out = torch.empty_like(q), torch.empty_like(k)
    if n > case["far"] // 2:
        positions = torch.arange(n, device="cuda")
    else:                                   # sequences at different places, as in a mixed batch
        positions = torch.randint(0, case["far"], (n,), generator=g, device="cuda")
    # base^(-2i/rot), the slow ones divided by `stretch` (a ramp between the two), and the matching output scale
    rot = case["rot"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    freqs = 10000.0 ** (-2.0 * i / rot)
    ramp = ((i / max(1, rot // 2 - 1) - 0.25) / 0.5).clamp(0, 1)
    freqs = freqs * (1 - ramp) + freqs / case["stretch"] * ramp
    return {"case": case, "q": q, "k": k, "q_out": q_out, "k_out": k_out, "positions": positions, "freqs": freqs,
            "scale": 0.1 * math.log(case["stretch"]) + 1.0}


def run(state):
    case = state["case"]
    if own:
        from libtbvcoll_amd import tbvcoll
        if case["op"] == "quantize":
            codes, scale = tbvcoll.quantize_int8(state["x"])
            return torch.mul(codes, scale[:, None]), scale
        if case["op"] == "matmul":
            return tbvcoll.matmul_int8(state["x"], state["x_scale"], state["w"], state["w_scale"], bias=state["bias"],
                                       dtype=_T[case["dtype"]])
        return tbvcoll.rotary(state["q"], state["k"], state["positions"], state["freqs"], scale=state["scale"],
                              interleaved=case["interleaved"], inverse=case["inverse"], q_out=state["q_out"],
                              k_out=state["k_out"])
    if case["op"] == "quantize":
        x = state["x"].double()             # the quotient is compared with halves: a rounded one could fall on the wrong side
        scale = (x.abs().amax(1) / 127).float().clamp_min(2.0 ** -126)
        codes = torch.round(x / scale.double()[:, None]).to(torch.int8)
        return torch.mul(codes, scale[:, None]), scale
    if case["op"] == "matmul":
        out = state["x"].float() @ state["w"].float().t()
        out = out * state["x_scale"][:, None] * state["w_scale"]
        if state["bias"] is not None:
            out = out + state["bias"].float()
        return out.to(_T[case["dtype"]])
    angle = state["positions"].double()[:, None] * state["freqs"]
    cos = (angle.cos() * state["scale"]).float()[:, None]
    sin = (angle.sin() * state["scale"]).float()[:, None]
    if case["inverse"]:
        sin = -sin
    return tuple(_rotate(state[which], cos, sin, case) for which in ("q", "k"))


def _rotate(x, cos, sin, case):
    rot = case["rot"]
    first, rest = x[..., :rot].float(), x[..., rot:]
    if case["interleaved"]:
        a, b = first[..., 0::2], first[..., 1::2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = first[..., :rot // 2], first[..., rot // 2:]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((y.to(x.dtype), rest), dim=-1)


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * size + n * 4 + case["rows"] * 4, "flops": 3 * n}
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * size + (n * size if case["bias"] else 0), "flops": 2 * m * n * k}
    values = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["head"]
    turned = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rot"]
    return {"bytes": 2 * values * size + 8 * case["tokens"] + 4 * case["rot"], "flops": 3 * turned}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].to(torch.float64)
        top = torch.maximum(x.max(dim=1).values, -x.min(dim=1).values)
        scale = torch.clamp((top / 127.0).to(torch.float32), min=2.0 ** -126).to(torch.float64)
        low = torch.floor(x / scale[:, None])
        over = x - low * scale[:, None] - scale[:, None] / 2          # beyond, at or before the half
        odd = torch.remainder(low, 2) == 1
        up = (over > 0) | ((over == 0) & odd)
        return (low + up) * scale[:, None], scale
    if case["op"] == "matmul":
        total = torch.mm(s["w"].to(torch.float64), s["x"].to(torch.float64).t().contiguous()).t()
        total = total * torch.outer(s["x_scale"].to(torch.float64), s["w_scale"].to(torch.float64))
        return total if s["bias"] is None else total + s["bias"].to(torch.float64)
    # a pair as a complex number, turned by exp(+-i angle)
    sign = -1.0 if case["inverse"] else 1.0
    turn = torch.polar(torch.full((case["tokens"], case["rot"] // 2), s["scale"], dtype=torch.float64, device="cuda"),
                       sign * torch.outer(s["positions"].to(torch.float64), s["freqs"]))
    outs = []
    for x in (s["q"], s["k"]):
        y = x.to(torch.float64)
        n, h, _ = y.shape
        r = case["rot"]
        pairs = y[..., :r].reshape(n, h, r // 2, 2) if case["interleaved"] else y[..., :r].reshape(n, h, 2, r // 2).transpose(2, 3)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        z = z if case["interleaved"] else z.transpose(2, 3)
        y = y.clone()
        y[..., :r] = z.reshape(n, h, r)
        outs.append(y)
    return tuple(outs)
