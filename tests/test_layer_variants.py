"""Every variant of the layer's kernels against the operators' definitions: several heads to a thread and several tokens to
a block (rotary), every width of lanes and registers (int8 rows), every tile (int8 product)."""
import os
import subprocess

import pytest
import torch

from gpu_util import dev, say
from libtbvcoll_amd import synth, tbvcoll
from test_layer_ops import DT, KERNELS, SHAPES, check, codes_of, scales_of, want_product, want_rotary, want_rows

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
gpu = pytest.mark.gpu

# Batch and tokens, heads of q and k, head and turned elements.  The kernel takes one head to a thread below 1024 tokens (or for
# one head), four where part of a head is copied, otherwise two, but one in the half layout beyond 4096 tokens; and several
# tokens to a block from 2048 tokens on where heads are small.
ROTARY = [(1, 1024, 2, 1, 64, 64), (1, 1025, 5, 2, 128, 128), (1, 1500, 3, 2, 80, 80), (1, 1030, 37, 4, 512, 512),      # two heads, the last thread with one; heads beyond a block
          (1, 1500, 5, 2, 96, 46), (1, 1025, 4, 1, 128, 64), (1, 3001, 2, 1, 72, 32), (1, 2047, 1, 1, 33, 18), (1, 1100, 9, 4, 192, 0),   # four heads: 7, 5, 3, 2, 13
          (1, 2049, 2, 1, 64, 64), (1, 8191, 2, 1, 64, 64), (1, 4097, 1, 1, 128, 128), (1, 8191, 2, 1, 128, 64), (1, 2051, 1, 0, 32, 32),  # several tokens to a block, the last block with fewer
          (1, 5000, 2, 1, 128, 128), (1, 4096, 3, 2, 128, 128), (1, 4097, 3, 2, 128, 128),                                 # either side of 4096
          (3, 700, 5, 2, 128, 128), (3, 1367, 2, 1, 48, 32), (2, 1024, 3, 0, 64, 64)]


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("batch,tokens,hq,hk,head,rot", ROTARY, ids=lambda v: str(v))
def test_rotary_of_many_tokens(name, interleaved, batch, tokens, hq, hk, head, rot):
    """Into part of a larger buffer, and in place in a packed one: the definition's values, and the rest as it was."""
    dt, all_heads = DT[name], hq + hk
    packed = dev(synth.normal(tokens + head, batch * tokens * (all_heads + 2) * head), dt).view(batch, tokens, all_heads + 2, head)
    store = torch.full_like(packed, 7.0)
    positions = (torch.arange(batch * tokens, device="cuda").view(batch, tokens) * 613) % 131072
    freqs = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / max(rot, 1))
    kw = dict(scale=1.25, interleaved=interleaved, inverse=bool(tokens % 2))
    heads = slice(1, 1 + all_heads)                                       # a head before and one behind stay as they are

    def parts(t):
        return t[:, :, 1:1 + hq], t[:, :, 1 + hq:1 + all_heads] if hk else None

    want, tol = want_rotary(packed[:, :, heads], positions, freqs, kw["scale"], interleaved, kw["inverse"])
    before = packed.clone()
    say("rotary", name, interleaved, batch, tokens, hq, hk, head, rot)
    tbvcoll.rotary(*parts(packed), positions, freqs, q_out=parts(store)[0], k_out=parts(store)[1], **kw)
    assert torch.equal(packed, before)
    check(store[:, :, heads], want, tol, dt, (name, interleaved, tokens))
    assert torch.equal(store[:, :, heads, rot:], packed[:, :, heads, rot:])
    assert bool((store[:, :, 0] == 7.0).all()) and bool((store[:, :, -1] == 7.0).all())
    tbvcoll.rotary(*parts(packed), positions, freqs, **kw)
    assert torch.equal(packed[:, :, heads], store[:, :, heads])
    assert torch.equal(packed[:, :, 0], before[:, :, 0]) and torch.equal(packed[:, :, -1], before[:, :, -1])


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("vectors", [8, 16, 32, 64, 128, 256, 512, 1024, 2048, 4096])
def test_rows_at_every_width(name, vectors):
    """A 16-byte vector below, at and above each width at which the rows take more lanes or registers; rows that do not fill
    a block."""
    per = 4 if name == "f32" else 8
    for cols in (vectors * per - per, vectors * per - 1, vectors * per, vectors * per + 1, vectors * per + per):
        rows = 35 if vectors <= 256 else 5
        x = dev(synth.normal(cols, rows * cols, 0.02), DT[name]).view(rows, cols)
        x[::3, cols - 1], x[1::3, 0] = 8.0, -8.0
        say("quantize", name, rows, cols)
        codes, scale = tbvcoll.quantize_int8(x)
        c, s = want_rows(x)
        assert torch.equal(scale.cpu(), s) and torch.equal(codes.cpu(), c), cols


LARGE = [(5001, 7000, 144), (5001, 7000, 1040), (4400, 8200, 528)]


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("m,n,k", LARGE)
def test_product_with_a_result_beyond_the_caches(name, m, n, k):
    """64 MiB and more in every type, with an edge either way; sums below 2^24 times 2^-9 are exact in fp32, then rounded."""
    x, w = codes_of(1, m, k).cuda(), codes_of(2, n, k).cuda()
    one, few = torch.ones(1, device="cuda"), torch.full((1,), 2.0 ** -9, device="cuda")
    out = torch.full((m, n + 8), 7.0, dtype=DT[name], device="cuda")
    say("product", name, m, n, k)
    tbvcoll.matmul_int8(x, one, w, few, out=out[:, :n])
    want = torch.matmul(x.float(), w.float().t().contiguous()) * 2.0 ** -9
    assert torch.equal(out[:, :n], want.to(DT[name])) and bool((out[:, n:] == 7.0).all())


ONCE = [(50, 5928, 8208), (33, 8151, 4128)]


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("m,n,k", ONCE)
def test_product_of_a_weight_that_is_read_once(name, m, n, k):
    dt = DT[name]
    x, w = codes_of(m + k, m, k), codes_of(n + 3 * k, n, k)
    xs, ws = scales_of(1, m), scales_of(2, n, 0.0005)
    say("product", name, m, n, k)
    got = tbvcoll.matmul_int8(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), dtype=dt)
    want, before = want_product(x, xs, w, ws, None)
    check(got, want, before, dt, (m, n, k, name))


PICKS = r"""
#include <stdio.h>
#include "tbv_tiles.h"
int main()
{
    unsigned m, n, k;
    while (scanf("%u %u %u", &m, &n, &k) == 3) printf("%d %d\n", tbv::pick_tile(tbv::kTiles, m, n, k), tbv::pick_tile(tbv::kAnyTiles, m, n, k));
    printf("%zu %zu\n", sizeof tbv::kTiles / sizeof *tbv::kTiles, sizeof tbv::kAnyTiles / sizeof *tbv::kAnyTiles);
}
"""


def test_the_shapes_reach_every_tile(tmp_path):
    """The products that the tests compute, by the library's own rule, so that another fit of it does not lose a kernel."""
    (tmp_path / "picks.cpp").write_text(PICKS)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "libtbvcoll_amd", "csrc"), str(tmp_path / "picks.cpp"),
                    "-o", str(tmp_path / "picks")], check=True)
    shapes = KERNELS + SHAPES + ONCE + LARGE
    out = subprocess.run([str(tmp_path / "picks")], input="".join(f"{m} {n} {k}\n" for m, n, k in shapes), capture_output=True, text=True, check=True).stdout
    *picks, sizes = [tuple(map(int, line.split())) for line in out.splitlines()]
    for held in (KERNELS, KERNELS + SHAPES):
        assert {p[0] for s, p in zip(shapes, picks) if s in held and s[2] % 16 == 0} == set(range(sizes[0]))
        assert {p[1] for s, p in zip(shapes, picks) if s in held and s[2] % 16 and s[2] > 16} == set(range(sizes[1]))
    large = picks[-len(LARGE):]
    assert {p[0] for p in large} == {sizes[0] - 1}                       # all of the largest tile, whose results pass the caches
    assert all(m * n * 2 >= 64 << 20 for m, n, k in LARGE)
    few = [16, 16, 16, 32, 64]                                            # rows of x of the tiles that read the weight once
    once = {p[0] for (m, n, k), p in zip(shapes, picks) if p[0] < len(few) and k % 16 == 0 and m <= few[p[0]] and n * k >= 32 << 20}
    assert once == set(range(len(few)))                                   # one row of blocks, a weight that is loaded past the L2s


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("head,rot", [(128, 128), (128, 64), (96, 46)])
def test_a_head_turns_alike_in_every_variant(name, interleaved, head, rot):
    """The same bits for a token among many, few or alone, in place or not, with or without a neighbour."""
    x = dev(synth.normal(head + rot, 5003 * 5 * head), DT[name]).view(5003, 5, head)
    pos, freqs = torch.arange(5003, device="cuda") * 29, 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device="cuda") / rot)
    say("rotary", name, interleaved, head, rot)

    def turn(t, p, k=None):
        return tbvcoll.rotary(t, k, p, freqs, scale=0.75, interleaved=interleaved, q_out=torch.empty_like(t), k_out=None if k is None else torch.empty_like(k))

    want = turn(x, pos)[0]
    for n in (1, 700, 1500, 2500, 4097):
        some = turn(x[:n, :3], pos[:n], x[:n, 3:4])
        assert torch.equal(some[0], want[:n, :3]) and torch.equal(some[1], want[:n, 3:4]), n
        here = x[:n].clone()
        tbvcoll.rotary(here, None, pos[:n], freqs, scale=0.75, interleaved=interleaved)
        assert torch.equal(here, want[:n]), n
        assert torch.equal(turn(x[:n, 2:3], pos[:n])[0], want[:n, 2:3]), n


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("n,k", [(1000, 1040), (1000, 1041), (72, 16), (72, 15)])
def test_a_row_of_the_product_is_alike_in_every_variant(name, n, k):
    """The same bits for a row of x in a large batch, a small one or alone, at an aligned address or not."""
    m, dt = 2100, DT[name]
    x, w, xs, ws = codes_of(1, m, k).cuda(), codes_of(2, n, k).cuda(), scales_of(3, m).cuda(), scales_of(4, n, 0.001).cuda()
    bias = dev(synth.normal(5, n), dt)
    say("product", name, m, n, k)
    want = tbvcoll.matmul_int8(x, xs, w, ws, bias=bias, dtype=dt)
    odd = torch.zeros(m * (k + 3) + 1, dtype=torch.int8, device="cuda")[1:].view(m, k + 3)[:, :k]
    odd.copy_(x)
    for rows in (1, 9, 20, 40, 100, 200, 400, 777, 1100):
        for t in (x, odd):
            assert torch.equal(tbvcoll.matmul_int8(t[7:7 + rows], xs[7:7 + rows], w, ws, bias=bias, dtype=dt), want[7:7 + rows]), rows
