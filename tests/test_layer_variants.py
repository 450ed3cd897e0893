"""Every variant of the layer's kernels against the operators' definitions: several heads to a thread and several tokens to
a block (rotary)."""
import pytest
import torch

from gpu_util import dev, say
from libtbvcoll_amd import synth, tbvcoll
from test_layer_ops import DT, check, want_rotary

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
