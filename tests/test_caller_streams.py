"""The caller's stream and the rails' side streams on the GPU's few hardware queues."""
import pytest
import torch

from gpu_util import dev, say, session
from libtbvcoll_amd import synth

pytestmark = pytest.mark.gpu


def exact_calls(tbv, seed, calls=3):
    for i in range(calls):
        a, p = (dev(synth.normal(seed + 10 * i + j, 1 << 18), torch.bfloat16) for j in (0, 1))
        tbv.stage_peer(p)
        out = torch.empty_like(a)
        assert tbv.all_reduce(a, out)
        torch.cuda.synchronize()
        assert torch.equal(out, a + p) and not tbv.err()


def test_the_default_stream_is_probed_too(capfd):
    """Its handle is null: that is a stream like the others, not one whose answer is known."""
    assert torch.cuda.current_stream().cuda_stream == 0
    for i in range(2):                                                   # (a second session asks again: its side streams are new)
        with session(rails=2, cap=1 << 20, TBV_WDOG=5) as tbv:
            capfd.readouterr()
            say("default stream, session", i)
            exact_calls(tbv, 20 + i)
            err = capfd.readouterr().err
            assert err.count("stream (nil) ") in (1, 2), err             # one line a rail, or one that says the queue is shared


def test_the_default_stream_with_many_streams_alive():
    """Sessions one after the other while more streams than hardware queues live: a side stream that comes to lie on the default
    stream's queue is found before a call relies on it."""
    streams = []
    for i in range(6):
        streams += [torch.cuda.Stream() for _ in range(3)]
        for s in streams:
            with torch.cuda.stream(s):
                torch.ones(16, device="cuda").mul_(2)
        torch.cuda.synchronize()
        with session(rails=2, cap=1 << 20, TBV_WDOG=5) as tbv:
            say("default stream beside", len(streams), "others")
            exact_calls(tbv, 50 + i)


def test_a_host_that_is_held_up_during_the_probe(capfd):
    """The wait is over by its bound before the host looks: that says nothing of separate queues, so the calls take the way
    that works on either."""
    with session(rails=2, cap=1 << 20, TBV_WDOG=5, TBV_PROBEDELAY=1000) as tbv:
        capfd.readouterr()
        say("probe with the host held up")
        exact_calls(tbv, 70)
        err = capfd.readouterr().err
        assert "shares a hardware queue" in err and "separate hardware queues" not in err, err
