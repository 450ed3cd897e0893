"""Calls of the layer's operators that their documentation allows, or that they have to refuse."""
import contextlib
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest
import torch

import test_layer_ops
from gpu_util import dev, say, session
from libtbvcoll_amd import synth, tbvcoll, vllm_intercept
from test_layer_autograd import launches, on_gpu, stand  # noqa: F401  (a fixture)
from test_layer_ops import DT, check, codes_of, scales_of, want_product, want_rows

gpu = pytest.mark.gpu


def bad_linear_calls(new):
    x, w, s = new(4, 64), new(32, 64, dtype=torch.int8), new(32)
    good = dict(x=x, w=w, w_scale=s)
    return [good | kw for kw in (dict(x=x.double()), dict(x=new()), dict(w=w.float()), dict(w=w[:, :63]), dict(w=w.view(2, 16, 64)), dict(out=new(4, 31)),
                                 dict(out=new(4, 32).half()), dict(out=new(32, 4).t()), dict(out=new(128)), dict(out=new(4, 64)[:, ::2]))]


def test_row_parallel_linear_refuses_before_it_declines(launches):  # noqa: F811
    tbvcoll.shutdown()                                                          # not initialised: every good call declines
    x, w, s = stand(4, 64), stand(32, 64, dtype=torch.int8), stand(32)
    assert tbvcoll.linear_int8_all_reduce(x, w, s) is None
    for bad in bad_linear_calls(stand) + [dict(x=x, w=torch.ones(32, 64, dtype=torch.int8), w_scale=s), dict(x=x, w=w, w_scale=s, out=torch.empty(4, 32))]:
        with pytest.raises(ValueError):
            tbvcoll.linear_int8_all_reduce(**bad)
    out = stand(4, 32)
    assert tbvcoll.linear_int8_all_reduce(x, w, s, out=out) is None and bool((out == 1).all()) and not launches


@gpu
def test_row_parallel_linear_into_an_output():
    x, (w, s) = dev(synth.normal(1, 4 * 64), torch.bfloat16).view(4, 64), (codes_of(1, 32, 64).cuda(), scales_of(2, 32).cuda())
    with session(rails=1, cap=4096) as tbv:
        one = tbv.matmul_int8(*tbv.quantize_int8(x), w, s)
        out = torch.full((4, 32), 3.0, dtype=torch.bfloat16, device="cuda")
        say("row-parallel linear into an output")
        assert tbv.linear_int8_all_reduce(x, w, s, out=out) is out              # no staged peer: it echoes this rank
        torch.cuda.synchronize()
        assert torch.equal(out, one + one)
        far = torch.full((132, 32), 3.0, dtype=torch.bfloat16, device="cuda")   # over the cap: declined, out as it was
        assert tbv.linear_int8_all_reduce(x.repeat(33, 1), w, s, out=far) is None
        torch.cuda.synchronize()
        assert bool((far == 3.0).all())
        none = tbv.linear_int8_all_reduce(x[:0], w, s)
        assert none.shape == (0, 32) and none.dtype is torch.bfloat16
        for bad in bad_linear_calls(on_gpu):
            with pytest.raises(ValueError):
                tbv.linear_int8_all_reduce(**bad)
        assert not tbv.err()


def test_row_parallel_linear_runs_on_its_tensors_device(launches, monkeypatch):  # noqa: F811
    """Tensors on another device than the current one (there is one GPU here: the devices are stand-ins)."""
    current, seen = [1], []

    @contextlib.contextmanager
    def device(i):
        before, current[0] = current[0], i
        yield
        current[0] = before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current[0], raising=False)
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(tbvcoll, "_lib", tbvcoll.load())
    monkeypatch.setattr(tbvcoll, "_cap", 1 << 20)
    monkeypatch.setattr(tbvcoll, "all_reduce", lambda t: seen.append((current[0], list(launches))) or True)
    assert tbvcoll.linear_int8_all_reduce(stand(4, 64), stand(32, 64, dtype=torch.int8), stand(32)).shape == (4, 32)
    assert seen == [(0, ["tbv_step_quantize_i8", "tbv_step_matmul_i8"])] and current == [1]


def part(t, *leading):
    """Columns 16 .. 79 of `leading` rows of a larger tensor."""
    return t.view(*leading, t.shape[-1])[..., 16:80]


def test_rows_of_part_of_a_larger_tensor():
    t = torch.zeros(24, 112)
    for leading in ((24,), (2, 12), (2, 3, 4), (24, 1), (1, 24), (2, 1, 12), (1, 1, 24), (2, 3, 1, 4)):
        x = part(t, *leading)
        assert tbvcoll._rows(x, x.shape, "x") == (24, 64, 112), leading
    for x, want in ((part(t, 2, 12)[:, :1], (2, 64, 12 * 112)), (part(t, 2, 12)[:1, :1], (1, 64, 64)), (part(t, 2, 12)[:, ::3], (8, 64, 3 * 112)),
                    (t.view(2, 3, 4, 112)[:, :, 0, :64], (6, 64, 448)), (t[:0].view(0, 3, 112)[..., :64], (0, 64, 64)), (t.view(2, 12, 112)[..., 5:6], (24, 1, 112))):
        assert tbvcoll._rows(x, x.shape, "x") == want
    for x in (part(t, 2, 12)[:, :5], t.view(2, 12, 112).transpose(0, 1), t.view(2, 12, 112).transpose(1, 2), t[:, None].expand(24, 2, 112),
              part(t, 2, 12).expand(3, 2, 12, 64), t.view(2, 3, 4, 112)[:, :, :2], t[None, :1].expand(5, 1, 112)):
        with pytest.raises(ValueError):
            tbvcoll._rows(x, x.shape, "x")


@gpu
@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("leading", [(2, 12), (2, 3, 4), (24, 1), (1, 24)])
def test_batches_that_are_part_of_a_larger_tensor(name, leading):
    """The columns of a packed projection, [batch, tokens, part of the columns]: read, and written with the rest left as it was."""
    dt = DT[name]
    x = part(dev(synth.normal(1, 24 * 112), dt).view(24, 112), *leading)
    store = torch.full((24, 112), 77, dtype=torch.int8, device="cuda")
    say("part of a larger tensor", name, leading)
    codes, scale = tbvcoll.quantize_int8(x, codes=part(store, *leading))
    c, s = want_rows(x)
    assert torch.equal(codes.cpu(), c) and torch.equal(scale.cpu(), s)
    assert torch.equal(tbvcoll.quantize_int8(x)[0], codes)
    w, ws = codes_of(2, 64, 64).cuda(), scales_of(3, 64).cuda()
    wide = torch.full((24, 112), 5.0, dtype=dt, device="cuda")
    tbvcoll.matmul_int8(codes, scale, w, ws, out=part(wide, *leading))
    want, before = want_product(c.reshape(24, 64), s.reshape(24), w, ws, None)
    check(wide[:, 16:80], want, before, dt, (name, leading))
    assert all(bool((t[:, :16] == v).all() and (t[:, 80:] == v).all()) for t, v in ((store, 77), (wide, 5.0)))


@gpu
@pytest.mark.parametrize("work", ["graph_and_two_streams()", "two_threads()", "autograd_function(False)", "autograd_function(True)", "FIRST_CALL_IN_A_CAPTURE"])
def test_a_process_with_graphs_and_streams_ends_well(work):
    """The work that the other tests run in processes of its own: here the process has to end with status 0 as well, its
    graphs and streams taken down."""
    say(work, "in a process of its own")
    code = f"import sys; sys.path[:0] = [{test_layer_ops.ROOT!r}, {os.path.join(test_layer_ops.ROOT, 'tests')!r}]; import test_layer_ops as t; t.{work}; print('DONE', flush=True)"
    if work == "FIRST_CALL_IN_A_CAPTURE":
        code = test_layer_ops.FIRST_CALL_IN_A_CAPTURE.format(root=test_layer_ops.ROOT) + "print('DONE', flush=True)\n"
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=110)
    assert p.returncode == 0 and "DONE" in p.stdout and "False" not in p.stdout, (p.returncode, p.stdout[-1000:], p.stderr[-3000:])


@gpu
def test_an_empty_batch_through_the_intercept():
    """No tokens (null pointers): nothing to sum, and the calls after it find the ring as it was."""
    class Group:
        unique_name, world_size = "tp:0", 2

        def all_reduce(self, t):
            return t * 3

    ps = SimpleNamespace(GroupCoordinator=Group, get_tp_group=Group)
    x, (w, s) = dev(synth.normal(1, 4 * 64), torch.bfloat16).view(4, 64), (codes_of(1, 32, 64).cuda(), scales_of(2, 32).cuda())
    tbvcoll.shutdown()
    one = tbvcoll.matmul_int8(*tbvcoll.quantize_int8(x), w, s)
    ic = vllm_intercept.install(ps, 0, "rail0", cap_bytes=4096)
    try:
        for i in range(10):                                                      # more calls than the ring has slots
            say("empty batch", i)
            none = ic.row_linear_int8(Group(), x[:0], w, s)
            assert none.shape == (0, 32) and none.dtype is torch.bfloat16
            assert torch.equal(ic.row_linear_int8(Group(), x, w, s), one + one)  # through the library (echoing peer)
        torch.cuda.synchronize()
        assert not tbvcoll.err()
    finally:
        ic.uninstall()
        tbvcoll.shutdown()
