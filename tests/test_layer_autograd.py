"""What the layer's operators tell autograd.  They write through raw pointers, so they have to say which of the caller's
tensors they wrote: a backward pass that had saved one must raise, as after any other in-place operation, not use the
overwritten values.

The CPU tests give the calls tensors that say they lie on a GPU and take the launch away: what is looked at is what the
call does before and after it."""
import pytest
import torch
from torch.autograd import forward_ad

from gpu_util import say
from libtbvcoll_amd import tbvcoll

gpu = pytest.mark.gpu


class Stand(torch.Tensor):
    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def stand(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype).as_subclass(Stand)


@pytest.fixture
def launches(monkeypatch):
    """The launches that would have been made, by name."""
    names = []
    monkeypatch.setattr(tbvcoll, "_launch", lambda fn, device, call: names.append(fn.__name__))
    return names


def on_gpu(*shape, dtype=torch.float32):
    return torch.ones(shape, dtype=dtype, device="cuda")


def writing_calls(new):
    """(name, call, tensors of the caller's that it writes), tensors from `new`."""
    x, q, k = new(4, 16), new(4, 2, 16), new(4, 1, 16)
    x8, w8, s, s1 = new(4, 16, dtype=torch.int8), new(8, 16, dtype=torch.int8), new(8), new(4)
    pos, freqs = new(4, dtype=torch.int64), new(8, dtype=torch.float64)
    codes, scale, out, q_out, k_out = new(4, 16, dtype=torch.int8), new(4), new(4, 8, dtype=torch.bfloat16), new(4, 2, 16), new(4, 1, 16)
    return [("codes", lambda: tbvcoll.quantize_int8(x, codes=codes), [codes]),
            ("scale", lambda: tbvcoll.quantize_int8(x, scale=scale), [scale]),
            ("codes and scale", lambda: tbvcoll.quantize_int8(x, codes, scale), [codes, scale]),
            ("product", lambda: tbvcoll.matmul_int8(x8, s1, w8, s, out=out), [out]),
            ("q in place", lambda: tbvcoll.rotary(q, None, pos, freqs), [q]),
            ("q and k in place", lambda: tbvcoll.rotary(q, k, pos, freqs), [q, k]),
            ("q out, k in place", lambda: tbvcoll.rotary(q, k, pos, freqs, q_out=q_out), [q_out, k]),
            ("both out", lambda: tbvcoll.rotary(q, k, pos, freqs, q_out=q_out, k_out=k_out), [q_out, k_out])], \
        [x, q, k, x8, w8, s, s1, pos, freqs, codes, scale, out, q_out, k_out]


def versions(new):
    """Every call moves the version of exactly the tensors that it wrote."""
    calls, tensors = writing_calls(new)
    for name, call, wrote in calls:
        say("versions", name)
        before = [t._version for t in tensors]
        call()
        moved = [t._version > b for t, b in zip(tensors, before)]
        assert moved == [any(t is w for w in wrote) for t in tensors], name


def test_written_tensors_move_on(launches):
    versions(stand)
    assert set(launches) == {"tbv_step_quantize_i8", "tbv_step_matmul_i8", "tbv_step_rotary"}


def test_inference_tensors_have_no_version(launches):
    with torch.inference_mode():
        for _, call, _ in writing_calls(stand)[0]:
            call()
    assert len(launches) == 8


@gpu
def test_written_tensors_move_on_gpu():
    versions(on_gpu)


@gpu
@pytest.mark.parametrize("how", ["in place", "a view in place", "an output", "under no_grad"])
def test_backward_notices_a_saved_tensor_that_was_turned(how):
    """q needs no gradient, but its product with a learned tensor saved it for the backward pass."""
    q, p = torch.randn(4, 2, 16, device="cuda"), torch.ones(4, 2, 16, device="cuda", requires_grad=True)
    pos, freqs = torch.arange(4, device="cuda"), torch.ones(8, dtype=torch.float64, device="cuda")
    y = (q * p).sum()
    say("rotary after a product saved q:", how)
    if how == "in place":
        tbvcoll.rotary(q, None, pos, freqs)
    elif how == "a view in place":
        tbvcoll.rotary(q[1:3], None, pos[:2], freqs)
    elif how == "an output":
        tbvcoll.rotary(torch.ones_like(q), None, pos, freqs, q_out=q)
    else:
        with torch.no_grad():
            tbvcoll.rotary(q, None, pos, freqs)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@gpu
def test_backward_notices_a_saved_result_buffer():
    """A result buffer that is used again, saved by the step before."""
    x, w = (torch.ones(n, 16, dtype=torch.int8, device="cuda") for n in (4, 8))
    one, p = torch.ones(1, device="cuda"), torch.ones(4, 8, device="cuda", requires_grad=True)
    out = tbvcoll.matmul_int8(x, one, w, one, dtype=torch.float32)
    y = (out * p).sum()
    say("product into a saved result")
    tbvcoll.matmul_int8(x, one, w, one, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def outputs_that_ask(new):
    """Calls into outputs that require a gradient (fp32 ones; codes are integers and cannot)."""
    def leaf(*shape, dtype=torch.float32):
        return new(*shape, dtype=dtype).requires_grad_()
    x, q, k, x8, w8, s, s1, pos, freqs = writing_calls(new)[1][:9]
    out, q_out, k_out = leaf(4, 8, dtype=torch.bfloat16), leaf(4, 2, 16), leaf(4, 1, 16)
    return [lambda: tbvcoll.quantize_int8(x, scale=leaf(4)), lambda: tbvcoll.matmul_int8(x8, s1, w8, s, out=out),
            lambda: tbvcoll.matmul_int8(x8, s1, w8, s, out=out[:, :]),                                    # a view of such a leaf
            lambda: tbvcoll.rotary(q, k, pos, freqs, q_out=q_out), lambda: tbvcoll.rotary(q, k, pos, freqs, k_out=k_out)]


def test_outputs_that_ask_for_a_gradient_are_refused(launches):
    for call in outputs_that_ask(stand):
        with pytest.raises(ValueError, match="gradient"):
            call()
    assert not launches
    with torch.no_grad():
        for call in outputs_that_ask(stand):
            call()
    assert len(launches) == 5


@gpu
def test_outputs_that_ask_for_a_gradient_are_refused_on_gpu():
    for call in outputs_that_ask(on_gpu):
        with pytest.raises(ValueError, match="gradient"):
            call()


def learned_frequencies(new):
    q, k, pos, freqs = (writing_calls(new)[1][i] for i in (1, 2, 7, 8))
    return lambda: tbvcoll.rotary(q, k, pos, freqs.requires_grad_())


def test_frequencies_that_ask_for_a_gradient_are_refused(launches):
    with pytest.raises(ValueError, match="gradient"):
        learned_frequencies(stand)()
    assert not launches
    with torch.no_grad():
        learned_frequencies(stand)()
    assert len(launches) == 1


@gpu
def test_frequencies_that_ask_for_a_gradient_are_refused_on_gpu():
    with pytest.raises(ValueError, match="gradient"):
        learned_frequencies(on_gpu)()


def dual_calls(new, dual):
    """Calls in which one tensor, read or written, carries a tangent, by its name."""
    def d(*shape, dtype=torch.float32):
        return dual(new(*shape, dtype=dtype))
    x, q, k, x8, w8, s, s1, pos, freqs = writing_calls(new)[1][:9]
    return {"x": lambda: tbvcoll.quantize_int8(d(4, 16)), "scale": lambda: tbvcoll.quantize_int8(x, scale=d(4)),
            "x_scale": lambda: tbvcoll.matmul_int8(x8, d(4), w8, s), "w_scale": lambda: tbvcoll.matmul_int8(x8, s1, w8, d(8)),
            "bias": lambda: tbvcoll.matmul_int8(x8, s1, w8, s, bias=d(8), dtype=torch.float32),
            "out": lambda: tbvcoll.matmul_int8(x8, s1, w8, s, out=d(4, 8)), "q": lambda: tbvcoll.rotary(d(4, 2, 16), k, pos, freqs),
            "a view of q": lambda: tbvcoll.rotary(d(4, 4, 16)[:, :2], None, pos, freqs),
            "k": lambda: tbvcoll.rotary(q, d(4, 1, 16), pos, freqs), "freqs": lambda: tbvcoll.rotary(q, k, pos, d(8, dtype=torch.float64)),
            "q_out": lambda: tbvcoll.rotary(q, k, pos, freqs, q_out=d(4, 2, 16)), "k_out": lambda: tbvcoll.rotary(q, k, pos, freqs, k_out=d(4, 1, 16))}


def tangents_are_refused(new):
    with forward_ad.dual_level():
        for call in dual_calls(new, lambda t: forward_ad.make_dual(t, torch.ones_like(t))).values():
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):      # (no_grad does not turn forward mode off)
                call()
        for call in dual_calls(new, lambda t: t).values():                              # inside a level, but none of them a dual
            call()


def test_tensors_with_a_tangent_are_refused(launches):
    tangents_are_refused(stand)
    assert len(launches) == 12


@gpu
def test_tensors_with_a_tangent_are_refused_on_gpu():
    tangents_are_refused(on_gpu)


@gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_jvp_in_a_function(interleaved):
    """Forward mode as a program has it: rotation is linear, so the tangent's image is its rotation, bit for bit."""
    pos, (freqs, _) = torch.arange(5, device="cuda") * 777, tbvcoll.rotary_frequencies(16)

    def turn(v):
        return tbvcoll.rotary(v, None, pos, freqs, interleaved=interleaved, q_out=torch.empty_like(v))[0]

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q):
            return turn(q)

        @staticmethod
        def jvp(ctx, t):
            return turn(t)

    q, t = torch.randn(5, 3, 16, device="cuda"), torch.randn(5, 3, 16, device="cuda")
    with forward_ad.dual_level():
        y, got = forward_ad.unpack_dual(Rotary.apply(forward_ad.make_dual(q, t)))
    assert torch.equal(y, turn(q)) and torch.equal(got, turn(t))


def test_a_leaf_written_under_no_grad_moves_on(launches):
    with torch.no_grad():
        for call, leaf in ((lambda t: tbvcoll.quantize_int8(stand(4, 16), scale=t), stand(4)),
                           (lambda t: tbvcoll.matmul_int8(stand(4, 16, dtype=torch.int8), stand(1), stand(8, 16, dtype=torch.int8), stand(1), out=t), stand(4, 8))):
            leaf.requires_grad_()
            before = leaf._version
            call(leaf)
            assert leaf._version > before
    assert len(launches) == 2
