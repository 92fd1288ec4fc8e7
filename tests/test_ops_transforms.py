"""Transformer-layer operators under torch's transformations: what would pass the work by is refused, what does not concern it is not."""
import pytest
import torch
import torch.autograd.forward_ad as fwd
from torch.fx.experimental.proxy_tensor import make_fx

from dorado_amd import capi, ops

FREQS = torch.ones(32, dtype=torch.float64)


def calls(device):
    """(name, f): f of one [1, 4, 2, 64] tensor, each operand in turn."""
    def x():
        return torch.ones((1, 4, 2, 64), dtype=torch.float16, device=device)
    f = FREQS.to(device)
    return [("x", lambda t: ops.rms_norm(t)), ("residual", lambda t: ops.rms_norm(x(), residual=t)),
            ("weight", lambda t: ops.rms_norm(x(), t[0, 0, 0])), ("q", lambda t: ops.rope(t, freqs=f)), ("k", lambda t: ops.rope(x(), t, freqs=f)[1]),
            ("query", lambda t: ops.attention(t, x(), x())), ("key", lambda t: ops.attention(x(), t, x())), ("value", lambda t: ops.attention(x(), x(), t))]


NAMES = [n for n, _ in calls("cpu")]


@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_refused(name):
    f, x = dict(calls("cpu"))[name], torch.ones((1, 4, 2, 64), dtype=torch.float16)
    with fwd.dual_level(), pytest.raises(capi.MibcNotSupported, match="tangents"):
        f(fwd.make_dual(x, x))
    with fwd.dual_level(), pytest.raises(capi.MibcError, match="no CPU form"):       # a tensor without one is as any other
        f(x)


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    f, x = dict(calls("cpu"))[name], torch.ones((1, 4, 2, 64), dtype=torch.float16)
    with pytest.raises(capi.MibcNotSupported, match="traced"):
        torch.jit.trace(f, (x,))
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(capi.MibcNotSupported, match="traced"):
            make_fx(f, tracing_mode=mode)(x)


def test_counters_may_watch():
    from torch.utils.flop_counter import FlopCounterMode
    with FlopCounterMode(display=False), pytest.raises(capi.MibcError, match="no CPU form"):
        ops.rms_norm(torch.ones((2, 64), dtype=torch.float16))


gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("name", NAMES)
def test_transformations_of_device_tensors_are_refused(name):
    f, x = dict(calls("cuda"))[name], torch.ones((1, 4, 2, 64), dtype=torch.float16, device="cuda")
    refused = (capi.MibcError, capi.MibcNotSupported, RuntimeError)
    with fwd.dual_level(), pytest.raises(capi.MibcNotSupported, match="tangents"):
        f(fwd.make_dual(x, x))
    with pytest.raises(capi.MibcNotSupported, match="traced"):
        torch.jit.trace(f, (x,))
    with pytest.raises(capi.MibcNotSupported, match="traced"):
        make_fx(f)(x)
    for transform in (lambda: torch.func.functionalize(f)(x), lambda: torch.vmap(f)(x[None]), lambda: torch.func.jvp(f, (x,), (x,)),
                      lambda: torch.func.grad(lambda y: f(y).float().sum())(x)):
        with pytest.raises(refused):
            transform()
    if name in ("residual", "value"):
        with pytest.raises(refused):
            f(torch._efficientzerotensor((1, 4, 2, 64), dtype=torch.float16, device="cuda"))


@gpu
def test_a_pending_negation_is_refused():
    z = torch.complex(torch.ones(3, 1), torch.full((3, 1), 2.0)).cuda()
    im = z.conj().imag
    assert im.is_neg()
    with pytest.raises(capi.MibcNotSupported, match="negation"):
        ops.rms_norm(im)
    y = ops.rms_norm(im.resolve_neg().clone(), eps=0.0)
    assert (y == -1).all()


@gpu
@pytest.mark.parametrize("which", ["norm", "sum", "rope", "keys", "attention"])
def test_written_tensors_get_a_new_version(which):
    # a tensor that a backward pass still needs is overwritten: autograd has to notice
    x, f = torch.rand((1, 4, 2, 64), device="cuda").half() + 0.5, FREQS.cuda()
    a = torch.rand_like(x).requires_grad_()
    y = (a * x).sum()                     # keeps x
    before = x._version
    with torch.no_grad():
        {"norm": lambda: ops.rms_norm(x, out=x), "sum": lambda: ops.rms_norm(x.clone(), sum_out=x), "rope": lambda: ops.rope(x, freqs=f, out=x),
         "keys": lambda: ops.rope(x.clone(), x, freqs=f, out=(torch.empty_like(x), x)), "attention": lambda: ops.attention(x, x.clone(), x.clone(), out=x)}[which]()
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():          # tensors without versions stay usable
        z = torch.ones((2, 64), dtype=torch.float16, device="cuda")
        ops.rms_norm(z, out=z)


@gpu
@pytest.mark.filterwarnings("ignore")
def test_compiled_callers_get_the_same_results():
    x, f = torch.rand((1, 4, 2, 64), device="cuda").half(), FREQS.cuda()

    def layer(t):
        y = ops.rms_norm(t * 2)
        q, k = ops.rope(y, y + 1, freqs=f)
        return ops.attention(q, k, y) + 1

    assert torch.equal(torch.compile(layer, backend="eager")(x), layer(x))


@gpu
def test_operators_work_beside_tangents():
    # a dual level that concerns none of the operands: whole numbers, codes and tensors without versions among them
    x, f, p = torch.ones((1, 4, 2, 64), dtype=torch.float16, device="cuda"), FREQS.cuda(), torch.arange(4, device="cuda", dtype=torch.int32)
    want = ops.rms_norm(x, quant="int8")[0], ops.rope(x, freqs=f, positions=p), ops.attention(x, x, x, k_len=p[3:])
    with fwd.dual_level():
        codes = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        got = ops.rms_norm(x, quant="int8", out=codes)[0], ops.rope(x, freqs=f, positions=p), ops.attention(x, x, x, k_len=p[3:])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.inference_mode(), fwd.dual_level():
        y = torch.ones_like(x)
        assert torch.equal(ops.rope(y, freqs=f, positions=p, out=y), want[1])
