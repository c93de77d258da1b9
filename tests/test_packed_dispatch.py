"""Calls of the packed operators go through torch's dispatcher: whatever watches or records torch's ops (dispatch modes,
tensor subclasses, traces, vmap, lazy negation) sees them as the ops they are."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from chess_transformer_b200 import ops
from chess_transformer_b200.build import build

NAMES = ["packed_attention", "cached_attention", "adapter_linear", "int8_adapter_linear"]


def calls(device, seed=0):
    """name -> (function of one floating tensor, that tensor): a small call of each operator."""
    g = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g).half().to(device)  # noqa: E731
    whole = lambda *shape: torch.randint(-9, 10, shape, generator=g, dtype=torch.int8).to(device)  # noqa: E731
    index = lambda *values: torch.tensor(values, dtype=torch.int32, device=device)  # noqa: E731
    q, k, v, cache = normal(5, 4, 64), normal(9, 2, 64), normal(9, 2, 64), normal(5, 7, 2, 64)
    x, weight, down, up, at, ids = normal(5, 64), normal(24, 64), normal(2, 8, 64), normal(2, 24, 8), index(0, 2, 5), index(1, 0)
    x8, weight8, w_scale = whole(5, 64), whole(24, 64), torch.rand(24, generator=g).to(device)
    return {
        "packed_attention": (lambda t: ops.packed_attention(t, k, v, at, index(0, 4, 9)), q),
        "cached_attention": (lambda t: ops.cached_attention(t, cache, cache, index(7, 0, 3, 1, 6)), q),
        "adapter_linear": (lambda t: ops.adapter_linear(t, weight, None, None, down, up, at, ids), x),
        "int8_adapter_linear": (lambda t: ops.int8_adapter_linear(x8, t, weight8, w_scale, None, None, down, up, at, ids), torch.rand(5, generator=g).to(device)),
    }


class Seen(TorchDispatchMode):
    """Notes the fry ops and answers them with zeros, without running them."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, function, types, args=(), kwargs=None):
        if function.namespace != "fry":
            return function(*args, **(kwargs or {}))
        self.names.append(function._schema.name.removeprefix("fry::"))
        return torch.zeros(1)


@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_the_op(name):
    call, tensor = calls("cpu")[name]
    with Seen() as seen:
        call(tensor)
    assert seen.names == [name]


class Tagged(torch.Tensor):
    names = []

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype)

    @classmethod
    def __torch_dispatch__(cls, function, types, args=(), kwargs=None):
        cls.names.append(function._schema.name)
        return torch.zeros(1)


def test_a_subclass_sees_the_op_wherever_it_is_an_operand():
    Tagged.names.clear()
    q, at = torch.zeros(3, 4, 64, dtype=torch.float16), torch.tensor([0, 3], dtype=torch.int32)
    ops.packed_attention(q, q, Tagged(q), at, at)
    ops.cached_attention(q, Tagged(q[None]), q[None], at)
    x, ids = torch.zeros(3, 64, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)
    ops.adapter_linear(x, x, None, None, Tagged(x[None]), x[None], at, ids)
    ops.int8_adapter_linear(x, x, Tagged(x), x, None, None, x[None], x[None], at, ids)
    assert Tagged.names == [f"fry::{name}" for name in NAMES]


@pytest.mark.parametrize("name", NAMES)
def test_fake_tensors_have_the_answers_shape(name):
    with FakeTensorMode():
        call, tensor = calls("cpu")[name]
        out = call(tensor)
    assert out.shape == ((5, 4, 64) if "attention" in name else (5, 24)) and out.dtype == torch.float16


@pytest.fixture(scope="module")
def gpu():
    build()
    return "cuda"


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_traced_call_answers_new_inputs(gpu, name):
    call, tensor = calls(gpu)[name]
    other = tensor.flip(0) * 0.5
    for traced in (torch.jit.trace(call, (tensor,)), make_fx(call)(tensor)):
        assert torch.equal(traced(other), call(other))
        assert torch.equal(traced(tensor), call(tensor))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_vmap_is_the_calls_one_by_one(gpu, name):
    call, tensor = calls(gpu)[name]
    batch = torch.stack([tensor, tensor.flip(0), tensor * 0.25])
    assert torch.equal(torch.func.vmap(call)(batch), torch.stack([call(t) for t in batch]))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES[:3])
def test_a_lazily_negated_operand_counts_as_negated(gpu, name):
    call, tensor = calls(gpu)[name]
    lazy = torch.view_as_complex(torch.stack([torch.zeros_like(tensor), tensor], -1)).conj().imag
    assert lazy.is_neg() and torch.equal(lazy, -tensor)
    assert torch.equal(call(lazy), call(-tensor))


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_backward_pass_is_refused(gpu, name):
    call, tensor = calls(gpu)[name]
    out = call(tensor.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no autograd formula"):
        out.sum().backward()
