"""What the serving operators refuse, on the CPU (fake tensors and the C ABI
before any launch)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from compiler import runtime
from compiler.runtime import cabi
from test_serving_host import ARG, attn_args

runtime.load()


def calls():
    """Per operator: arguments, and which of them are floating tensors."""
    def t(*shape, dtype=torch.bfloat16):
        return torch.empty(*shape, dtype=dtype, device="cuda")
    cache = t(4, 16, 2, 64), t(4, 16, 2, 64)
    ints = t(3, dtype=torch.int32)
    return {"add_rms_norm": (t(3, 256), t(3, 256), t(256), 1e-5),
            "add_rms_norm_quant": (t(3, 256), t(3, 256), t(256), 1e-5, 128),
            "rope_append": (t(3, 8, 64), t(3, 2, 64), t(3, 2, 64), t(9, 32), t(9, 32), ints, ints, *cache),
            "paged_attention": (t(3, 8, 64), *cache, t(2, 4, dtype=torch.int32), ints, ints[:2])}


FLOATS = {"add_rms_norm": 3, "add_rms_norm_quant": 3, "rope_append": 9, "paged_attention": 3}
CASES = [(op, i) for op, n in FLOATS.items() for i in range(n) if not (op == "rope_append" and i in (5, 6))]


@pytest.mark.parametrize("op,at", CASES)
def test_inputs_with_a_tangent_are_refused(op, at):
    """No derivative is defined in forward mode either: a tangent would be
    dropped without a word."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    f = getattr(torch.ops.b200, op)
    with FakeTensorMode(allow_non_fake_inputs=True), forward_ad.dual_level():
        args = list(calls()[op])
        with torch.no_grad():
            f(*args)
        args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        for grad in (True, False):  # no_grad does not switch forward mode off
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="no gradient is defined"):
                f(*args)


@pytest.mark.parametrize("op", list(FLOATS))
def test_functional_jvp_is_refused(op):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode(allow_non_fake_inputs=True):
        first, *rest = calls()[op]
        f = lambda x: getattr(torch.ops.b200, op)(x, *rest)  # noqa: E731
        with pytest.raises(RuntimeError, match="no gradient is defined"):
            torch.func.jvp(f, (first,), (torch.ones_like(first),))


@pytest.mark.parametrize("kw", [dict(scale=-1.0), dict(scale=-1e-30), dict(scale=float("-inf")), dict(softcap=3e38)])
def test_paged_attention_refuses_scales_and_caps_it_cannot_apply(kw):
    """A negative scale is not the default; a cap whose base-2 form overflows."""
    assert cabi.library().b200k_paged_attention(ctypes.byref(attn_args(**kw)), None) == ARG


@pytest.mark.gpu
def test_a_scale_that_cannot_be_applied_is_refused_by_the_operator():
    """Negative, not a number, or below what fp32 holds (which reads as 0, the default)."""
    import serving_reference as ref

    x = ref.paged_inputs([1, 2], [40, 20], 8, 2, 64, 16, torch.bfloat16)
    op = torch.ops.b200.paged_attention
    for scale, cap in ((-1.0, 0.0), (-0.1, 30.0), (float("nan"), 0.0), (1e-60, 0.0), (0.1, 1e-60), (0.1, 3e38), (0.1, 1e60)):
        with pytest.raises(RuntimeError):
            op(*x, scale, cap)
    assert torch.equal(op(*x, -0.0), op(*x)) and torch.equal(op(*x, 0.125, 0.0), op(*x))


@pytest.mark.gpu
def test_one_tensor_as_both_caches_is_refused():
    """Keys and values would be written to the same places."""
    from test_gpu_rope_append import make

    *args, kc, vc = make(8, 4, 2, 64, 64, 16, torch.bfloat16)
    for same in (kc, kc.view_as(kc)):
        with pytest.raises(RuntimeError, match="same memory"):
            torch.ops.b200.rope_append(*args, kc, same)
    torch.ops.b200.rope_append(*args, kc, vc)
    torch.ops.b200.rope_append(*args, kc[:0], kc[:0])  # nothing to write, slots past the cache
    assert runtime.gemm_status() == 9
