"""Compiled decode steps whose caches are parts of larger tensors: K and V as
halves of one tensor, indexed in the graph or passed as two views, and the
layers' caches stacked in one tensor.  Appends to those stay functional (the
tensor is copied); results and caches equal eager ones, op by op and replayed,
and places outside the appended slots keep their contents."""
import pytest
import torch

from compiler import runtime

pytestmark = pytest.mark.gpu
runtime.load()
LAYERS = 4


def stacks(layout, store):
    """Per layer K and V of `store`, by what the layout calls a cache."""
    if layout == "stacked":  # [layers, pages, ...] for K and for V
        return [(store[0][i], store[1][i]) for i in range(LAYERS)]
    return [(both[:, 0], both[:, 1]) for both in store]


@pytest.mark.parametrize("layout", ["halves in the graph", "halves passed", "stacked"])
@pytest.mark.parametrize("pages", [7, 9000])  # outputs below and above what a replay clones
def test_equal_to_eager(layout, pages):
    from compiler.backend import custom_backend
    from test_inplace_append import _model

    step, model = _model(LAYERS)
    shape = (pages, step.PAGE, step.HKV, step.D)
    bf = dict(device="cuda", dtype=torch.bfloat16)
    if layout == "stacked":
        mine = [torch.randn(LAYERS, *shape, **bf) for _ in range(2)]
    else:
        mine = [torch.randn(pages, 2, *shape[1:], **bf) for _ in range(LAYERS)]
    eager = [t.clone() for t in mine]

    if layout == "halves passed":
        f = lambda x, cos, sin, store, index: model(x, cos, sin, store, index)  # noqa: E731
        give = lambda store: stacks(layout, store)  # noqa: E731
    else:
        f = lambda x, cos, sin, store, index: model(x, cos, sin, stacks(layout, store), index)  # noqa: E731
        give = lambda store: store  # noqa: E731
    torch._dynamo.reset()
    compiled = torch.compile(f, backend=custom_backend, dynamic=False)
    cos, sin = (torch.randn(64, step.D // 2, device="cuda") for _ in range(2))
    index = step.Cache([40, 40])  # its page table alone
    with torch.no_grad():
        for i in range(5):
            pos, slots, _, _, table, q_start, kv_len = index.step([(i, i + 1)] * 2)
            x = torch.randn(2, step.DIM, **bf)
            rest = (pos, slots, table, q_start, kv_len)
            got, want = compiled(x, cos, sin, give(mine), rest), f(x, cos, sin, give(eager), rest)
            assert torch.equal(got, want)
            for a, b in zip(mine, eager):
                assert torch.equal(a, b)
    assert runtime.gemm_status() == 0
