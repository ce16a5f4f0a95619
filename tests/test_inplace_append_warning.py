"""An append that a compiled graph does not keep in place is warned of: it copies
the tensor that holds its cache."""
import warnings

import pytest

from compiler.optimization.inplace_append import inplace_append
from test_inplace_append import graph


@pytest.mark.parametrize("steps,returns", [
    (["append", "attend first state"], ("kc", "vc")), (["view argument", "append"], ("kc", "vc")),
    (["append"], ("kc", "vc", "first"))])
def test_warned_of(steps, returns):
    with pytest.warns(UserWarning, match="1 b200::rope_append of a compiled graph copy"):
        inplace_append(graph(steps, returns))


@pytest.mark.parametrize("steps", [["append", "attend"], ["append", "attend", "append"], ["attend"]])
def test_not_warned_of(steps):
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        inplace_append(graph(steps))
