"""What rotary_embedding refuses when a program is built; nothing runs."""
import pytest

from cinn_amd import _lib
from cinn_amd.common import Float, Int
from cinn_amd.frontend import NetBuilder

from helpers import compile_only


def made(x=(4, 3, 32), positions=(4,), x_type=None, p_type=None, **options):
    b = NetBuilder("rotary")
    X = b.create_input(x_type or Float(16), list(x), "x")
    P = b.create_input(p_type or Int(32), list(positions), "positions")
    return b, b.rotary_embedding(X, P, **options)


@pytest.mark.parametrize("case", [
    dict(x=(32,), positions=(1,)), dict(positions=(5,)), dict(positions=(4, 3)), dict(heads=4), dict(heads=-1),
    dict(rotary_dim=31), dict(rotary_dim=34), dict(x=(4, 3, 33)), dict(x=(4, 3, 600)), dict(theta=0.0),
    dict(theta=float("nan")), dict(factor=-1.0), dict(original_length=-1), dict(original_length=10, low=4.0, high=4.0),
    dict(x_type=Float(64)), dict(x_type=Int(32)), dict(p_type=Float(32)), dict(p_type=Int(8))])
def test_refused(case):
    with pytest.raises(_lib.CinnError):
        made(**case)


def test_tensors_of_many_elements_are_refused():
    b, y = made((1 << 20, 32, 128), (1 << 20,), heads=1)
    with pytest.raises(_lib.CinnError, match="2\\^31"):
        compile_only(b, [y])


@pytest.mark.parametrize("case", [dict(), dict(x=(4, 3, 600), rotary_dim=512), dict(x=(2, 2, 3, 33), positions=(2, 2), rotary_dim=32),
                                  dict(x=(3, 32), positions=(1,)), dict(heads=2, p_type=Int(64))])
def test_one_call(case):
    b, y = made(**case)
    comp = compile_only(b, [y])
    assert comp.num_instructions() == 1
