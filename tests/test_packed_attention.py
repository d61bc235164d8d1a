"""What packed_attention refuses when a program is built or compiled; nothing runs."""
import pytest

from cinn_amd import _lib
from cinn_amd.common import Float, Int
from cinn_amd.frontend import NetBuilder

from helpers import compile_only


def made(q=(40, 8, 64), k=(40, 2, 64), v=(40, 2, 64), offsets=(4,), q_type=None, v_type=None, o_type=None, **options):
    b = NetBuilder("packed")
    Q = b.create_input(q_type or Float(16), list(q), "q")
    K = b.create_input(q_type or Float(16), list(k), "k")
    V = b.create_input(v_type or q_type or Float(16), list(v), "v")
    O = b.create_input(o_type or Int(32), list(offsets), "offsets")
    return b, b.packed_attention(Q, K, V, O, **options)


@pytest.mark.parametrize("case", [
    dict(q=(40, 512)), dict(k=(41, 2, 64)), dict(v=(40, 2, 32)), dict(k=(40, 3, 64), v=(40, 3, 64)), dict(v=(40, 1, 64)),
    dict(offsets=(1,)), dict(offsets=(2, 2)), dict(q=(40, 8, 136), k=(40, 2, 136), v=(40, 2, 136)), dict(heads=9), dict(heads=8, q_head=1),
    dict(kv_heads=3), dict(k_head=-1), dict(k_head=2), dict(v_head=1), dict(heads=-2), dict(heads=3), dict(scale=float("nan")),
    dict(q_type=Float(64)), dict(v_type=Float(32)), dict(o_type=Int(64)), dict(o_type=Float(32))])
def test_refused(case):
    with pytest.raises(_lib.CinnError):
        made(**case)


@pytest.mark.parametrize("kind,d", [(Float(16), 60), (Float(16), 4), (Float(32), 6)])
def test_rows_of_odd_bytes_are_refused(kind, d):
    b, o = made((9, 2, d), (9, 1, d), (9, 1, d), q_type=kind)
    with pytest.raises(_lib.CinnError, match="16-byte"):
        compile_only(b, [o])


@pytest.mark.parametrize("case", [
    dict(q=(4, 1 << 18, 128), k=(4, 1, 128), v=(4, 1, 128)), dict(q=(4, 1, 128), k=(4, 1 << 18, 128), v=(4, 1, 128), kv_heads=1),
    dict(q=(1 << 22, 8, 128), k=(1 << 22, 1, 128), v=(1 << 22, 1, 128)), dict(offsets=(1 << 23,)), dict(q=(1 << 28, 1, 8), k=(1 << 28, 1, 8), v=(1 << 28, 1, 8))])
def test_sizes_that_its_offsets_do_not_hold_are_refused(case):
    b, o = made(**case)
    with pytest.raises(_lib.CinnError, match="32 MiB|2\\^31|too many"):
        compile_only(b, [o])


@pytest.mark.parametrize("case", [dict(), dict(heads=4, kv_heads=1, q_head=3, k_head=1, v_head=0), dict(k_head=1, v_head=1), dict(offsets=(2,))])
def test_one_call(case):
    b, o = made(**case)
    comp = compile_only(b, [o])
    assert comp.num_instructions() == 1 and o.shape() == [40, case.get("heads", 8), 64]
