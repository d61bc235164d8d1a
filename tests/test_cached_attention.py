"""What cached_attention refuses when a program is built or compiled; nothing runs."""
import pytest

from cinn_amd import _lib
from cinn_amd.common import Float, Int
from cinn_amd.frontend import NetBuilder

from helpers import compile_only


def made(q=(3, 5, 8, 64), k=(3, 5, 2, 64), v=(3, 5, 2, 64), k_pages=(7, 16, 2, 64), v_pages=None, table=(3, 4), lengths=(3,), parents=(3, 5),
         q_type=None, page_type=None, i_type=None, **options):
    b = NetBuilder("cached")
    kind, whole = q_type or Float(16), i_type or Int(32)
    Q, K, V = (b.create_input(kind, list(shape), n) for n, shape in (("q", q), ("k", k), ("v", v)))
    KP, VP = (b.create_input(page_type or kind, list(shape), n) for n, shape in (("kp", k_pages), ("vp", v_pages or k_pages)))
    T, L = b.create_input(whole, list(table), "table"), b.create_input(whole, list(lengths), "lengths")
    P = b.create_input(whole, list(parents), "parents") if parents else None
    return b, b.cached_attention(Q, K, V, KP, VP, T, L, parents=P, **options)


@pytest.mark.parametrize("case", [
    dict(q=(3, 40, 64)), dict(k=(3, 4, 2, 64)), dict(v=(3, 5, 2, 32)), dict(k=(3, 5, 3, 64), v=(3, 5, 3, 64)), dict(k_pages=(7, 2, 16, 64)),
    dict(k_pages=(7, 16, 2, 32)), dict(v_pages=(8, 16, 2, 64)), dict(k_pages=(7, 32, 64)), dict(table=(4, 4)), dict(table=(3,)),
    dict(lengths=(4,)), dict(lengths=(3, 1)), dict(parents=(3, 4)), dict(parents=(5,)), dict(page_layout="heads"),
    dict(page_layout="head_row"), dict(q_type=Float(64)), dict(page_type=Float(32)), dict(i_type=Int(64)), dict(heads=9), dict(kv_heads=1),
    dict(k_head=1), dict(q=(3, 65, 8, 64), k=(3, 65, 2, 64), v=(3, 65, 2, 64), parents=(3, 65)), dict(table=(3, 1 << 26)),
    dict(q=(3, 5, 8, 136), k=(3, 5, 2, 136), v=(3, 5, 2, 136), k_pages=(7, 16, 2, 136)), dict(scale=float("inf"))])
def test_refused(case):
    with pytest.raises(_lib.CinnError):
        made(**case)


def test_rows_of_odd_bytes_are_refused():
    b, o = made((3, 5, 8, 60), (3, 5, 2, 60), (3, 5, 2, 60), (7, 16, 2, 60))
    with pytest.raises(_lib.CinnError, match="16-byte"):
        compile_only(b, [o])


@pytest.mark.parametrize("case", [
    dict(q=(3, 5, 1 << 18, 128), k=(3, 5, 2, 128), v=(3, 5, 2, 128), k_pages=(7, 16, 2, 128)),
    dict(q=(3, 5, 2, 128), k=(3, 5, 1 << 18, 128), v=(3, 5, 2, 128), k_pages=(7, 16, 2, 128), kv_heads=2),
    dict(q=(1 << 17, 1, 32, 64), k=(1 << 17, 1, 2, 64), v=(1 << 17, 1, 2, 64), table=(1 << 17, 4), lengths=(1 << 17,), parents=None),
    dict(q=(1 << 16, 1, 8, 64), k=(1 << 16, 1, 2, 64), v=(1 << 16, 1, 2, 64), table=(1 << 16, 1 << 15), lengths=(1 << 16,), parents=None),
    dict(k_pages=(1 << 30, 16, 2, 64))])
def test_sizes_that_its_offsets_do_not_hold_are_refused(case):
    b, o = made(**case)
    with pytest.raises(_lib.CinnError, match="32 MiB|2\\^31|2\\^40|too many"):
        compile_only(b, [o])


@pytest.mark.parametrize("case", [dict(), dict(parents=None), dict(k_pages=(7, 2, 16, 64), page_layout="head_row"),
                                  dict(heads=4, q_head=2, kv_heads=2, v_head=0), dict(k_pages=(1, 1, 2, 64), table=(3, 1))])
def test_one_call(case):
    b, o = made(**case)
    comp = compile_only(b, [o])
    assert comp.num_instructions() == 1 and o.shape() == [3, 5, case.get("heads", 8), 64]
