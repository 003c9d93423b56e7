"""What the decoding strategies refuse before anything reaches a GPU, through plans that were created offline."""
import ctypes as C

import pytest

from fastforwardattention_b200 import capi

SMS, SMEM_CTA, SMEM_SM = 148, 232448, 233472
P16, ODD = C.c_void_p(4096), C.c_void_p(4100)
ARG, RANGE, WORKSPACE = -4, -3, -6


@pytest.fixture
def plan():
    L = capi.lib()
    p = C.c_void_p()
    capi.check(L.ffa_plan_create_offline(capi.BF16, 4, 8, 128, 4096, 0, SMS, SMEM_CTA, SMEM_SM, C.byref(p)))
    yield L, p
    L.ffa_plan_destroy(p)


def tree_args(p, **kw):
    a = dict(plan=p, q=P16, k=P16, v=P16, kc=P16, vc=P16, tree=P16, per_sample=0, groups=1, tokens=8, out=P16, scale=1.0, t=100, lengths=None,
             right=1, table=None, max_pages=0, page_rows=0, scratch=None, bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(plan=None), ARG), (dict(q=None), ARG), (dict(tree=None), ARG), (dict(out=ODD), ARG), (dict(kc=ODD), ARG),
    (dict(groups=0), RANGE), (dict(tokens=0), RANGE), (dict(tokens=-3), RANGE), (dict(groups=3, tokens=400), RANGE), (dict(tokens=1 << 30, groups=4), RANGE),
    (dict(t=-1), RANGE), (dict(t=4096), RANGE), (dict(t=4089), RANGE), (dict(right=0), ARG),
    (dict(table=P16, max_pages=4, page_rows=100), RANGE), (dict(table=P16, max_pages=4, page_rows=128), RANGE),
    (dict(), ARG)])   # the last one is in order, but this plan cannot launch
def test_tree_attention_refusals(plan, kw, code):
    L, p = plan
    assert L.ffa_tree_attention(*tree_args(p, **kw)) == code, L.ffa_last_error()


@pytest.mark.parametrize("kw,code", [(dict(plan=None), ARG), (dict(kc=None), ARG), (dict(vc=ODD), ARG), (dict(path=None), ARG), (dict(n=-1), RANGE),
                                     (dict(n=1025), RANGE), (dict(t=4096), RANGE), (dict(), ARG)])
def test_tree_accept_refusals(plan, kw, code):
    L, p = plan
    a = dict(plan=p, kc=P16, vc=P16, path=P16, n=4, t=100, lengths=None, table=None, max_pages=0, page_rows=0, stream=None)
    a.update(kw)
    assert L.ffa_tree_accept(*a.values()) == code, L.ffa_last_error()


def test_tree_scratch(plan):
    L, p = plan
    n = C.c_size_t(7)
    assert L.ffa_tree_scratch_bytes(p, 1, 8, 4000, C.byref(n)) == 0 and n.value > 0 and n.value % 4 == 0
    assert L.ffa_tree_scratch_bytes(p, 1, 8, 10, C.byref(n)) == 0 and n.value == 0   # a short cache is not split
    assert L.ffa_tree_scratch_bytes(p, 1, 8, 10, None) == ARG
    assert L.ffa_tree_scratch_bytes(p, 1, 2000, 10, C.byref(n)) == RANGE
    assert L.ffa_tree_scratch_bytes(None, 1, 8, 10, C.byref(n)) == ARG
