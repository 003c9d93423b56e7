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
             right=1, table=None, max_pages=0, page_rows=0, pool=64, scratch=None, bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(plan=None), ARG), (dict(q=None), ARG), (dict(tree=None), ARG), (dict(out=ODD), ARG), (dict(kc=ODD), ARG),
    (dict(groups=0), RANGE), (dict(tokens=0), RANGE), (dict(tokens=-3), RANGE), (dict(groups=3, tokens=400), RANGE), (dict(tokens=1 << 30, groups=4), RANGE),
    (dict(t=-1), RANGE), (dict(t=4096), RANGE), (dict(t=4089), RANGE), (dict(right=0), ARG),
    (dict(table=P16, max_pages=4, page_rows=100), RANGE), (dict(table=P16, max_pages=4, page_rows=128), RANGE),
    (dict(table=P16, max_pages=32, page_rows=128, pool=0), RANGE), (dict(table=P16, max_pages=32, page_rows=128, pool=1 << 30), RANGE),
    (dict(scale=float("nan")), RANGE), (dict(scale=float("inf")), RANGE),
    (dict(), ARG)])   # the last one is in order, but this plan cannot launch
def test_tree_attention_refusals(plan, kw, code):
    L, p = plan
    assert L.ffa_tree_attention(*tree_args(p, **kw)) == code, L.ffa_last_error()


@pytest.mark.parametrize("kw,code", [(dict(plan=None), ARG), (dict(kc=None), ARG), (dict(vc=ODD), ARG), (dict(path=None), ARG), (dict(n=-1), RANGE),
                                     (dict(n=1025), RANGE), (dict(t=4096), RANGE), (dict(), ARG)])
def test_tree_accept_refusals(plan, kw, code):
    L, p = plan
    a = dict(plan=p, kc=P16, vc=P16, path=P16, n=4, t=100, lengths=None, table=None, max_pages=0, page_rows=0, pool=64, stream=None)
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


@pytest.mark.parametrize("kw,code", [(dict(plan=None), ARG), (dict(kc=ODD), ARG), (dict(w=None), ARG), (dict(pos=None), ARG), (dict(rows=None), ARG), (dict(kept=None), ARG),
                                     (dict(most=-1), RANGE), (dict(most=4097), RANGE), (dict(keep=0), RANGE), (dict(keep=4097), RANGE), (dict(recent=-1), RANGE),
                                     (dict(recent=90, first=11), RANGE), (dict(recent=2 ** 31 - 1, first=2 ** 31 - 1), RANGE), (dict(), ARG)])
def test_evict_refusals(plan, kw, code):
    L, p = plan
    a = dict(plan=p, kc=P16, vc=P16, w=P16, pos=P16, rows=P16, most=4096, keep=100, recent=10, first=4, kept=P16, stream=None)
    a.update(kw)
    assert L.ffa_evict(*a.values()) == code, L.ffa_last_error()


def test_evict_refuses_more_rows_than_a_selection_holds():
    L = capi.lib()
    p = C.c_void_p()
    capi.check(L.ffa_plan_create_offline(capi.F16, 1, 1, 64, 1 << 20, 0, SMS, SMEM_CTA, SMEM_SM, C.byref(p)))
    assert L.ffa_evict(p, P16, P16, P16, P16, P16, (1 << 19) + 1, 100, 0, 0, P16, None) == RANGE
    L.ffa_plan_destroy(p)


def test_accumulate_refusals(plan):
    L, p = plan
    assert L.ffa_attention_accumulate(None, P16, P16, P16, P16, P16, P16, 1.0, 5, None, P16, None, None, None) == ARG
    assert L.ffa_attention_accumulate(p, P16, P16, P16, P16, P16, P16, 1.0, 5, None, None, None, None, None) == ARG
    assert L.ffa_attention_accumulate(p, P16, P16, P16, P16, P16, P16, 1.0, 5, None, P16, None, None, None) == ARG   # offline


@pytest.mark.parametrize("kw,code", [(dict(dtype=3), -1), (dict(batch=0), RANGE), (dict(vocab=0), RANGE), (dict(beams=0), RANGE), (dict(beams=33), RANGE), (dict(num=0), RANGE),
                                     (dict(num=65), RANGE), (dict(stride=99), RANGE), (dict(pad=-1), RANGE), (dict(pad=100), RANGE), (dict(logits=None), ARG),
                                     (dict(logits=C.c_void_p(4097)), ARG), (dict(scores=None), ARG), (dict(tokens=None), ARG),
                                     (dict(beams=32, vocab=1 << 27, stride=1 << 27), RANGE)])
def test_beam_select_refusals(kw, code):
    a = dict(dtype=capi.F16, batch=2, beams=4, vocab=100, stride=100, logits=P16, scores=P16, finished=None, pad=0, num=8, best=P16, parents=P16,
             tokens=P16, stream=None)
    a.update(kw)
    L = capi.lib()
    assert L.ffa_beam_select(*a.values()) == code, L.ffa_last_error()


@pytest.mark.parametrize("kw,code", [(dict(plan=None), ARG), (dict(kc=None), ARG), (dict(vc=ODD), ARG), (dict(parents=None), ARG), (dict(beams=0), RANGE), (dict(beams=3), RANGE),
                                     (dict(beams=64), RANGE), (dict(first=-1), RANGE), (dict(first=51), RANGE), (dict(rows=4097), RANGE), (dict(), ARG)])
def test_reorder_refusals(plan, kw, code):
    L, p = plan
    a = dict(plan=p, kc=P16, vc=P16, parents=P16, beams=4, first=0, rows=50, stream=None)
    a.update(kw)
    assert L.ffa_cache_reorder(*a.values()) == code, L.ffa_last_error()


@pytest.mark.parametrize("T,resident", [(20, 3), (32, 3), (40, 1), (64, 1), (100, 1)])
def test_fp32_trees_are_split_for_the_ctas_that_their_registers_allow(T, resident):
    """Head_dim 64, 17 query rows and more: 75 registers for each of 256 threads with two rows to a thread, 134 with four.  A split over more CTAs than
    are resident would run in waves."""
    L = capi.lib()
    p, n = C.c_void_p(), C.c_size_t()
    capi.check(L.ffa_plan_create_offline(capi.F32, 1, 32, 64, 5000, 0, SMS, SMEM_CTA, SMEM_SM, C.byref(p)))
    capi.check(L.ffa_tree_scratch_bytes(p, 1, T, 4000, C.byref(n)))
    tile = 32 if T <= 32 else 64
    tiles, rows = -(-T // tile), min(T, tile)
    splits = n.value // (32 * tiles * rows * (64 + 4) * 4)
    assert splits > 1 and 32 * tiles * splits <= SMS * resident
    L.ffa_plan_destroy(p)
