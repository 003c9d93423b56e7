"""The host's side of paged sequences: which paths of a drafted tree they take.  The engine is a stand-in that records its calls."""
import types

import pytest
import torch

import fastforwardattention_b200 as pkg
from fastforwardattention_b200 import paged


class Engine:
    def __init__(self, *args):
        self.accepted = []

    def attention_per_sample(self, q, *args, **kw):
        return q

    def tree_attention_per_sample(self, q, k, v, tree, *args, **kw):
        if tree.shape[-1] != k.shape[2]:
            raise RuntimeError("tree")
        return q

    def tree_accept_per_sample(self, path, table, rows):
        self.accepted.append(path.tolist())


@pytest.fixture
def seqs(monkeypatch):
    monkeypatch.setattr(pkg, "_extension", lambda: types.SimpleNamespace(PagedEngine=Engine))
    pool = paged.PagePool(8, 2, 64, torch.float16, "cpu", page_rows=128)
    K = torch.zeros(2, 2, 200, 64, dtype=torch.float16)
    return paged.PagedFastForwardAttn(pool, K, K, 384, lengths=[200, 120])


def draft(seqs, T, tree=None):
    x = torch.zeros(2, 2, T, 64, dtype=torch.float16)
    return seqs.tree_attention(x, x, x, torch.ones(T, T, dtype=torch.bool) if tree is None else tree, 0.1)


def test_a_path_may_only_name_drafted_tokens(seqs):
    draft(seqs, 5)
    for path in ([[5], []], [[0, 7], [1]], [[], [0, 1, 2, 3, 4, 5]]):   # their rows lie in pages that exist, but nothing was drafted there
        with pytest.raises(ValueError, match="was not drafted"):
            seqs.tree_accept(path)
    assert seqs.lengths == [200, 120] and seqs.engine.accepted == []
    seqs.tree_accept([[0, 4], [2]])
    assert seqs.lengths == [202, 121] and seqs.rows.tolist() == [202, 121] and seqs.engine.accepted == [[[0, 4], [2, -1]]]


def test_a_tree_is_accepted_once_and_before_anything_else(seqs):
    with pytest.raises(ValueError, match="was not drafted"):
        seqs.tree_accept([[0], [0]])
    draft(seqs, 5)
    seqs.tree_accept([[1], [0]])
    with pytest.raises(ValueError, match="was not drafted"):   # the rows have moved
        seqs.tree_accept([[2], []])
    draft(seqs, 5)
    x = torch.zeros(2, 2, 1, 64, dtype=torch.float16)
    seqs.attention(x, x, x, 0.1)                                # appends over the first drafted row
    with pytest.raises(ValueError, match="was not drafted"):
        seqs.tree_accept([[1], [0]])
    seqs.tree_accept([[], []])                                  # nothing kept is always in order
    draft(seqs, 3)
    with pytest.raises(RuntimeError):                           # a refused call writes nothing: the tree before it stands
        draft(seqs, 4, torch.ones(2, 2, dtype=torch.bool))
    seqs.tree_accept([[2], []])
    assert seqs.lengths == [203, 122]


def test_a_released_sequence_has_no_tree(seqs):
    draft(seqs, 5)
    seqs.release()
    with pytest.raises(ValueError, match="was not drafted"):
        seqs.tree_accept([[0], []])
