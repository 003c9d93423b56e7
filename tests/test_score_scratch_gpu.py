"""The score scratch comes when a step first asks for it; graphs recorded before, and the status word, are not touched by that."""
import pytest
import torch

pytestmark = pytest.mark.gpu

B, H, D, L, n = 1, 4, 64, 3000, 2900   # long enough that a pair's parts are merged through the workspace


class Contiguous:
    def __init__(self):
        from fastforwardattention_b200 import FastForwardAttn

        g = torch.Generator("cuda").manual_seed(1)
        kc, vc = (torch.randn(B, H, L, D, generator=g, device="cuda").half() for _ in range(2))
        self.engine = FastForwardAttn.adopt(kc, vc)
        self.engine.set_cluster_merge(False)

    def step(self, q, rows, p=0.0, out=None):
        return self.engine.attention_per_sample(q, q, q, 0.1, rows, p, out=out)


class Paged:
    def __init__(self):
        from fastforwardattention_b200 import _extension

        g = torch.Generator("cuda").manual_seed(1)
        kp, vp = (torch.randn(23, H, 128, D, generator=g, device="cuda").half() for _ in range(2))
        self.engine = _extension().PagedEngine(kp, vp, B, 23)
        self.table = torch.arange(23, dtype=torch.int32, device="cuda")[None].contiguous()

    def step(self, q, rows, p=0.0, out=None):
        return self.engine.attention_per_sample(q, q, q, self.table, 0.1, rows, p, out=out)


def inputs():
    q = torch.randn(B, H, 1, D, device="cuda").half()
    return q, torch.full((B,), n, dtype=torch.int32, device="cuda")


def recorded(e, q, rows):
    want = e.step(q, rows)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        e.step(q, rows, out=out)
    return graph, out, want


@pytest.mark.parametrize("kind,first", [(Contiguous, "pruned"), (Paged, "pruned"), (Contiguous, "accumulating")])
def test_graphs_recorded_before_stay_valid(kind, first):
    e = kind()
    q, rows = inputs()
    graph, out, want = recorded(e, q, rows)
    if first == "pruned":
        e.step(q, rows, p=1e-3)
    else:
        w = torch.zeros(B, H, L, device="cuda")
        e.engine.attention_accumulate(q, q, q, 0.1, rows, w, torch.zeros(B, H, L, dtype=torch.int32, device="cuda"), rows)
    filler = [torch.full((1 << 18,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]   # takes freed memory, if there is any
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want) and torch.equal(e.step(q, rows), want)
    assert e.engine.device_status() == 0 and all((f == 7).all() for f in filler)


@pytest.mark.parametrize("kind", [Contiguous, Paged])
def test_status_bits_outlive_the_first_pruned_step(kind):
    e = kind()
    q, rows = inputs()
    graph, out, want = recorded(e, q, rows)
    rows.fill_(-1)
    e.step(q, rows)                              # a bit from before
    rows.fill_(n)
    e.step(q, rows, p=1e-3)
    assert e.engine.device_status() == 2 and e.engine.device_status() == 0
    rows.fill_(-1)
    graph.replay()                               # and one from a graph recorded before
    assert e.engine.device_status() == 2 and e.engine.device_status() == 0


def test_status_bits_outlive_growing():
    e = Contiguous()
    q, rows = inputs()
    e.step(q, rows.new_full((B,), -1))
    e.engine.grow(L + 128)
    assert e.engine.device_status() == 2 and e.engine.device_status() == 0
    e.step(q, rows, p=1e-3)
    assert e.engine.device_status() == 0


@pytest.mark.parametrize("kind", [Contiguous, Paged])
def test_the_first_pruned_step_is_not_captured(kind):
    e, twin = kind(), kind()
    q, rows = inputs()
    want = twin.step(q, rows, p=1e-3)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="outside of a graph capture"):
            e.step(q, rows, p=1e-3)
        e.step(q, rows, out=out)
    for _ in range(3):                           # refused, and nothing else changed
        assert torch.equal(e.step(q, rows, p=1e-3), want)
        graph.replay()
        assert torch.equal(out, e.step(q, rows))
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        e.step(q, rows, p=1e-3, out=out)
    out.zero_()
    second.replay()
    assert torch.equal(out, want) and e.engine.device_status() == 0
