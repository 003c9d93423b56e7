"""Decode steps that accumulate attention weights, and eviction down to a budget of rows, against their plain definitions."""
import math

import pytest
import torch

from oracle import decoding_oracle as D64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def engine(dt, B, H, D, L, seed=0):
    from fastforwardattention_b200 import FastForwardAttn

    g = torch.Generator("cuda").manual_seed(seed)
    kc, vc = (torch.randn(B, H, L, D, generator=g, device="cuda").to(dt) for _ in range(2))
    w = torch.rand(B, H, L, generator=g, device="cuda") ** 3
    pos = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, H, L).contiguous()
    return FastForwardAttn.adopt(kc, vc), kc, vc, w, pos, g


def check_evict(ffa, kc, vc, w, pos, rows, keep, recent, first, max_row=-1):
    caches, ww, pp, kept = D64.evict([kc, vc], w, pos, rows, keep, recent, first)
    got = ffa.evict(torch.tensor(rows, dtype=torch.int32, device="cuda"), w, pos, keep, recent=recent, first=first, max_row=max_row)
    assert torch.equal(got, kept)
    assert torch.equal(w.nan_to_num(-7.0), ww.nan_to_num(-7.0)) and torch.equal(pos, pp)
    assert torch.equal(kc, caches[0]) and torch.equal(vc, caches[1])
    assert ffa.device_status() == 0
    return got


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("B,H,n", [(1, 1, 0), (1, 2, 1), (2, 3, 37), (3, 2, 997), (1, 8, 1256), (2, 2, 5000)])
def test_step_accumulates(dt, D, B, H, n):
    ffa, kc, vc, w, pos, g = engine(dt, B, H, D, n + 3, seed=n + D)
    rows = [max(0, n - 5 * b) for b in range(B)]
    sl = torch.tensor(rows, dtype=torch.int32, device="cuda")
    seen = sl + 1000
    w[:, :, n:] = float("nan")   # what the new row's slot held is replaced, and nothing behind it is touched
    for step in range(2):
        q, k, v = (torch.randn(B, H, 1, D, generator=g, device="cuda").to(dt) for _ in range(3))
        want, bound, p, pb = D64.step_weights(q, k, v, kc, vc, D ** -0.5, rows)
        before, kb, vb = w.clone(), kc.clone(), vc.clone()
        out = ffa.attention_accumulate(q, k, v, D ** -0.5, sl, w, pos, seen, max_row=n)
        D64.assert_within(out, want, bound)
        for b, m in enumerate(rows):
            base = before[b, :, : m + 1].double()
            base[:, m] = 0
            total = base + p[b, :, : m + 1]
            assert ((w[b, :, : m + 1].double() - total).abs() <= pb[b, :, : m + 1] + D64.U * total).all()
            assert torch.equal(w[b, :, m + 1:].nan_to_num(-7.0), before[b, :, m + 1:].nan_to_num(-7.0))
            assert (pos[b, :, m] == m + 1000).all()
            kb[b, :, m], vb[b, :, m] = k[b, :, 0], v[b, :, 0]
            pos[b, :, m] = m
        assert torch.equal(kc, kb) and torch.equal(vc, vb)
        w.copy_(before)
    assert ffa.device_status() == 0


@pytest.mark.parametrize("dt", DTYPES)
def test_step_agrees_with_the_decode_step(dt):
    """The accumulating step's output next to `attention` on the same caches, in the sizes that take each cut of the work."""
    for B, H, D, n in [(1, 4, 64, 9), (1, 32, 64, 999), (4, 40, 64, 300), (20, 32, 128, 200)]:
        ffa, kc, vc, w, pos, g = engine(dt, B, H, D, n + 1, seed=n)
        q, k, v = (torch.randn(B, H, 1, D, generator=g, device="cuda").to(dt) for _ in range(3))
        sl = torch.full((B,), n, dtype=torch.int32, device="cuda")
        w.zero_()
        ffa.set_cluster_merge(False)   # the splits' partials through global memory, the last arriver adds all weights
        through_global = ffa.attention_accumulate(q, k, v, D ** -0.5, sl, w, pos, sl, max_row=n)
        wg = w.clone()
        ffa.set_cluster_merge(True)
        w.zero_()
        out = ffa.attention_accumulate(q, k, v, D ** -0.5, sl, w, pos, sl, max_row=n)
        _, bound, _, pb = D64.step_weights(q, k, v, kc, vc, D ** -0.5, [n] * B)
        assert ((out.double() - through_global.double()).abs() <= 2 * bound).all() and ((w.double() - wg.double()).abs() <= 2 * pb).all()
        ref = ffa.attention(q, k, v, D ** -0.5, n, 0)
        _, bound, _, pb = D64.step_weights(q, k, v, kc, vc, D ** -0.5, [n] * B)
        assert ((out.double() - ref.double()).abs() <= 2 * bound).all()   # each within its bound of the exact value
        assert ((w.double().sum(-1) - 1).abs() <= pb.sum(-1)).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("n,keep,recent,first", [(2, 1, 0, 0), (33, 32, 0, 0), (33, 32, 32, 0), (64, 32, 8, 4), (65, 64, 10, 0), (100, 37, 12, 5), (1000, 333, 100, 0),
                                                 (1000, 999, 250, 4), (1256, 1, 1, 0), (4100, 2048, 512, 4), (20000, 5001, 1, 3), (49152, 49151, 5, 1),
                                                 (49153, 49152, 5, 1), (49153, 49100, 0, 0)])
def test_evict(dt, D, n, keep, recent, first):
    ffa, kc, vc, w, pos, g = engine(dt, 2, 3, D, n + 2, seed=n + keep)
    # positions as an earlier eviction leaves them: distinct, in any order, with gaps
    pos.copy_((torch.rand(2, 3, n + 2, generator=g, device="cuda").argsort(-1) * 3).int())
    check_evict(ffa, kc, vc, w, pos, [n, n], keep, recent, first)


def test_evict_ties_extremes_and_protected_rows():
    dt, D, L = torch.float16, 64, 300
    for fill in ("ties", "two values", "zeros", "nan", "inf", "negative", "duplicates"):
        ffa, kc, vc, w, pos, g = engine(dt, 1, 4, D, L, seed=3)
        if fill == "ties":
            w.fill_(0.25)
        elif fill == "two values":
            w.copy_((w > 0.1).float())
        elif fill == "zeros":
            w.zero_()
            w[:, :, ::2] = -0.0
        elif fill == "nan":
            w[:, :, ::3] = float("nan")
        elif fill == "inf":
            w[:, :, ::5], w[:, :, 1::5] = float("inf"), -float("inf")
        elif fill == "negative":
            w.sub_(0.3)
        else:
            pos.fill_(7)   # all rows count as the newest: more rows protected than may stay
        check_evict(ffa, kc, vc, w, pos, [290], 101, 0 if fill != "duplicates" else 3, 0)


def test_evict_ragged_lengths_and_bounds():
    dt, D, L = torch.bfloat16, 128, 700
    ffa, kc, vc, w, pos, g = engine(dt, 6, 2, D, L, seed=5)
    kept = check_evict(ffa, kc, vc, w, pos, [700, 0, 100, 101, 99, 650], 100, 30, 4)
    assert (kept[1] == -1).all() and (kept[4, :, 99] == -1).all()
    kb, vb, wb = kc.clone(), vc.clone(), w.clone()
    got = ffa.evict(torch.tensor([300, 701, -1, 400, 299, 300], dtype=torch.int32, device="cuda"), w, pos, 100, max_row=300)
    assert ffa.device_status() == 2
    for b in (1, 2, 3):
        assert (got[b] == -1).all() and torch.equal(kc[b], kb[b]) and torch.equal(vc[b], vb[b]) and torch.equal(w[b], wb[b])
    assert (got[[0, 4, 5]] >= 0).all()


def test_evict_a_very_long_pair():
    """More rows than any shared-memory copy of the keys could hold, and the kernel's stated limit."""
    dt, D, n = torch.float16, 64, (1 << 19) - 5
    ffa, kc, vc, w, pos, g = engine(dt, 1, 1, D, n + 5, seed=7)
    rows = torch.tensor([n], dtype=torch.int32, device="cuda")
    kb, wb = kc.clone(), w.clone()
    keep = 200_003
    kept = ffa.evict(rows, w, pos, keep, recent=1000, first=4)[0, 0].long()
    assert ffa.device_status() == 0
    stay = torch.zeros(n, dtype=torch.bool, device="cuda")
    key = wb[0, 0, :n].clone()
    key[n - 1000:], key[:4] = math.inf, math.inf
    stay[torch.sort(key, descending=True, stable=True).indices[:keep]] = True
    assert torch.equal(torch.sort(kept).values, stay.nonzero().flatten())
    own = torch.arange(keep, device="cuda")
    assert torch.equal(kept[stay[:keep]], own[stay[:keep]])
    assert torch.equal(kept[~stay[:keep]], stay[keep:].nonzero().flatten() + keep)
    assert torch.equal(kc[0, 0, :keep], kb[0, 0, kept]) and torch.equal(w[0, 0, :keep], wb[0, 0, kept])
    assert torch.equal(kc[0, 0, keep:], kb[0, 0, keep:]) and torch.equal(pos[0, 0, :keep].long(), kept)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("slack", [1, 7])
def test_a_generation_under_a_budget(dt, slack):
    """EvictingFastForwardAttn against the plain loop: outputs within the steps' bounds while both keep the same rows."""
    from fastforwardattention_b200 import EvictingFastForwardAttn

    B, H, D, Lp, budget, recent, first = 3, 2, 64, 90, 48, 11, 2
    g = torch.Generator("cuda").manual_seed(11)
    K, V = (torch.randn(B, H, Lp, D, generator=g, device="cuda").to(dt) for _ in range(2))
    wp = torch.rand(B, H, Lp, generator=g, device="cuda")
    lens = [90, 30, 48]
    ffa = EvictingFastForwardAttn(K, V, budget, recent=recent, first=first, slack=slack, lengths=lens, weights=wp)
    L = ffa.engine.max_len
    kc, vc = (torch.zeros(B, H, L, D, dtype=dt, device="cuda") for _ in range(2))
    kc[:, :, :Lp], vc[:, :, :Lp] = K, V
    w = torch.zeros(B, H, L, device="cuda")
    w[:, :, :Lp] = wp
    pos = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, H, L).contiguous()
    off = torch.zeros(B, H, L, 1, dtype=torch.float64, device="cuda")   # how far the weights may be apart
    rows, seen = list(lens), list(lens)

    def cut():
        nonlocal kc, vc, w, pos, off, rows
        (kc, vc, off), w, pos, _ = D64.evict([kc, vc, off], w, pos, rows, budget, recent, first)
        rows = [min(n, budget) for n in rows]

    cut()
    for step in range(25):
        q, k, v = (torch.randn(B, H, 1, D, generator=g, device="cuda").to(dt) for _ in range(3))
        want, bound, p, pb = D64.step_weights(q, k, v, kc, vc, D ** -0.5, rows)
        D64.assert_within(ffa.attention(q, k, v, D ** -0.5), want, bound, f"step {step}")
        for b, n in enumerate(rows):
            w[b, :, n], off[b, :, n] = 0, 0
            kc[b, :, n], vc[b, :, n], pos[b, :, n] = k[b, :, 0], v[b, :, 0], seen[b]
        w = (w.double() + p).float()
        off = off + (pb + 2 * D64.U * w.double())[..., None]
        rows, seen = [n + 1 for n in rows], [n + 1 for n in seen]
        if max(rows) > budget + slack - 1:
            cut()
        assert ffa.lengths == rows == ffa.rows.tolist() and ffa.seen.tolist() == seen
        for b, n in enumerate(rows):   # the same tokens are left (their weights differ by roundings of fp32 only)
            assert torch.equal(ffa.positions[b, :, :n], pos[b, :, :n])
            assert ((ffa.weights[b, :, :n].double() - w[b, :, :n].double()).abs() <= off[b, :, :n, 0]).all()
    kf, vf = ffa.engine.get_cache()
    for b, n in enumerate(rows):
        assert torch.equal(kf[b, :, :n], kc[b, :, :n]) and torch.equal(vf[b, :, :n], vc[b, :, :n])
    assert ffa.engine.device_status() == 0


def test_captured_steps_and_evictions():
    dt, B, H, D, n = torch.bfloat16, 2, 4, 64, 200
    ffa, kc, vc, w, pos, g = engine(dt, B, H, D, n + 1, seed=13)
    twin, kt, vt, wt, pt, _ = engine(dt, B, H, D, n + 1, seed=13)
    rows, grown = (torch.full((B,), x, dtype=torch.int32, device="cuda") for x in (n, n + 1))
    seen = torch.full((B,), n, dtype=torch.int32, device="cuda")
    q, k, v = (torch.randn(B, H, 1, D, generator=g, device="cuda").to(dt) for _ in range(3))
    out = torch.empty(B, H, D, dtype=dt, device="cuda")

    def step(e, w, pos, seen, out):
        e.attention_accumulate(q, k, v, D ** -0.5, rows, w, pos, seen, out=out, max_row=n)
        kept = e.evict(grown, w, pos, n, recent=50, max_row=n + 1)
        seen += 1
        return kept

    other = torch.empty_like(out)
    t_seen = seen.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):   # the first call binds the score scratch
        step(ffa, w, pos, seen, out)
    torch.cuda.current_stream().wait_stream(side)
    step(twin, wt, pt, t_seen, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(ffa, w, pos, seen, out)
    for _ in range(4):
        for x in (q, k, v):
            x.normal_()
        graph.replay()
        want = step(twin, wt, pt, t_seen, other)
        assert torch.equal(out, other) and torch.equal(kept, want) and torch.equal(w, wt) and torch.equal(pos, pt)
        assert torch.equal(kc, kt) and torch.equal(vc, vt)
    assert ffa.device_status() == 0


def test_the_first_accumulating_step_is_not_captured_and_keeps_recorded_graphs_alive():
    dt, B, H, D, n = torch.float16, 1, 4, 64, 3000
    ffa, kc, vc, w, pos, g = engine(dt, B, H, D, n + 2, seed=19)
    q, k, v = (torch.randn(B, H, 1, D, generator=g, device="cuda").to(dt) for _ in range(3))
    rows = torch.full((B,), n, dtype=torch.int32, device="cuda")
    want = ffa.attention_per_sample(q, k, v, 0.1, rows)
    out = torch.empty_like(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ffa.attention_per_sample(q, k, v, 0.1, rows, out=out)
    refused = torch.cuda.CUDAGraph()
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="outside of a graph capture"):
            ffa.attention_accumulate(q, k, v, 0.1, rows, w, pos, rows)
        ffa.attention_per_sample(q, k, v, 0.1, rows, out=out)
    ffa.attention_accumulate(q, k, v, 0.1, rows, w, pos, rows)   # binds a larger workspace
    filler = [torch.full((1 << 20,), 7, dtype=torch.int32, device="cuda") for _ in range(8)]   # takes freed memory, if there is any
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    assert ffa.device_status() == 0 and len(filler) == 8


def test_refusals_from_python():
    dt, B, H, D, L = torch.float16, 2, 2, 64, 40
    ffa, kc, vc, w, pos, g = engine(dt, B, H, D, L, seed=17)
    rows = torch.full((B,), 30, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, H, 1, D, dtype=dt, device="cuda")
    good = dict(seq_lengths=rows, weights=w, positions=pos, keep=20)
    for change, match in [(dict(keep=0), "keep"), (dict(keep=41), "keep"), (dict(recent=-1), "recent"), (dict(recent=15, first=6), "recent"),
                          (dict(weights=w.half()), "weights"), (dict(weights=w[:, :, :30]), "weights"), (dict(positions=pos.long()), "positions"),
                          (dict(seq_lengths=rows.long()), "seq_lengths"), (dict(seq_lengths=rows.cpu()), "seq_lengths"), (dict(max_row=41), "max_row")]:
        with pytest.raises(RuntimeError, match=match):
            ffa.evict(**{**good, **change})
    good = dict(q=q, k=q, v=q, softmax_scale=1.0, seq_lengths=rows, weights=w, positions=pos, seen=rows)
    for change, match in [(dict(q=q.float()), "q must"), (dict(k=q[:1]), "k must"), (dict(weights=w[..., ::2]), "weights"), (dict(seen=rows[:1]), "seen"),
                          (dict(max_row=40), "max_row"), (dict(out=torch.empty(B, H, D, device="cuda")), "out must")]:
        with pytest.raises(RuntimeError, match=match):
            ffa.attention_accumulate(**{**good, **change})
    wb = w.clone()
    ffa.attention_accumulate(**{**good, "seq_lengths": torch.tensor([40, 10], dtype=torch.int32, device="cuda")})   # row 40 of 40
    assert ffa.device_status() == 2 and torch.equal(w[0], wb[0]) and not torch.equal(w[1], wb[1])
