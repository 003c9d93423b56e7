"""Attention of a tree of drafted tokens over a cache, and the acceptance of a path, against their 64-bit definitions."""
import math

import pytest
import torch

from oracle import decoding_oracle as D64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def random_tree(T, g, B=None):
    def one():
        see = torch.zeros(T, T, dtype=torch.bool)
        for j in range(T):
            if j:
                see[j] = see[int(torch.randint(0, j, (1,), generator=g))]
            see[j, j] = True
        return see
    return one() if B is None else torch.stack([one() for _ in range(B)])


def setup(dt, B, H, G, D, n, T, L=None, seed=0, per_sample=True):
    from fastforwardattention_b200 import FastForwardAttn

    g = torch.Generator().manual_seed(seed)
    L = L or n + T + 5
    r = lambda *s: torch.randn(*s, generator=g).to(dt).cuda()
    kc, vc = r(B, H, L, D), r(B, H, L, D)
    q, k, v = r(B, H * G, T, D), r(B, H, T, D), r(B, H, T, D)
    tree = random_tree(T, g, B if per_sample else None).cuda()
    return FastForwardAttn.adopt(kc, vc), kc, vc, q, k, v, tree


def check(ffa, kc, vc, q, k, v, tree, rows, call, first=None, what="", scale=None):
    kb, vb = kc.clone(), vc.clone()
    want, bound = D64.tree_attention(q, k, v, kb, vb, tree, q.shape[-1] ** -0.5 if scale is None else scale, rows, first)
    out = call()
    D64.assert_within(out, want, bound, what)
    T = k.shape[2]
    for b, n in enumerate(rows):
        kb[b, :, n:n + T], vb[b, :, n:n + T] = k[b], v[b]
    assert torch.equal(kb, kc) and torch.equal(vb, vc), what + ": the caches hold other rows than the appended ones"
    assert ffa.device_status() == 0
    return out


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("G,T,n", [(1, 1, 0), (1, 1, 1), (1, 3, 200), (1, 8, 63), (2, 5, 64), (1, 33, 129), (4, 33, 65), (1, 100, 31), (8, 40, 300),
                                   (1, 64, 64), (1, 129, 7)])
def test_against_definition(dt, D, G, T, n):
    ffa, kc, vc, q, k, v, tree = setup(dt, 2, 3, G, D, n, T, seed=T * 1000 + n, per_sample=T % 2 == 1)
    check(ffa, kc, vc, q, k, v, tree, [n, n], lambda: ffa.tree_attention(q, k, v, tree, D ** -0.5, n), what=f"{dt} {D} {G} {T} {n}")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T,G", [(1, 1), (7, 1), (20, 2), (64, 4)])
def test_long_cache_is_split_over_ctas(dt, T, G):
    n, D = 4099, 128
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, 2, G, D, n, T, seed=T)
    out = check(ffa, kc, vc, q, k, v, tree, [n], lambda: ffa.tree_attention(q, k, v, tree, D ** -0.5, n))
    for _ in range(3):   # the splits are merged in a fixed order, and the arrival counters are ready again
        assert torch.equal(out, ffa.tree_attention(q, k, v, tree, D ** -0.5, n))


@pytest.mark.parametrize("dt", DTYPES)
def test_per_sample_lengths_and_bound(dt):
    B, D, T, n = 6, 64, 13, 700
    ffa, kc, vc, q, k, v, tree = setup(dt, B, 2, 1, D, n, T, seed=5)
    rows = [0, 1, 64, 333, 699, 700]
    sl = torch.tensor(rows, dtype=torch.int32, device="cuda")
    for bound in (-1, n, n + 3):
        check(ffa, kc, vc, q, k, v, tree, rows, lambda: ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, sl, max_row=bound))


@pytest.mark.parametrize("dt", DTYPES)
def test_left_padding(dt):
    B, D, T, n = 5, 128, 9, 257
    ffa, kc, vc, q, k, v, tree = setup(dt, B, 2, 2, D, n, T, seed=6)
    first = [0, 1, 64, 200, 257]
    for b, lo in enumerate(first):   # what the padding rows hold never matters
        kc[b, :, :lo], vc[b, :, :lo] = float("nan"), float("inf")
    kb, vb = kc.clone(), vc.clone()
    want, bound = D64.tree_attention(q, k, v, kb, vb, tree, D ** -0.5, [n] * B, first)
    out = ffa.tree_attention(q, k, v, tree, D ** -0.5, n, seq_lengths=torch.tensor(first, dtype=torch.int32, device="cuda"))
    D64.assert_within(out, want, bound)
    assert ffa.device_status() == 0


@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("G,T", [(1, 8), (3, 3), (1, 15), (2, 8), (1, 17)])
def test_few_query_rows_in_fp32(D, G, T):
    """Row counts around those where the fp32 kernels take turns; lengths and padding that leave warps without keys; a row that sees nothing
    but the cache, and at length 0 nothing at all; with several CTAs to a pair and with few."""
    n, some = 1500, [0, 5, 41, 1499, 1500, 1497, 64, 1425]
    for B in (4, 64):
        at = (some * B)[:B]
        dev = torch.tensor(at, dtype=torch.int32, device="cuda")
        for padded in (False, True):
            ffa, kc, vc, q, k, v, tree = setup(torch.float32, B, 4, G, D, n, T, seed=D + T)
            lo, hi = (at, [n] * B) if padded else ([0] * B, at)
            for b in range(B):   # what is outside the valid rows never matters
                for c in (kc, vc):
                    c[b, :, :lo[b]], c[b, :, hi[b]:] = float("nan"), float("inf")
            tree[..., T - 1, :] = False
            want, bound = D64.tree_attention(q, k, v, kc.clone(), vc.clone(), tree, D ** -0.5, hi, lo)
            if padded:
                out = ffa.tree_attention(q, k, v, tree, D ** -0.5, n, seq_lengths=dev)
            else:
                out = ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, dev, max_row=n)
                assert (out[0].view(4, G, T, D)[:, :, T - 1] == 0).all()
            D64.assert_within(out, want, bound, f"{B} sequences, padded {padded}")
            for b in range(B):
                assert torch.equal(kc[b, :, hi[b]:hi[b] + T], k[b]) and torch.equal(vc[b, :, hi[b]:hi[b] + T], v[b])
            assert ffa.device_status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,T", [(0, 6), (130, 6), (130, 70), (4000, 20)])
def test_hidden_and_stale_values_have_no_influence(dt, n, T):
    """NaN and infinities in cache rows behind the last one, and in drafted tokens that a row does not see."""
    D = 64
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, 2, 1, D, n, T, seed=n + T, L=n + T + 90)
    kc[:, :, n:], vc[:, :, n:] = float("nan"), float("inf")
    bad = T - 2
    k[:, :, bad], v[:, 0, bad] = float("nan"), float("inf")
    v[:, 1, bad] = float("nan")
    tree[:, :, bad] = False
    want, bound = D64.tree_attention(q, k, v, kc, vc, tree, D ** -0.5, [n])
    assert torch.isfinite(want).all()
    D64.assert_within(ffa.tree_attention(q, k, v, tree, D ** -0.5, n), want, bound)


@pytest.mark.parametrize("dt", DTYPES)
def test_a_visible_infinity_reaches_the_rows_that_see_it_and_no_others(dt):
    D, T, n = 64, 12, 100
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, 1, 1, D, n, T, seed=9)
    v[0, 0, 3, 5], v[0, 0, 4, 6] = float("inf"), float("nan")
    want, bound = D64.tree_attention(q, k, v, kc, vc, tree, D ** -0.5, [n])
    assert not torch.isfinite(want).all() and torch.isfinite(want[0, 0, 0]).all()
    D64.assert_within(ffa.tree_attention(q, k, v, tree, D ** -0.5, n), want, bound)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("row", [5, 64, 70, 250, 299])
def test_a_broken_key_makes_the_rows_that_see_it_nan(dt, row):
    """NaN in one element of a cached key (every row sees it), and in a drafted one (its descendants do)."""
    D, T, n = 128, 9, 300
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, 2, 1, D, n, T, seed=row)
    kc[0, 0, row, 77] = float("nan")
    k[0, 1, 4, 3] = float("nan")
    want, bound = D64.tree_attention(q, k, v, kc, vc, tree, D ** -0.5, [n])
    assert torch.isnan(want[0, 0]).all() and torch.isnan(want[0, 1, 4]).all() and torch.isfinite(want[0, 1, 0]).all()
    D64.assert_within(ffa.tree_attention(q, k, v, tree, D ** -0.5, n), want, bound)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_any_scale(dt, scale):
    D, T, n = 64, 30, 200
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, 2, 2, D, n, T, seed=41)
    check(ffa, kc, vc, q, k, v, tree, [n], lambda: ffa.tree_attention(q, k, v, tree, scale, n), scale=scale)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("T", [4, 40, 140])
def test_rows_that_see_nothing_are_zero(dt, T):
    D = 128
    ffa, kc, vc, q, k, v, tree = setup(dt, 2, 1, 1, D, 0, T, seed=11)
    tree[0] = False
    tree[1, 1] = False
    out = check(ffa, kc, vc, q, k, v, tree, [0, 0], lambda: ffa.tree_attention(q, k, v, tree, D ** -0.5, 0))
    assert (out[0] == 0).all() and (out[1, :, 1] == 0).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_scores_that_grow_along_the_cache(dt):
    """The running maximum moves by far more than any exponent range, upwards in every tile; and once downwards."""
    D, n, T = 64, 640, 17
    for sign in (1.0, -1.0):
        ffa, kc, vc, q, k, v, tree = setup(dt, 1, 2, 1, D, n, T, seed=13)
        q[:] = 1.0
        ramp = torch.linspace(-8, 8, n, device="cuda") * sign
        kc[:, :, :n] = ramp[:, None].to(dt)
        check(ffa, kc, vc, q, k, v, tree, [n], lambda: ffa.tree_attention(q, k, v, tree, D ** -0.5, n))


@pytest.mark.parametrize("dt", DTYPES)
def test_strided_inputs_out_argument_and_other_stream(dt):
    B, H, D, T, n = 2, 4, 64, 11, 90
    ffa, kc, vc, q, k, v, tree = setup(dt, B, H, 1, D, n, T, seed=17)
    wide = torch.randn(B, T, 3, H, D, device="cuda").to(dt)   # a fused projection's output
    q, k, v = (wide[:, :, i].transpose(1, 2) for i in range(3))
    big = torch.zeros(B, 2 * T, 2 * T, dtype=torch.bool, device="cuda")
    big[:, ::2, 1::2] = tree
    out = torch.full((B, H, T, D), 7.0, dtype=dt, device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = check(ffa, kc, vc, q, k, v, big[:, ::2, 1::2], [n] * B,
                    lambda: ffa.tree_attention(q, k, v, big[:, ::2, 1::2], D ** -0.5, n, out=out))
    side.synchronize()
    assert got.data_ptr() == out.data_ptr()
    assert torch.equal(ffa.tree_attention(q, k, v, tree.to(torch.uint8), D ** -0.5, n), out)


@pytest.mark.parametrize("dt", DTYPES)
def test_captured_and_replayed_with_lengths_on_the_device(dt):
    B, H, D, T, n = 2, 2, 128, 21, 2500
    ffa, kc, vc, q, k, v, tree = setup(dt, B, H, 1, D, n, T, L=n + 4 * T, seed=19)
    rows = torch.full((B,), n, dtype=torch.int32, device="cuda")
    path = torch.tensor([[0, 2, 5], [1, -1, -1]], dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, rows, out=out, max_row=n + 3 * T)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, rows, out=out, max_row=n + 3 * T)
        ffa.tree_accept_per_sample(path, rows)
        rows += (path >= 0).sum(1, dtype=torch.int32)
    now = [n, n]
    for _ in range(3):
        for x in (q, k, v):
            x.normal_()
        kb, vb = kc.clone(), vc.clone()
        want, bound = D64.tree_attention(q, k, v, kb, vb, tree, D ** -0.5, now)
        graph.replay()
        D64.assert_within(out, want, bound)
        for cache, new in ((kb, k), (vb, v)):
            for b, m in enumerate(now):
                cache[b, :, m:m + T] = new[b]
            cache.copy_(D64.tree_accept(cache, [[0, 2, 5], [1]], now))
        assert torch.equal(kb, kc) and torch.equal(vb, vc)
        now = [now[0] + 3, now[1] + 1]
    assert rows.tolist() == now and ffa.device_status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_accept_moves_the_path_to_the_front(dt, D):
    from fastforwardattention_b200 import FastForwardAttn

    B, H, L, n = 4, 3, 120, 37
    kc, vc = (torch.randn(B, H, L, D, device="cuda").to(dt) for _ in range(2))
    ffa = FastForwardAttn.adopt(kc, vc)
    paths = [list(range(1, 40, 2)), [], [0, 1, 2, 50], [L - n - 6]]
    flat = torch.full((B, 20), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        flat[b, : len(p)] = torch.tensor(p, dtype=torch.int32)
    rows = [n, n + 1, n + 2, n + 5]
    want = [D64.tree_accept(c, paths, rows) for c in (kc, vc)]
    ffa.tree_accept_per_sample(flat.cuda(), torch.tensor(rows, dtype=torch.int32, device="cuda"))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]) and ffa.device_status() == 0
    want = [D64.tree_accept(c, [[2, 3]] * B, [n] * B) for c in (kc, vc)]
    ffa.tree_accept(torch.tensor([[2, 3]] * B, dtype=torch.int32, device="cuda"), n)
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])
    ffa.tree_accept(torch.empty(B, 0, dtype=torch.int32, device="cuda"), n)
    assert torch.equal(kc, want[0])


def test_what_the_device_refuses():
    """Lengths and paths that only the device sees: reported, zeros out, nothing appended or moved for that sample; the others go on."""
    dt, B, D, T, n = torch.float16, 4, 64, 6, 50
    ffa, kc, vc, q, k, v, tree = setup(dt, B, 2, 1, D, n, T, L=64, seed=23)
    kb, vb = kc.clone(), vc.clone()
    rows = torch.tensor([n, 59, -1, 10], dtype=torch.int32, device="cuda")   # 59 + 6 > 64
    out = ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, rows)
    assert ffa.device_status() == 2
    want, bound = D64.tree_attention(q, k, v, kb, vb, tree, D ** -0.5, [n, 0, 0, 10])
    for b in (0, 3):
        D64.assert_within(out[b], want[b], bound[b])
    assert (out[1:3] == 0).all() and torch.equal(kc[1:3], kb[1:3]) and torch.equal(vc[1:3], vb[1:3])
    ffa.tree_attention_per_sample(q, k, v, tree, D ** -0.5, rows.clamp(0, 40), max_row=30)   # above the stated bound
    assert ffa.device_status() == 2
    kb = kc.clone()
    ffa.tree_accept_per_sample(torch.tensor([[0, 2], [2, 1], [3, 3], [13, 14]], dtype=torch.int32, device="cuda"),
                               torch.tensor([20, 20, 20, 50], dtype=torch.int32, device="cuda"))
    assert ffa.device_status() == 4
    assert torch.equal(kc[1:], kb[1:]) and torch.equal(kc[0], D64.tree_accept(kb, [[0, 2], [], [], []], [20] * 4)[0])


def test_refusals_from_python():
    dt, B, H, D, T, n = torch.bfloat16, 2, 2, 64, 4, 20
    ffa, kc, vc, q, k, v, tree = setup(dt, B, H, 1, D, n, T, L=32, seed=29)
    s = D ** -0.5
    for bad, match in [((q.float(), k, v, tree, s, n), "dtype"), ((q[:, :1], k, v, tree, s, n), "multiple"), ((q, k[:, :, :2], v, tree, s, n), "k must be"),
                       ((q, k, v.cpu(), tree, s, n), "v must be"), ((q, k, v, tree.float(), s, n), "tree"), ((q, k, v, tree[:, :2], s, n), "tree"),
                       ((q, k, v, tree, s, 32), "outside"), ((q, k, v, tree, s, 29), "exceeds the cache"), ((q, k, v, tree, s, -1), "outside")]:
        with pytest.raises(RuntimeError, match=match):
            ffa.tree_attention(*bad)
    with pytest.raises(RuntimeError, match="seq_lengths"):
        ffa.tree_attention_per_sample(q, k, v, tree, s, torch.zeros(B, dtype=torch.int64, device="cuda"))
    with pytest.raises(RuntimeError, match="out must"):
        ffa.tree_attention(q, k, v, tree, s, n, out=torch.empty(B, H, T, D, device="cuda"))
    many = torch.ones(1025, 1025, dtype=torch.bool, device="cuda")
    with pytest.raises(RuntimeError, match="1024"):
        ffa.tree_attention(torch.zeros(B, H, 1025, D, dtype=dt, device="cuda"), k, v, many, s, n)
    with pytest.raises(RuntimeError, match="path"):
        ffa.tree_accept(torch.zeros(B, 2, dtype=torch.int64, device="cuda"), n)
    assert ffa.device_status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_paged_sequences_draft_and_accept(dt, D):
    from fastforwardattention_b200 import PagedFastForwardAttn, PagePool

    B, H, T = 3, 2, 24
    lens = [130, 250, 1]
    pool = PagePool(16, H, D, dt, "cuda", page_rows=128)
    pool.k.fill_(float("nan")), pool.v.fill_(float("nan"))
    K, V = (torch.randn(B, H, 256, D, device="cuda").to(dt) for _ in range(2))
    seqs = PagedFastForwardAttn(pool, K, V, 512, lengths=lens)
    kc, vc = (torch.zeros(B, H, 512, D, dtype=dt, device="cuda") for _ in range(2))
    for b, n in enumerate(lens):
        kc[b, :, :n], vc[b, :, :n] = K[b, :, :n], V[b, :, :n]
    g = torch.Generator().manual_seed(31)
    now = list(lens)
    for step in range(3):
        q, k, v = (torch.randn(B, h, T, D, generator=g).to(dt).cuda() for h in (2 * H, H, H))
        tree = random_tree(T, g, B).cuda()
        want, bound = D64.tree_attention(q, k, v, kc, vc, tree, D ** -0.5, now)
        D64.assert_within(seqs.tree_attention(q, k, v, tree, D ** -0.5), want, bound, f"step {step}")
        path = [[0, 3, 7, 20], [step], list(range(step))]
        seqs.tree_accept(path)
        for b, p in enumerate(path):
            for i, j in enumerate(p):
                kc[b, :, now[b] + i], vc[b, :, now[b] + i] = k[b, :, j], v[b, :, j]
        now = [n + len(p) for n, p in zip(now, path)]
        assert seqs.lengths == now == seqs.rows.tolist()
    q, k, v = (torch.randn(B, H, 1, D, generator=g).to(dt).cuda() for _ in range(3))
    one = torch.ones(1, 1, dtype=torch.bool, device="cuda")
    want, bound = D64.tree_attention(q, k, v, kc, vc, one, D ** -0.5, now)
    D64.assert_within(seqs.attention(q, k, v, D ** -0.5)[:, :, None], want, bound, "one-token step")
    assert seqs.engine.device_status() == 0
    for bad in ([[0], [0]], [[1, 0], [], []], [[-1], [], []], [[300], [], []]):
        with pytest.raises(ValueError):
            seqs.tree_accept(bad)


@pytest.mark.parametrize("dt", DTYPES)
def test_drafting_agrees_with_one_token_steps(dt):
    """Speculative decoding as it is used: a tree over the cache, its accepted path kept, then a one-token step; the one-token steps
    over the same path give the same outputs."""
    from fastforwardattention_b200 import FastForwardAttn

    B, H, D, n, T = 2, 4, 64, 300, 10
    g = torch.Generator().manual_seed(37)
    K, V = (torch.randn(B, H, n, D, generator=g).to(dt).cuda() for _ in range(2))
    a, c = FastForwardAttn(K, V, n + 32, False), FastForwardAttn(K, V, n + 32, False)
    tree = random_tree(T, g)
    path = tree[T - 1].nonzero().flatten().tolist()
    tree = tree.cuda()
    q, k, v = (torch.randn(B, H, T, D, generator=g).to(dt).cuda() for _ in range(3))
    _, bound = D64.tree_attention(q, k, v, *a.get_cache(), tree, D ** -0.5, [n] * B)
    out = a.tree_attention(q, k, v, tree, D ** -0.5, n)
    a.tree_accept(torch.tensor([path] * B, dtype=torch.int32, device="cuda"), n)
    for i, j in enumerate(path):
        step = c.attention(q[:, :, j].contiguous(), k[:, :, j].contiguous(), v[:, :, j].contiguous(), D ** -0.5, n + i, 0)
        assert ((step.double() - out[:, :, j].double()).abs() <= 2 * bound[:, :, j]).all()
    for x, y in zip(a.get_cache(), c.get_cache()):
        assert torch.equal(x[:, :, : n + len(path)], y[:, :, : n + len(path)])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_offsets_beyond_32_bits(dt):
    """Caches of more than 2^31 elements (2^33 bytes in fp32): the last pair's rows, attended, appended and moved."""
    from fastforwardattention_b200 import FastForwardAttn

    B, H, L, D, T = 8, 32, 66000, 128, 6
    kc, vc = (torch.empty(B, H, L, D, dtype=dt, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(43)
    n = L - T
    for c in (kc, vc):
        c.zero_()
        c[-1, -1, -3000:] = torch.randn(3000, D, generator=g).to(dt).cuda()
        c[-1, -1, : n - 2000] = torch.randn(1, D, generator=g).to(dt).cuda()
    q, k, v = (torch.randn(B, H, T, D, generator=g).to(dt).cuda() for _ in range(3))
    tree = random_tree(T, g).cuda()
    ffa = FastForwardAttn.adopt(kc, vc)
    last = lambda x: x[-1:, -1:]
    want, bound = D64.tree_attention(last(q), last(k), last(v), last(kc), last(vc), tree, D ** -0.5, [n])
    out = ffa.tree_attention(q, k, v, tree, D ** -0.5, n)
    D64.assert_within(last(out), want, bound)
    assert torch.equal(last(kc)[:, :, n:], last(k)) and torch.equal(last(vc)[:, :, n:], last(v))
    ffa.tree_accept(torch.tensor([[1, 3, 5]] * B, dtype=torch.int32, device="cuda"), n)
    assert torch.equal(kc[-1, -1, n: n + 3], k[-1, -1, [1, 3, 5]])
    before = vc[-1, -1, 65000:].clone()
    ffa.reorder(torch.tensor([[0, 1, 2, 3, 4, 5, 7, 6]], dtype=torch.int32, device="cuda"), L, first_row=65000)
    assert torch.equal(vc[-2, -1, 65000:], before) and ffa.device_status() == 0


def test_a_full_cache_accepts_an_empty_path():
    dt, B, D = torch.bfloat16, 2, 64
    ffa, kc, vc, q, k, v, tree = setup(dt, B, 1, 1, D, 20, 4, L=24, seed=47)
    kb = kc.clone()
    ffa.tree_accept_per_sample(torch.tensor([[-1, -1], [0, 3]], dtype=torch.int32, device="cuda"), torch.tensor([24, 20], dtype=torch.int32, device="cuda"))
    assert ffa.device_status() == 0 and torch.equal(kc[0], kb[0]) and torch.equal(kc[1, :, 21], kb[1, :, 23])


@pytest.mark.parametrize("dt", DTYPES)
def test_two_engines_on_two_streams(dt):
    """Calls that run at the same time on engines of their own."""
    D, T, n = 128, 30, 3000
    cases = [setup(dt, 1, 2, 1, D, n, T, seed=50 + i) for i in range(2)]
    want = [c[0].tree_attention(*c[3:7], D ** -0.5, n) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c[0].tree_attention(*c[3:7], D ** -0.5, n))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dt", DTYPES)
def test_pages_that_are_missing_or_outside_the_pool_are_refused(dt):
    """Every sequence stands on its own: those whose rows have no page are reported and left, the others go on."""
    from fastforwardattention_b200 import PagePool, _extension

    B, H, D, T, pr = 5, 2, 64, 20, 128
    pool = PagePool(12, H, D, dt, "cuda", page_rows=pr)
    pool.k.normal_(), pool.v.normal_()
    engine = _extension().PagedEngine(pool.k, pool.v, B, 4)
    rows = [120, 120, 250, 130, 10]
    table = torch.tensor([[0, 1, -1, -1], [2, -1, -1, -1], [3, 12, 4, -1], [-1, 5, 6, -1], [7, -1, -1, -1]], dtype=torch.int32)
    q, k, v = (torch.randn(B, H, T, D, device="cuda").to(dt) for _ in range(3))
    tree = torch.ones(T, T, dtype=torch.bool, device="cuda").tril()
    sl = torch.tensor(rows, dtype=torch.int32, device="cuda")
    kb, vb = pool.k.clone(), pool.v.clone()
    out = engine.tree_attention_per_sample(q, k, v, tree, table.cuda(), D ** -0.5, sl)
    assert engine.device_status() == 4 and (out[1:4] == 0).all()
    flat = lambda p, pages: torch.cat([p[i] for i in pages], 1)[None]
    for b, pages in ((0, [0, 1]), (4, [7])):
        one = slice(b, b + 1)
        want, bound = D64.tree_attention(q[one], k[one], v[one], flat(kb, pages), flat(vb, pages), tree, D ** -0.5, [rows[b]])
        D64.assert_within(out[one], want, bound)
        assert torch.equal(flat(pool.k, pages)[0, :, rows[b]: rows[b] + T], k[b])
    assert torch.equal(pool.k[[2, 3, 4, 5, 6, 8, 9, 10, 11]], kb[[2, 3, 4, 5, 6, 8, 9, 10, 11]])
    kb = pool.k.clone()
    path = torch.tensor([[0, 19], [0, 19], [1, 2], [3, 4], [118, 119]], dtype=torch.int32, device="cuda")
    engine.tree_accept_per_sample(path, table.cuda(), sl)
    assert engine.device_status() == 4
    # sequences 1 (row 139), 2 (row 251) and 4 (row 128) name rows of missing pages; of sequence 3 only the first page is missing, and its
    # rows 133, 134 -> 130, 131 lie in the second one (page 5, rows 5, 6 -> 2, 3)
    kb[5, :, 2:4] = kb[5, :, 5:7].clone()
    assert torch.equal(pool.k[0, :, 121], kb[1, :, 11]) and torch.equal(pool.k[2:], kb[2:])


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 256])
@pytest.mark.parametrize("T", [1, 8, 40, 100])
@pytest.mark.parametrize("n", [130, 5000])
def test_an_infinity_in_a_cached_row_is_one_in_the_result(dt, D, T, n):
    """Every row sees it with a weight above 0, however many rows share the key tiles and however many CTAs the pair."""
    ffa, kc, vc, q, k, v, tree = setup(dt, 2, 2, 1, D, n, T, seed=D + T + n)
    q *= 0.5   # (fp32 weights do not vanish: scores stay within a few dozen)
    vc[0, 0, 3, 5], vc[0, 0, n - 1, D - 1] = float("inf"), -float("inf")
    vc[0, 1, 64, 17], vc[0, 1, 100, 17] = float("inf"), -float("inf")   # of both signs: NaN
    vc[1, 0, 65, 30], vc[1, 0, 2, 31] = float("nan"), float("inf")
    v[0, 0, 0, 6] = -float("inf")                                        # and one in a drafted token, next to a cached one's column
    want, bound = D64.tree_attention(q, k, v, kc, vc, tree, D ** -0.5, [n, n])
    assert torch.isinf(want[0, 0, :, 5]).all() and torch.isnan(want[0, 1, :, 17]).all() and torch.isfinite(want[1, 1]).all()
    out = ffa.tree_attention(q, k, v, tree, D ** -0.5, n)
    D64.assert_within(out, want, bound)


def close_bound(q, k, v, k_cache, v_cache, tree, scale, rows, top=1.0):
    """The exact result, and how far a kernel may be from it: the fp32 bound, and of a = sum p |v| a half step for weights rounded to the type, or its
    square for weights that are sums of two numbers of it (up to 32 query rows), and 6e-6 (the exponentials' 2.7e-6 in the weights and in their
    sum); in fp16, whose weights are held at 2^7 times their size, what is below 2^-25 of that
    vanishes, 2^-32 of the largest weight (`top`: of all); then one rounding of the result."""
    wide = [x.float() for x in (q, k, v, k_cache, v_cache)]
    out, err = D64.tree_attention(*wide, tree, scale, rows)
    a, _ = D64.tree_attention(*wide[:2], wide[2].abs(), wide[3], wide[4].abs(), tree, scale, rows)
    h = D64.half_step(q.dtype)
    few = q.shape[1] // k.shape[1] * q.shape[2] <= 32
    err = err + ((h * h if few else h) + 6e-6) * a
    if q.dtype == torch.float16:
        n = max(rows)
        err = err + 2.0 ** -32 * top * (wide[4][:, :, :n].abs().sum(2).amax() + wide[2].abs().sum(2).amax())
    return out, err + h * (out.abs() + err)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("G,T,n", [(1, 1, 700), (1, 8, 63), (1, 27, 1000), (2, 16, 400), (4, 8, 5000), (1, 33, 300), (1, 100, 300)])
def test_weights_keep_more_bits_than_the_tensors(dt, D, G, T, n):
    """With up to 32 query rows the only rounding to the tensors' type is the result's, as in the one-token step."""
    ffa, kc, vc, q, k, v, tree = setup(dt, 2, 2, G, D, n, T, seed=T + n)
    want, bound = close_bound(q, k, v, kc, vc, tree, D ** -0.5, [n, n])
    D64.assert_within(ffa.tree_attention(q, k, v, tree, D ** -0.5, n), want, bound)


@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 40, 70])
@pytest.mark.parametrize("units", [6.5, 40.5, 300.5, 1200.5])
def test_many_light_keys_beside_heavy_ones(dt, T, units):
    """Attention sinks: every 256th key takes a weight of 1 and has no value, each of the others has `units` of fp16's smallest steps (2^-24), and
    the result is theirs alone: what is lost of their weights shows whole."""
    H, D, n = 2, 64, 16384
    ffa, kc, vc, q, k, v, tree = setup(dt, 1, H, 1, D, n, T, seed=T)
    scale = math.log(2.0 ** 24 / units) / D   # q . k of a sink: D
    q.fill_(1.0), kc.zero_(), k.zero_()
    kc[:, :, ::256] = 1.0
    vc += 1.0
    vc[:, :, ::256] = 0.0
    want, bound = close_bound(q, k, v, kc, vc, tree, scale, [n], top=256 / n)
    D64.assert_within(ffa.tree_attention(q, k, v, tree, scale, n), want, bound)


def test_paths_that_repeat_an_index_at_the_end_of_a_paged_sequence():
    """The last row of the last sequence has no table entry behind it: such a path is refused before its pages are looked up."""
    from fastforwardattention_b200 import PagePool, _extension

    B, H, D, pr = 2, 2, 64, 128
    pool = PagePool(4, H, D, torch.float16, "cuda", page_rows=pr)
    pool.k.normal_(), pool.v.normal_()
    kb, vb = pool.k.clone(), pool.v.clone()
    engine = _extension().PagedEngine(pool.k, pool.v, B, 2)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    last = torch.tensor([2 * pr - 1] * B, dtype=torch.int32, device="cuda")
    for path in ([[0, 0], [0, 0]], [[0, 0, 0, 0]] * 2, [[0, 1], [0, 1]]):
        engine.tree_accept_per_sample(torch.tensor(path, dtype=torch.int32, device="cuda"), table, last)
        assert engine.device_status() == 4 and torch.equal(pool.k, kb) and torch.equal(pool.v, vb)
    engine.tree_accept_per_sample(torch.tensor([[0, -1], [0, -1]], dtype=torch.int32, device="cuda"), table, last)
    assert engine.device_status() == 0 and torch.equal(pool.k, kb)
