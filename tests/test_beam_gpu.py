"""Selection over beams and vocabulary, and the reordering of the caches, against their plain definitions."""
import math

import pytest
import torch

from oracle import decoding_oracle as D64

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


def check(logits, scores, num, finished=None, pad=0):
    from fastforwardattention_b200 import beam_select

    want, parents, tokens = D64.beam_select(logits, scores, num, finished, pad)
    got = beam_select(logits, scores, num, finished=finished, pad_token=pad)
    assert torch.equal(got[1].cpu(), parents) and torch.equal(got[2].cpu(), tokens)
    s = got[0].cpu().double()
    fin = want > -INF
    assert torch.equal(s > -INF, fin)
    # one rounding of the result, and the logarithm of a sum: its terms are exact to a dozen half steps of fp32 (the exponential's four, its
    # argument's, |x - m| exp(x - m) of which stay below one each), and a lane adds up its share of them in fp32
    terms = -(-logits.shape[-1] // (32 * (128 // logits.shape[1])))
    assert ((s - want).abs()[fin] <= D64.U * want.abs()[fin] + (12 + terms) * D64.U).all()
    return got


def candidates(dt, B, N, V, seed=0, spread=3.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(B, N, V, generator=g, device="cuda") * spread).to(dt), torch.randn(B, N, generator=g, device="cuda")


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,N,V,num", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 17, 4), (1, 4, 50272, 8), (3, 5, 1001, 10), (2, 8, 50400, 16), (1, 32, 3001, 64),
                                       (5, 7, 256, 14), (1, 1, 200003, 64), (40, 2, 333, 2), (80, 3, 1200, 6), (150, 4, 700, 64), (300, 1, 901, 3),
                                       (300, 17, 100, 20), (200, 32, 64, 64)])
def test_select(dt, B, N, V, num):
    check(*candidates(dt, B, N, V, seed=V + num), num)


@pytest.mark.parametrize("dt", DTYPES)
def test_select_first_step_one_live_beam(dt):
    logits, scores = candidates(dt, 3, 16, 5000, seed=1)
    logits[:] = logits[:, :1]   # all beams have seen the same prompt
    scores.fill_(-INF)
    scores[:, 0] = 0.0
    _, parents, _ = check(logits, scores, 32)
    assert (parents == 0).all()
    scores.zero_()              # or all are alive: equal candidates, the lowest beam first
    check(logits, scores, 32)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [5000, 5001, 5002, 5003])
def test_select_equal_beams_at_any_alignment(dt, V):
    """Identical rows give identical sums wherever they start in memory: their candidates tie, and the lowest beam comes first."""
    logits, _ = candidates(dt, 2, 8, V, seed=V)
    logits[:] = logits[:, :1]
    _, parents, tokens = check(logits, torch.zeros(2, 8, device="cuda"), 16)
    assert (parents == torch.arange(8, device="cuda").repeat(2)).all() and (tokens[:, :8] == tokens[:, :1]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_select_ties(dt):
    """More candidates reach the border than any list holds: equal logits everywhere, or in blocks."""
    scores = torch.tensor([[0.0, 0.0, -0.5], [-1.0, 2.0, 2.0]], device="cuda")
    logits = torch.zeros(2, 3, 40001, dtype=dt, device="cuda")
    check(logits, scores, 64)
    logits[:, :, 5000:] = 1.0
    logits[:, 1, 39990:] = 1.5
    check(logits, scores, 40)
    logits[1, 2, 17] = 30.0     # one candidate above a sea of equal ones
    check(logits, scores, 7)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,N,num", [(2, 8, 16), (2, 32, 64), (40, 8, 16), (160, 16, 40), (310, 4, 64)])
def test_select_one_beam_far_ahead(dt, B, N, num):
    """All candidates come from one beam, whose tokens lie close together."""
    logits, scores = candidates(dt, B, N, 4000, seed=N, spread=0.5)
    scores[torch.arange(B), torch.arange(B) % N] += 30.0
    _, parents, _ = check(logits, scores, num)
    assert (parents.cpu() == (torch.arange(B) % N)[:, None]).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_select_masked_and_broken_logits(dt):
    logits, scores = candidates(dt, 6, 4, 900, seed=2)
    logits[0] = -INF                          # nothing at all
    logits[1, :, 3:] = -INF                   # three tokens left to each beam
    logits[2, 1, 5], logits[2, 2, 6] = float("nan"), INF
    logits[3, 0], logits[3, 1] = float("nan"), torch.finfo(dt).min
    logits[4, :, ::2] = torch.finfo(dt).min   # masked by the lowest value of the type
    scores[5, 1], scores[5, 2] = -INF, float("nan")
    got = check(logits, scores, 16)
    assert (got[0][0] == -INF).all() and (got[1][0] == 0).all() and (got[2][0] == 0).all()


@pytest.mark.parametrize("dt", DTYPES)
def test_select_finished_beams(dt):
    logits, scores = candidates(dt, 4, 5, 2000, seed=3)
    finished = torch.zeros(4, 5, dtype=torch.bool, device="cuda")
    finished[0, 2], finished[1, :4], finished[2, :] = True, True, True
    logits[1, 0] = float("nan")               # a finished beam's logits are not looked at
    scores[3, 0] = -50.0
    check(logits, scores, 10, finished, 7)


@pytest.mark.parametrize("dt", DTYPES)
def test_select_padded_and_unaligned_rows(dt):
    big, scores = candidates(dt, 3, 4, 1037, seed=4)
    big[..., 1000:] = 100.0                   # a padded vocabulary's tail is not part of it
    check(big[:, :, :1000], scores, 8)
    check(big[:, :, 3:1000], scores, 8)       # rows that start anywhere
    check(big[:, ::2, 1:900], scores[:, ::2], 8)
    check(big.transpose(0, 1)[:3, :3, :999], scores[:3, :3], 4)
    check(big[:, 1:2, :998], scores[:, 1:2], 4)


def test_select_scores_that_lie_close():
    """Two beams whose candidates differ by less than a rounding of fp32 at their size."""
    logits = torch.zeros(1, 2, 4096, device="cuda")
    logits[0, 0, 7] = 9.0
    logits[0, 1, 8] = 9.0
    scores = torch.tensor([[-100.0, -100.0]], device="cuda")
    logits[0, 1, 9] = -0.02                   # a little less in the sum: this beam's candidates are better by 1.6e-6 (a step at 100 is 7.6e-6)
    _, parents, tokens = check(logits, scores, 2)
    assert parents.tolist() == [[1, 0]] and tokens.tolist() == [[8, 7]]


def test_select_captured_on_another_stream_twice_at_once():
    from fastforwardattention_b200 import beam_select

    a, sa = candidates(torch.bfloat16, 4, 4, 5003, seed=5)
    b, sb = candidates(torch.bfloat16, 4, 4, 5003, seed=6)
    want = [beam_select(x, s, 8) for x, s in ((a, sa), (b, sb))]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam_select(a, sa, 8)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            again = beam_select(b, sb, 8)
    torch.cuda.synchronize()
    for x, y in zip((got, again), want):
        assert all(torch.equal(i, j) for i, j in zip(x, y))


def test_select_refusals():
    from fastforwardattention_b200 import beam_select

    x, s = candidates(torch.float16, 2, 4, 100)
    for args, kw, match in [((x.cpu(), s, 4), {}, "CUDA"), ((x.double(), s, 4), {}, "unsupported"), ((x[0], s, 4), {}, "logits"), ((x, s.half(), 4), {}, "scores"),
                            ((x, s[:, :2], 4), {}, "scores"), ((x, s, 0), {}, "num"), ((x, s, 65), {}, "num"), ((x, s, 4), dict(pad_token=100), "pad_token"),
                            ((x, s, 4), dict(finished=torch.zeros(2, 4, device="cuda")), "finished"),
                            ((torch.zeros(1, 33, 8, device="cuda"), torch.zeros(1, 33, device="cuda"), 4), {}, "at most 32")]:
        with pytest.raises(RuntimeError, match=match):
            beam_select(*args, **kw)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("groups,beams", [(1, 1), (3, 2), (2, 4), (1, 5), (2, 8), (1, 11), (1, 32)])
def test_reorder(dt, D, groups, beams):
    from fastforwardattention_b200 import FastForwardAttn

    g = torch.Generator("cuda").manual_seed(beams)
    H, L = 3, 70
    kc, vc = (torch.randn(groups * beams, H, L, D, generator=g, device="cuda").to(dt) for _ in range(2))
    ffa = FastForwardAttn.adopt(kc, vc)
    for kind, (first, rows) in zip(("random", "cycle", "one", "same"), ((0, L), (13, 14), (7, 61), (0, L))):
        if kind == "random":
            parents = torch.randint(0, beams, (groups, beams), generator=g, device="cuda")
        elif kind == "cycle":
            parents = (torch.arange(beams, device="cuda") + 1).remainder(beams).expand(groups, beams)
        else:
            parents = torch.full((groups, beams), beams - 1, device="cuda") if kind == "one" else torch.arange(beams, device="cuda").expand(groups, beams)
        parents = parents.int()
        want = [D64.reorder(c, parents, first, rows) for c in (kc, vc)]
        ffa.reorder(parents, rows, first_row=first)
        assert torch.equal(kc, want[0]) and torch.equal(vc, want[1]), kind
    ffa.reorder(parents, 9, first_row=9)
    assert ffa.device_status() == 0


def test_reorder_refusals():
    from fastforwardattention_b200 import FastForwardAttn

    kc, vc = (torch.randn(6, 2, 30, 64, device="cuda") for _ in range(2))
    ffa = FastForwardAttn.adopt(kc, vc)
    kb = kc.clone()
    ffa.reorder(torch.tensor([[1, 0, 3], [2, 2, 2]], dtype=torch.int32, device="cuda"), 20)
    assert ffa.device_status() == 4
    assert torch.equal(kc[:3], kb[:3]) and torch.equal(kc[3, :, :20], kb[5, :, :20])
    ffa.reorder(torch.tensor([[-1, 0, 1], [0, 1, 2]], dtype=torch.int32, device="cuda"), 20)
    assert ffa.device_status() == 4
    good = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for args, kw, match in [((good.long(), 20), {}, "parents"), ((good[:1], 20), {}, "parents"), ((good.cpu(), 20), {}, "parents"), ((good, 31), {}, "rows"),
                            ((good, 20), dict(first_row=21), "rows"), ((good, 20), dict(first_row=-1), "rows")]:
        with pytest.raises(RuntimeError, match=match):
            ffa.reorder(*args, **kw)


@pytest.mark.parametrize("dt", DTYPES)
def test_beam_search_as_it_is_used(dt):
    """Steps of a beam search over the engine's caches against the same search on plain tensors that are gathered beam by beam."""
    from fastforwardattention_b200 import FastForwardAttn, beam_select

    B, N, H, D, Lp, V, steps = 2, 4, 2, 64, 40, 777, 6
    g = torch.Generator("cuda").manual_seed(9)
    K, V_ = (torch.randn(B, H, Lp, D, generator=g, device="cuda").to(dt).repeat_interleave(N, 0) for _ in range(2))
    emb = torch.randn(V, H * D, generator=g, device="cuda")
    ffa = FastForwardAttn(K, V_, Lp + steps, False)
    scores = torch.full((B, N), -INF, device="cuda")
    scores[:, 0] = 0
    tokens = torch.zeros(B, N, dtype=torch.int32, device="cuda")
    plain = [K.clone(), V_.clone()]
    history = [[[] for _ in range(N)] for _ in range(B)]
    for t in range(steps):
        x = emb[tokens.flatten().long()].to(dt).view(B * N, H, 1, D)
        out = ffa.attention(x, x, x, D ** -0.5, Lp + t, 0)
        plain = [torch.cat([c, x], 2) for c in plain]
        logits = (out.float().view(B, N, H * D) @ emb.T).to(dt)
        scores, parents, tokens = beam_select(logits, scores, N)
        ffa.reorder(parents, Lp + t + 1, first_row=Lp)
        at = (torch.arange(B, device="cuda")[:, None] * N + parents).flatten().long()
        plain = [c[at] for c in plain]
        history = [[history[b][parents[b, j]] + [int(tokens[b, j])] for j in range(N)] for b in range(B)]
        for c, p in zip(ffa.get_cache(), plain):
            assert torch.equal(c[:, :, : Lp + t + 1], p)
    assert all(len(set(map(tuple, h))) == N for h in history)   # the beams of a sample are different sequences
    assert (scores[:, :-1] >= scores[:, 1:]).all() and ffa.device_status() == 0


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,beams,V,live", [(1, 1, 500, 1), (3, 1, 2047, 1), (1, 4, 700, 1), (40, 8, 1000, 1), (1, 2, 17, 2), (2, 3, 300, 2), (1, 8, 3001, 2)])
@pytest.mark.parametrize("num", [1, 9, 16])
def test_short_vocabularies_and_few_live_beams(dt, B, beams, V, live, num):
    """Fewer parts that hold anything than candidates to find, with and without ties at the border."""
    g = torch.Generator().manual_seed(V + num)
    for ties in (False, True):
        x = torch.randn(B, beams, V, generator=g)
        x = ((x * 2).round() if ties else x).to(dt).cuda()
        scores = -torch.rand(B, beams, generator=g).cuda()
        scores[:, live:] = float("-inf")
        finished = torch.zeros(B, beams, dtype=torch.bool, device="cuda")
        if live > 1:
            finished[:, 1] = True
        check(x, scores, num, finished, V - 1)


@pytest.mark.parametrize("dt", DTYPES)
def test_select_infinitely_good_beams(dt):
    """A score of +inf is above -inf: its beam's tokens are all equally good, the lowest first."""
    logits, scores = candidates(dt, 4, 3, 700, seed=8)
    scores[0, 1], scores[1, 0], scores[1, 2], scores[2, :], scores[3, 2] = INF, INF, INF, INF, INF
    logits[0, 1, 1] = -INF                    # no candidate
    finished = torch.zeros(4, 3, dtype=torch.bool, device="cuda")
    finished[3, 2] = True
    from fastforwardattention_b200 import beam_select

    want, parents, tokens = D64.beam_select(logits, scores, 9, finished, 5)
    got = beam_select(logits, scores, 9, finished=finished, pad_token=5)
    assert torch.equal(got[1].cpu(), parents) and torch.equal(got[2].cpu(), tokens)
    assert torch.equal(got[0].cpu() == INF, want == INF) and (want[0] == INF).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,N", [(1, 2), (149, 16)])
def test_select_sums_of_long_vocabularies(dt, B, N):
    """Equal terms whose fp32 sum would lose a part of the same sign at every addition: the scores are exact to one rounding and to what
    the kernel states for the log-sum (here, with arguments of 0.3: 2^-22 + 0.3 x 2.5 x 2^-24 + 11 x 2^-24 + 2^-22 = 1.2e-6), and two beams that lie
    further apart come in the right order."""
    from fastforwardattention_b200 import beam_select

    V = 50400
    logits = torch.full((B, N, V), -0.3001, device="cuda").to(dt)
    logits[:, :, :256] = 0.0                  # every lane starts with the largest logit
    logits[:, 1, 256:] = torch.tensor(-0.3301, device="cuda").to(dt)
    exact = torch.logsumexp(logits[0].double(), -1)
    # the first beam's best tokens are 4e-6 better than the second's
    scores = torch.full((B, N), -50.0, device="cuda")
    scores[:, 0], scores[:, 1] = 0.0, (exact[1] - exact[0] - 4e-6).float()
    s = scores[0].double()[:, None] + (0.0 - exact[:, None])
    gap = float(s[0] - s[1])
    assert 3.7e-6 < gap < 4.3e-6
    best, parents, tokens = beam_select(logits, scores, 8)
    assert (parents == 0).all() and (tokens == torch.arange(8, device="cuda")).all()
    assert ((best.double() - s[0]).abs() <= D64.U * s[0].abs() + 1.2e-6).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("kind", ["random", "ascending", "steep"])
def test_select_log_sums_are_as_exact_as_stated(dt, kind):
    """The kernel states 3e-6 for a log-sum, whatever the batch (the cluster of a sample shrinks with it) and the order of the logits."""
    from fastforwardattention_b200 import beam_select

    g = torch.Generator("cuda").manual_seed(9)
    for B, N, V in [(1, 3, 50272), (40, 8, 50400), (149, 16, 50400)]:
        if kind == "random":
            logits = torch.randn(B, N, V, generator=g, device="cuda") * torch.linspace(0.5, 6, N, device="cuda")[:, None]
        else:
            ramp = torch.linspace(-1, 0, V, device="cuda") * (2.0 if kind == "ascending" else 300.0)
            logits = ramp * torch.linspace(0.3, 1, N, device="cuda")[:, None] + torch.zeros(B, 1, 1, device="cuda")
        logits = logits.to(dt)
        scores = torch.randn(B, N, generator=g, device="cuda")
        best, parents, tokens = beam_select(logits, scores, 8)
        for b in (0, B - 1):
            x = logits[b].double()
            s = scores[b].double()[:, None] + (x - torch.logsumexp(x, -1, keepdim=True))
            want = s[parents[b].long(), tokens[b].long()]
            assert ((best[b].double() - want).abs() <= D64.U * want.abs() + 3e-6).all(), (kind, B)
            assert (want >= s.flatten().topk(8).values - 6e-6).all()
