"""Measured calls of the decoding strategies over the KV caches, beside their plain forms in elementary torch operations.

Three operators, each with its step and the movement of cache rows that follows it:
  tree     attention of a tree of drafted tokens over a cache, then acceptance of a verified path
  evict    a decode step that accumulates attention weights, then eviction down to a budget of rows
  beam     selection over beams and vocabulary, and the reordering of the caches by parent beam
"""
import math

import numpy
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # a handful of drafted tokens for one fp32 sequence of an OPT-1.3B-shaped layer: launch latency counts
        dict(name="tree fp32 batch 1", op="tree", dtype="f32", B=1, H=32, G=1, D=64, n=995, T=5, ragged=False, path=3),
        # the fp16 batch of the same decoder, sequences of different lengths, a 27-token tree, then acceptance
        dict(name="tree fp16 ragged", op="tree", dtype="f16", B=10, H=32, G=1, D=64, n=1237, T=27, ragged=True, path=6),
        # wide heads, the whole 128-row query tile
        dict(name="tree fp16 wide heads", op="tree", dtype="f16", B=8, H=16, G=1, D=256, n=1920, T=100, ragged=False, path=0),
        # grouped heads (4 query heads a cache head) over a long cache: more query rows than one tile holds
        dict(name="tree bf16 grouped long", op="tree", dtype="bf16", B=2, H=8, G=4, D=128, n=32705, T=33, ragged=False, path=8),
        # the largest: a 64-token tree for every sequence of a large batch
        dict(name="tree bf16 large", op="tree", dtype="bf16", B=32, H=32, G=1, D=128, n=8128, T=64, ragged=False, path=0),
        # one generated token under a budget: accumulate, then drop one row; one sequence, fp32
        dict(name="evict step fp32 batch 1", op="step", dtype="f32", B=1, H=32, D=64, n=500, recent=125, first=4),
        # the same loop over a large batch
        dict(name="evict step bf16 large", op="step", dtype="bf16", B=32, H=32, D=128, n=2047, recent=512, first=4),
        # a finished prompt cut down to its budget: fp16 ragged batch
        dict(name="evict prompt fp16 ragged", op="evict", dtype="f16", B=10, H=32, D=64, n=1000, keep=333, recent=101, first=0, ragged=True),
        # selection for one sample's four beams over the OPT vocabulary: latency
        dict(name="beam select fp16 one", op="select", dtype="f16", B=1, beams=4, V=50272, num=8, finished=False),
        # selection for many samples over the GPT-J vocabulary, some beams finished
        dict(name="beam select bf16 many", op="select", dtype="bf16", B=32, beams=8, V=50400, num=16, finished=True),
        # caches of two samples' five beams behind a prompt that they share
        dict(name="beam reorder fp16 shared", op="reorder", dtype="f16", B=2, beams=5, H=32, D=64, n=1256, start=1000),
        # whole caches of a large batch
        dict(name="beam reorder bf16 large", op="reorder", dtype="bf16", B=8, beams=4, H=32, D=128, n=2048, start=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["tree", "tree", "step", "evict", "select", "reorder"])
    most = {"tree": 4.3e9, "step": 1.0e9, "evict": 1.0e9, "reorder": 1.0e9}
    while True:
        if op == "select":
            c = dict(op=op, dtype=dtype, B=_log(rng, 1, 32), beams=rng.randint(1, 8), V=_log(rng, 500, 50400), num=rng.randint(1, 16),
                     finished=rng.random() < 0.5)
            return c
        H, D = rng.choice([4, 8, 16, 32]), rng.choice([64, 80, 128, 256])
        c = dict(op=op, dtype=dtype, B=_log(rng, 1, 32), H=H, D=D)
        if op == "tree":
            c.update(G=rng.choice([1, 1, 2, 4, 8]), n=_log(rng, 1, 32768), T=_log(rng, 1, 100), ragged=rng.random() < 0.5)
            c["path"] = rng.randint(0, min(c["T"], 8))
            if c["G"] * c["T"] > 256:
                continue
        elif op == "step":
            n = _log(rng, 8, 8192)
            c.update(n=n, recent=rng.randint(0, n // 2), first=rng.randint(0, min(4, n // 4)))
        elif op == "evict":
            n = _log(rng, 16, 8192)
            keep = rng.randint(max(1, n // 8), n)
            c.update(n=n, keep=keep, recent=rng.randint(0, keep // 2), first=rng.randint(0, keep // 4), ragged=rng.random() < 0.5)
        else:
            n = _log(rng, 4, 8192)
            c.update(B=_log(rng, 1, 8), beams=rng.randint(2, 8), n=n, start=rng.randint(0, n - 1))
        rows = c["B"] * c.get("beams", 1) * H * c["n"]
        cache = 2 * rows * D * SIZES[dtype]
        flops = 4 * rows * D * c.get("G", 1) * c.get("T", 1)
        if cache <= most[op] and flops <= (275e9 if dtype != "f32" else 30e9):
            return c


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=g)
    return x if scale == 1.0 else x.mul_(scale)


def _lengths(c):
    """Rows of each sequence before the call: a third of the length apart at most where they differ."""
    return [c["n"] - (b * 61) % (c["n"] // 3 + 1) if c.get("ragged") else c["n"] for b in range(c["B"])]


def _tree(c, seed):
    """Ancestor matrix [B, T, T] of random trees (token j's parent is one of the tokens before it) and a root-to-node path of each."""
    B, T, A = c["B"], c["T"], c["path"]
    g = torch.Generator().manual_seed(seed)
    see = torch.zeros(B, T, T, dtype=torch.bool)
    for j in range(T):
        if j:
            parent = (torch.rand(B, generator=g) * min(j, 16)).long() + max(0, j - 16)
            see[:, j] = see[torch.arange(B), parent]
        see[:, j, j] = True
    path = torch.full((B, max(A, 1)), -1, dtype=torch.int32)
    for b in range(B):
        nodes = see[b, T - 1 - b % 2 if T > 1 else 0].nonzero().flatten()[:A]
        path[b, : len(nodes)] = nodes.int()
    return see.cuda(), path.cuda()


def prepare(case, seed):
    c = case
    dt = DTYPES[c["dtype"]]
    g = torch.Generator("cuda").manual_seed(seed)
    st = dict(c=c, seed=seed)
    if c["op"] == "select":
        B, N, V = c["B"], c["beams"], c["V"]
        st["logits"] = _normal(g, (B, N, V), dt, 2.0)
        st["scores"] = _normal(g, (B, N), torch.float32, 3.0)
        st["finished"] = torch.rand(B, N, generator=g, device="cuda") < 0.2 if c["finished"] else None
        return st
    if c["op"] == "reorder":
        B, N = c["B"], c["beams"]
        shape = (B * N, c["H"], c["n"] + 8, c["D"])
        # after a selection about half of the beams go on from another beam's cache
        other = torch.randint(0, N, (B, N), generator=g, device="cuda")
        stay = torch.rand(B, N, generator=g, device="cuda") < 0.4
        st["parents"] = torch.where(stay, torch.arange(N, device="cuda"), other).int()
    else:
        B = c["B"]
        room = {"tree": c.get("T", 0) + 8, "step": 16, "evict": 0}[c["op"]]
        shape = (B, c["H"], c["n"] + room, c["D"])
        st["rows"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")
    st["k_cache"], st["v_cache"] = _normal(g, shape, dt), _normal(g, shape, dt)
    if c["op"] == "tree":
        T = c["T"]
        st["q"] = _normal(g, (B, c["H"] * c["G"], T, c["D"]), dt)
        st["k"], st["v"] = _normal(g, (B, c["H"], T, c["D"]), dt), _normal(g, (B, c["H"], T, c["D"]), dt)
        st["tree"], st["path"] = _tree(c, seed)
    if c["op"] in ("step", "evict"):
        # weights of a history: a few tokens that much attention went to, many that little went to
        H, L = c["H"], shape[2]
        st["weights"] = torch.empty(B, H, L, device="cuda").exponential_(generator=g).square_()
        st["positions"] = torch.arange(L, dtype=torch.int32, device="cuda").expand(B, H, L).contiguous()
    if c["op"] == "step":
        st["q"], st["k"], st["v"] = (_normal(g, (B, c["H"], 1, c["D"]), dt) for _ in range(3))
        st["grown"] = st["rows"] + 1
        st["seen"] = st["rows"].clone()   # tokens seen so far: the next token's position
    if own:
        from fastforwardattention_b200 import FastForwardAttn

        st["ffa"] = FastForwardAttn.adopt(st["k_cache"], st["v_cache"])
    return st


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    op = state["c"]["op"]
    if op == "tree":
        return _run_tree(state)
    if op == "step":
        return _run_step(state)
    if op == "evict":
        return _run_evict(state)
    return _run_select(state) if op == "select" else _run_reorder(state)


def _run_tree(st):
    c = st["c"]
    scale = c["D"] ** -0.5
    if own:
        ffa = st["ffa"]
        if c["ragged"]:
            out = ffa.tree_attention_per_sample(st["q"], st["k"], st["v"], st["tree"], scale, st["rows"], max_row=c["n"])
            if c["path"]:
                ffa.tree_accept_per_sample(st["path"], st["rows"])
        else:
            out = ffa.tree_attention(st["q"], st["k"], st["v"], st["tree"], scale, c["n"])
            if c["path"]:
                ffa.tree_accept(st["path"], c["n"])
        return dict(out=out, k=st["k_cache"], v=st["v_cache"])
    kc, vc, q = st["k_cache"], st["v_cache"], st["q"]
    B, H, G, T, D, L = c["B"], c["H"], c["G"], c["T"], c["D"], kc.shape[2]
    rows = st["rows"].long()
    batch = torch.arange(B, device=q.device)[:, None]
    at = rows[:, None] + torch.arange(T, device=q.device)
    kc[batch, :, at] = st["k"].transpose(1, 2)
    vc[batch, :, at] = st["v"].transpose(1, 2)
    rel = torch.arange(L, device=q.device) - rows[:, None]                                            # [B, L]: drafted token of a row
    drafted = (rel >= 0) & (rel < T)
    sees = st["tree"].gather(2, rel.clamp(0, T - 1)[:, None, :].expand(B, T, L))
    sees = torch.where(drafted[:, None], sees, (rel < 0)[:, None])                                    # [B, T, L]
    s = torch.matmul(q.float().view(B, H, G * T, D), kc.float().transpose(2, 3)).view(B, H, G, T, L).mul_(scale)
    s.masked_fill_(~sees[:, None, None], -math.inf)
    p = s.sub_(s.amax(-1, keepdim=True)).exp_().view(B, H, G * T, L)
    out = torch.matmul(p, vc.float()).div_(p.sum(-1, keepdim=True)).view(B, H * G, T, D).to(q.dtype)
    if c["path"]:
        path = st["path"].long()
        to = rows[:, None] + torch.arange(path.shape[1], device=q.device)
        src = torch.where(path >= 0, rows[:, None] + path, to)
        kc[batch, :, to] = kc[batch, :, src]
        vc[batch, :, to] = vc[batch, :, src]
    return dict(out=out, k=kc, v=vc)


def _evict_plain(st, rows, keep, recent, first):
    kc, vc, w, pos = st["k_cache"], st["v_cache"], st["weights"], st["positions"]
    B, H, L, D = kc.shape
    r = torch.arange(L, device=kc.device)
    valid = (r < rows[:, None])[:, None].expand(B, H, L)
    newest = pos.masked_fill(~valid, -1).amax(-1, keepdim=True)
    protected = (pos > newest - recent) | (pos < first)
    key = w.masked_fill(protected, math.inf).masked_fill(~valid, -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros_like(valid).scatter_(-1, order, True) & valid
    freed = ~kept[..., :keep] & valid[..., :keep]
    moving = kept & (r >= keep)
    survivors = torch.sort((~moving).to(torch.int8), dim=-1, stable=True).indices[..., :keep]         # rows >= keep that stay, ascending
    rank = (freed.cumsum(-1) - 1).clamp(min=0)
    src = torch.where(freed, survivors.gather(-1, rank), r[:keep])
    wide = src[..., None].expand(B, H, keep, D)
    kc[:, :, :keep] = kc.gather(2, wide)
    vc[:, :, :keep] = vc.gather(2, wide)
    w[..., :keep] = w.gather(2, src)
    pos[..., :keep] = pos.gather(2, src)
    return torch.where(valid[..., :keep], src, -1).int()


def _run_step(st):
    c = st["c"]
    scale, n = c["D"] ** -0.5, c["n"]
    if own:
        ffa = st["ffa"]
        out = ffa.attention_accumulate(st["q"], st["k"], st["v"], scale, st["rows"], st["weights"], st["positions"], st["seen"], max_row=n)
        kept = ffa.evict(st["grown"], st["weights"], st["positions"], n, recent=c["recent"], first=c["first"], max_row=n + 1)
    else:
        kc, vc, q = st["k_cache"], st["v_cache"], st["q"]
        kc[:, :, n] = st["k"][:, :, 0]
        vc[:, :, n] = st["v"][:, :, 0]
        s = torch.matmul(q.float(), kc[:, :, : n + 1].float().transpose(2, 3)).mul_(scale)            # [B, H, 1, n + 1]
        p = s.sub_(s.amax(-1, keepdim=True)).exp_()
        p.div_(p.sum(-1, keepdim=True))
        out = torch.matmul(p, vc[:, :, : n + 1].float())[:, :, 0].to(q.dtype)
        st["weights"][..., n] = 0
        st["weights"][..., : n + 1] += p[:, :, 0]
        st["positions"][..., n] = st["seen"][:, None]
        kept = _evict_plain(st, st["grown"], n, c["recent"], c["first"])
    st["seen"].add_(1)
    return dict(out=out, kept=kept, weights=st["weights"], positions=st["positions"], k=st["k_cache"], v=st["v_cache"])


def _run_evict(st):
    c = st["c"]
    # the trackers start from what the prompt's attention left; the caches' rows behind the budget are never written
    now = dict(st, weights=st["weights"].clone(), positions=st["positions"].clone())
    if own:
        kept = st["ffa"].evict(st["rows"], now["weights"], now["positions"], c["keep"], recent=c["recent"], first=c["first"], max_row=c["n"])
    else:
        kept = _evict_plain(now, st["rows"], c["keep"], c["recent"], c["first"])
    return dict(kept=kept, weights=now["weights"], positions=now["positions"], k=st["k_cache"], v=st["v_cache"])


def _run_select(st):
    c = st["c"]
    if own:
        from fastforwardattention_b200 import beam_select

        return beam_select(st["logits"], st["scores"], c["num"], finished=st["finished"], pad_token=1)
    # scores of different beams lie next to each other: the logarithm of the sum is taken in 64 bits
    x = st["logits"].double()
    B, N, V = x.shape
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    s = st["scores"].double()[..., None] + (x - lse)
    if st["finished"] is not None:
        done = torch.full_like(s, -math.inf)
        done[..., 1] = st["scores"].double()
        s = torch.where(st["finished"][..., None], done, s)
    best, at = torch.sort(s.view(B, N * V), dim=-1, descending=True, stable=True)
    # fewer candidates than asked for: the others are (-inf, beam 0, the pad token)
    best = torch.nn.functional.pad(best[:, : c["num"]], (0, max(0, c["num"] - N * V)), value=-math.inf)
    at = torch.nn.functional.pad(at[:, : c["num"]], (0, max(0, c["num"] - N * V)))
    none = best == -math.inf
    return best.float(), (at // V).masked_fill(none, 0).int(), (at % V).masked_fill(none, 1).int()


def _run_reorder(st):
    c = st["c"]
    n, start = c["n"], c["start"]
    if own:
        st["ffa"].reorder(st["parents"], n, first_row=start)
    else:
        B, N = st["parents"].shape
        src = (torch.arange(B, device="cuda")[:, None] * N + st["parents"]).flatten().long()
        st["k_cache"][:, :, start:n] = st["k_cache"][src, :, start:n]
        st["v_cache"][:, :, start:n] = st["v_cache"][src, :, start:n]
    return dict(k=st["k_cache"], v=st["v_cache"])


def work(case):
    c = case
    s = SIZES[c["dtype"]]
    if c["op"] == "select":
        n = c["B"] * c["beams"] * c["V"]
        return dict(bytes=n * s + c["B"] * c["num"] * 12, flops=3 * n)
    H, D = c["H"], c["D"]
    if c["op"] == "tree":
        B, G, T = c["B"], c["G"], c["T"]
        rows = sum(_lengths(c))
        moved = B * c["path"]
        data = 2 * H * rows * D * s + 4 * B * H * T * D * s + 2 * B * H * G * T * D * s + B * T * T + 4 * H * moved * D * s
        return dict(bytes=data, flops=4 * G * H * T * D * (rows + B * T))
    if c["op"] == "step":
        pairs = c["B"] * H
        return dict(bytes=pairs * (2 * (c["n"] + 6) * D * s + 4 * 3 * c["n"]), flops=4 * pairs * c["n"] * D)
    if c["op"] == "evict":
        # about keep / rows of the rows behind the budget survive and move (K and V, read and written)
        data = 0
        for n in _lengths(c):
            moved = max(0, n - c["keep"]) * c["keep"] / n
            data += H * (8 * n + 4 * c["keep"] + 4 * moved * D * s)
        return dict(bytes=data, flops=4 * H * sum(_lengths(c)))
    moved = 0.6 * (c["beams"] - 1) * c["B"] * H * (c["n"] - c["start"])
    return dict(bytes=4 * moved * D * s + 4 * c["B"] * c["beams"], flops=1)


# ---- the definition, in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    global own
    mine, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = mine
    return {"tree": _exact_tree, "step": _exact_step, "evict": _exact_evict, "select": _exact_select, "reorder": _exact_reorder}[case["op"]](st)


def _softmax_rows(scores):
    """exp(s) / sum exp(s) of each row, 64 bits."""
    e = torch.exp(scores - scores.max(dim=-1, keepdim=True).values)
    return e / e.sum(dim=-1, keepdim=True)


def _exact_tree(st):
    c = st["c"]
    H, G, T, D = c["H"], c["G"], c["T"], c["D"]
    k, v = st["k_cache"], st["v_cache"]
    out = torch.empty(c["B"], H * G, T, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(c)):
        for h in range(H):
            keys = torch.cat([k[b, h, :n], st["k"][b, h]]).double()
            values = torch.cat([v[b, h, :n], st["v"][b, h]]).double()
            hide = torch.cat([torch.zeros(T, n, dtype=torch.bool, device="cuda"), ~st["tree"][b]], 1)
            scores = torch.einsum("gtd,nd->gtn", st["q"][b, h * G:(h + 1) * G].double(), keys) / math.sqrt(D)
            out[b, h * G:(h + 1) * G] = _softmax_rows(scores.masked_fill(hide, -math.inf)) @ values
        order = list(range(T))
        for i, j in enumerate(x for x in st["path"][b].tolist() if x >= 0 and c["path"]):
            order[i] = j
        # a path only ever moves a token down onto one that was moved before or is dropped
        k[b, :, n:n + T], v[b, :, n:n + T] = st["k"][b][:, order], st["v"][b][:, order]
    return dict(out=out, k=k, v=v)


def _exact_drop(st, rows, keep, recent, first):
    """Pair by pair, with sets: what stays, and where it goes."""
    w, pos, k, v = st["weights"], st["positions"], st["k_cache"], st["v_cache"]
    B, H = w.shape[:2]
    kept = torch.full((B, H, keep), -1, dtype=torch.int32)
    wl, pl = w.cpu().numpy(), pos.cpu().numpy()
    to, frm = [], []
    for b in range(B):
        n = int(rows[b])
        for h in range(H):
            kept[b, h, : min(n, keep)] = torch.arange(min(n, keep), dtype=torch.int32)
            if n <= keep:
                continue
            newest = pl[b, h, :n].max()
            safe = (pl[b, h, :n] > newest - recent) | (pl[b, h, :n] < first)
            rank = numpy.lexsort((numpy.arange(n), -wl[b, h, :n], ~safe))   # protected rows, then by weight, then by row
            if safe.sum() >= keep:
                rank = numpy.flatnonzero(safe)
            stay = set(rank[:keep].tolist())
            holes = [r for r in range(keep) if r not in stay]
            for d, s in zip(holes, sorted(r for r in stay if r >= keep)):
                kept[b, h, d] = s
                to.append((b, h, d))
                frm.append((b, h, s))
    if to:
        t, f = torch.tensor(to, device="cuda").T, torch.tensor(frm, device="cuda").T
        for x in (k, v, w, pos):
            x[t[0], t[1], t[2]] = x[f[0], f[1], f[2]]
    return kept.cuda()


def _exact_step(st):
    c = st["c"]
    n, scale = c["n"], 1 / math.sqrt(c["D"])
    if c["B"] * c["H"] * n > 20_000_000:
        return None
    k, v = st["k_cache"], st["v_cache"]
    k[:, :, n], v[:, :, n] = st["k"][:, :, 0], st["v"][:, :, 0]
    p = _softmax_rows(torch.einsum("bhd,bhnd->bhn", st["q"][:, :, 0].double(), k[:, :, : n + 1].double()) * scale)
    out = torch.einsum("bhn,bhnd->bhd", p, v[:, :, : n + 1].double())
    w = st["weights"].double()
    w[..., : n] += p[..., : n]
    w[..., n] = p[..., n]
    st["weights"] = w
    st["positions"][..., n] = n
    kept = _exact_drop(st, st["grown"].tolist(), n, c["recent"], c["first"])
    return dict(out=out, kept=kept, weights=w, positions=st["positions"], k=k, v=v)


def _exact_evict(st):
    c = st["c"]
    if c["B"] * c["H"] * c["n"] > 20_000_000:
        return None
    kept = _exact_drop(st, st["rows"].tolist(), c["keep"], c["recent"], c["first"])
    return dict(kept=kept, weights=st["weights"].double(), positions=st["positions"], k=st["k_cache"], v=st["v_cache"])


def _exact_select(st):
    c = st["c"]
    rows = []
    for b in range(c["B"]):
        cand = []
        for i in range(c["beams"]):
            s0 = float(st["scores"][b, i])
            if st["finished"] is not None and bool(st["finished"][b, i]):
                cand.append((-s0, i, 1))
                continue
            x = st["logits"][b, i].double().cpu()
            lse = float(torch.logsumexp(x, 0))
            some = torch.topk(x, min(c["V"], c["num"])).values[-1]   # no other logit of the beam can be chosen; equal ones by index
            for t in (x >= some).nonzero().flatten().tolist():
                cand.append((-(s0 + (float(x[t]) - lse)), i, t))
        rows.append((sorted(cand) + [(math.inf, 0, 1)] * c["num"])[: c["num"]])
    made = lambda k, dt: torch.tensor([[x[k] for x in r] for r in rows], dtype=dt, device="cuda")  # noqa: E731
    return -made(0, torch.float64), made(1, torch.int32), made(2, torch.int32)


def _exact_reorder(st):
    c = st["c"]
    N = c["beams"]
    for x in (st["k_cache"], st["v_cache"]):
        for b, parents in enumerate(st["parents"].tolist()):
            before = x[b * N:(b + 1) * N].clone()
            for j, p in enumerate(parents):
                x[b * N + j, :, c["start"]:c["n"]] = before[p, :, c["start"]:c["n"]]
    return dict(k=st["k_cache"], v=st["v_cache"])
