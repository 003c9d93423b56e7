"""Plain 64-bit definitions of the decoding strategies over the caches (drafted trees, eviction by accumulated weight, beam
search), and the error bounds their kernels are held to.  CPU or GPU tensors; nothing here is fast."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24   # half a step of fp32


def half_step(dtype) -> float:
    """Relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def tree_attention(q, k, v, k_cache, v_cache, tree, scale, rows, first=None):
    """q [B, G*H, T, D]; k, v [B, H, T, D]; caches [B, H, L, D]; rows, first: per-sample lists.  Returns (out, bound) in float64:
    the exact result of these inputs and how far a kernel of q's dtype may be from it."""
    B, HG, T, D = q.shape
    H = k.shape[1]
    G = HG // H
    out = torch.zeros(B, HG, T, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n, lo = int(rows[b]), int(first[b]) if first is not None else 0
        see = tree[b] if tree.dim() == 3 else tree
        see = torch.cat([torch.ones(T, n - lo, dtype=torch.bool, device=q.device), see.bool()], 1)
        for h in range(H):
            keys = torch.cat([k_cache[b, h, lo:n], k[b, h]]).double()
            vals = torch.cat([v_cache[b, h, lo:n], v[b, h]]).double()
            for g in range(G):
                x = q[b, h * G + g].double()
                s = torch.where(see, (x @ keys.T) * scale, -math.inf)
                m = s.amax(-1, keepdim=True)
                p = torch.where(see, (s - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
                total = p.sum(-1, keepdim=True)
                p = torch.where(total == 0, 0.0, p / total)   # a NaN score makes its row NaN
                # a token that a row does not see has no part in it, whatever its values: 0 * inf is not formed
                o = torch.stack([p[t][see[t]] @ vals[see[t]] for t in range(T)])
                a = torch.stack([p[t][see[t]] @ vals[see[t]].abs() for t in range(T)])
                out[b, h * G + g] = o
                # dot product: D products and sums in fp32, one product with the scale; exp: its argument's rounding and two more steps
                mag = torch.where(see, (x.abs() @ keys.abs().T) * abs(scale), 0.0)
                ds = (D + 2) * U * mag.nan_to_num(0, 0, 0).amax(-1, keepdim=True)
                smax = torch.where(see, s.abs(), 0.0).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
                dp = ds + 4 * U * (1 + smax)
                rel = 2 * dp + (n - lo + T + 8) * U
                err = rel * a
                if q.dtype != torch.float32:
                    # weights rounded to the tensors' type, with up to 32 query rows as sums of two numbers of it; exponentials to 2.7e-6, in the weights and
                    # in their sum
                    err = err + (half_step(q.dtype) ** (2 if G * T <= 32 else 1) + 6e-6) * a
                    if q.dtype == torch.float16:                   # what is below half of fp16's smallest step, of 2^7 times a weight
                        err = err + 2.0 ** -32 * torch.stack([vals[see[t]].abs().sum(0) for t in range(T)])
                bound[b, h * G + g] = err + half_step(q.dtype) * (o.abs() + err) + 1e-30
    return out, bound


def tree_accept(cache, path, rows):
    """cache [B, H, L, D] -> a copy with rows n + path[b][i] at n + i."""
    out = cache.clone()
    for b, p in enumerate(path):
        for i, j in enumerate(p):
            out[b, :, rows[b] + i] = cache[b, :, rows[b] + j]
    return out


def assert_within(got, want, bound, what=""):
    """Element by element; infinities and NaN have to be the same."""
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fin), f"{what}: finite values differ"
    assert torch.equal(got[~fin].nan_to_num(7.0, 1e300, -1e300), want[~fin].nan_to_num(7.0, 1e300, -1e300)), f"{what}: infinities differ"
    err = (got - want).abs()[fin]
    over = err > bound[fin]
    assert not over.any(), f"{what}: {int(over.sum())} of {over.numel()} off, worst {(err / bound[fin]).max().item():.2f} x the bound"


def step_weights(q, k, v, k_cache, v_cache, scale, rows):
    """One accumulating step: (out [B, H, D], its bound, p [B, H, L] with p[.., rows[b]] the new token's, p's bound), float64."""
    B, H, L, D = k_cache.shape
    one = torch.ones(1, 1, dtype=torch.bool, device=q.device)
    out, bound = tree_attention(q.view(B, H, 1, D), k.view(B, H, 1, D), v.view(B, H, 1, D), k_cache, v_cache, one, scale, rows)
    p = torch.zeros(B, H, L, dtype=torch.float64, device=q.device)
    pb = torch.zeros_like(p)
    for b in range(B):
        n = int(rows[b])
        for h in range(H):
            keys = torch.cat([k_cache[b, h, :n], k.view(B, H, D)[b, h][None]]).double()
            x = q.view(B, H, D)[b, h].double()
            s = keys @ x * scale
            w = torch.softmax(s, 0)
            mag = ((keys.abs() @ x.abs()) * abs(scale)).max()
            rel = 2 * ((D + 2) * U * mag + 4 * U * (1 + s.abs().max())) + (n + 8) * U
            p[b, h, : n + 1], pb[b, h, : n + 1] = w, rel * w
    return out[:, :, 0], bound[:, :, 0], p, pb


def evict(caches, weights, positions, rows, keep, recent, first):
    """Plain eviction of copies: (caches, weights, positions, kept)."""
    caches = [c.clone() for c in caches]
    weights, positions = weights.clone(), positions.clone()
    B, H = weights.shape[:2]
    kept = torch.full((B, H, keep), -1, dtype=torch.int32, device=weights.device)
    for b in range(B):
        n = int(rows[b])
        for h in range(H):
            src = list(range(min(n, keep)))
            if n > keep:
                w = weights[b, h, :n].tolist()
                p = positions[b, h, :n].tolist()
                newest = max(p)
                safe = [x > newest - recent or x < first for x in p]
                value = [-math.inf if x != x else x for x in w]
                order = sorted(range(n), key=lambda r: (not safe[r], 0.0 if safe[r] else -value[r], 0 if safe[r] else w[r] != w[r], r))
                stay = set(order[:keep])
                freed = [r for r in range(keep) if r not in stay]
                for d, s in zip(freed, sorted(r for r in stay if r >= keep)):
                    src[d] = s
                at = torch.tensor(src, device=weights.device)
                for c in (*caches, weights, positions):
                    c[b, h, :keep] = c[b, h][at].clone()
            kept[b, h, : len(src)] = torch.tensor(src, dtype=torch.int32)
    return caches, weights, positions, kept


def beam_select(logits, scores, num, finished=None, pad_token=0):
    """(scores float64, parents, tokens) by sorting every candidate."""
    B, N, V = logits.shape
    rows = []
    for b in range(B):
        cand = []
        for i in range(N):
            s0 = float(scores[b, i])
            if finished is not None and bool(finished[b, i]):
                cand.append((s0, i, pad_token))
                continue
            x = logits[b, i].double().cpu()
            if torch.isnan(x).any() or (x == math.inf).any() or not (s0 > -math.inf):
                continue
            s = torch.where(x > -math.inf, s0 + (x - torch.logsumexp(x, 0)), -math.inf)   # (+inf + -inf is no score either)
            cand += [(float(s[t]), i, t) for t in torch.argsort(s, descending=True, stable=True)[:num].tolist()]
        cand = sorted((c for c in cand if c[0] > -math.inf), key=lambda c: (-c[0], c[1], c[2]))
        rows.append((cand + [(-math.inf, 0, pad_token)] * num)[:num])
    t = torch.tensor(rows, dtype=torch.float64)
    return t[..., 0], t[..., 1].int(), t[..., 2].int()


def reorder(cache, parents, first_row, rows):
    out = cache.clone()
    N = parents.shape[1]
    for g, ps in enumerate(parents.tolist()):
        for j, p in enumerate(ps):
            out[g * N + j, :, first_row:rows] = cache[g * N + p, :, first_row:rows]
    return out
