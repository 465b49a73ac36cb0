"""Decoding over a bounded KV cache in float64 on the CPU (test infrastructure only).

The reference has no counterpart; the definitions are those of include/flash_evict.h
(fe_decode_attention, fe_replay_path, fe_insert_tokens), taken one head at a time. `attend` and
`replay` also return what a tolerance needs: sums of absolute values next to the sums.
"""
import math

import torch


def _head(x, *at):
    return x[at].detach().cpu().double()


def visible(tree, t):
    """Bool [t, t]: the causal chunk where there is no tree."""
    return torch.ones((t, t), dtype=torch.bool).tril() if tree is None else tree.cpu()


def attend(q, k, v, k_cache, v_cache, length, tree=None, scale=None, importance=None, value_norm=None, recency_decay=0.):
    """dict: out, lse, mass_v (sum p |v|), sum_v (sum |v| over visible keys), dots (largest
    scale * sum |q k| of a row) and, with importance, importance, new_importance and the part of each
    that this call added (added, new_importance itself)."""
    b, hq, t, d = q.shape
    hk, c = k_cache.shape[1:3]
    g = hq // hk
    scale = d ** -0.5 if scale is None else scale
    r = {"out": torch.zeros((b, hq, t, d), dtype=torch.float64), "lse": torch.full((b, hq, t), -math.inf, dtype=torch.float64)}
    r["mass_v"], r["sum_v"], r["dots"] = torch.zeros_like(r["out"]), torch.zeros_like(r["out"]), torch.zeros((b, hq, t), dtype=torch.float64)
    added, new = torch.zeros((b, hk, c), dtype=torch.float64), torch.zeros((b, hk, t), dtype=torch.float64)
    w = torch.tensor([math.exp(recency_decay * (i - (t - 1))) for i in range(t)], dtype=torch.float64)
    for i in range(b):
        see_new = visible(tree if tree is None or tree.ndim == 2 else tree[i], t)
        for j in range(hk):
            n = min(max(int(length[i, j]), 0), c)
            kc, vc = _head(k_cache, i, j)[:n], _head(v_cache, i, j)[:n]
            kn, vn = _head(k, i, j), _head(v, i, j)
            for h in range(j * g, (j + 1) * g):
                for u in range(t):
                    seen = see_new[u].nonzero().flatten()
                    keys, vals = torch.cat((kc, kn[seen])), torch.cat((vc, vn[seen]))
                    if not len(keys):
                        continue
                    row = _head(q, i, h, u)
                    x = scale * (keys @ row)
                    z = torch.logsumexp(x, 0)
                    p = torch.exp(x - z)
                    r["out"][i, h, u], r["lse"][i, h, u] = p @ vals, z
                    r["mass_v"][i, h, u], r["sum_v"][i, h, u] = p @ vals.abs(), vals.abs().sum(0)
                    r["dots"][i, h, u] = (keys.abs() @ row.abs()).max() * abs(scale)
                    added[i, j, :n] += w[u] * p[:n]
                    new[i, j, seen] += w[u] * p[n:]
            if value_norm is not None:
                added[i, j, :n] *= _head(value_norm, i, j)[:n]
                new[i, j] *= vn.abs().sum(1)
    if importance is not None:
        out = importance.detach().cpu().double().clone()
        for i in range(b):
            for j in range(hk):
                n = min(max(int(length[i, j]), 0), c)
                out[i, j, :n] = out[i, j, :n] * math.exp(-recency_decay * t) + added[i, j, :n]
        r.update(importance=out, new_importance=new, added=added)
    return r


def path_nodes(path, i, t):
    """Batch row i's accepted nodes: up to the first entry outside [0, t); all t without a path."""
    if path is None:
        return list(range(t))
    nodes = []
    for x in path[i].tolist():
        if not 0 <= x < t:
            break
        nodes.append(x)
    return nodes


def replay(q, k, v, k_cache, length, lse, path, importance, scale=None, value_norm=None, recency_decay=0.):
    """dict: importance, new_importance, added, dots (largest scale * sum |q k|)."""
    b, hq, t, d = q.shape
    hk, c = k_cache.shape[1:3]
    g = hq // hk
    a = t if path is None else path.shape[1]
    scale = d ** -0.5 if scale is None else scale
    out = importance.detach().cpu().double().clone()
    added, new = torch.zeros((b, hk, c), dtype=torch.float64), torch.zeros((b, hk, a), dtype=torch.float64)
    dots = 0.
    for i in range(b):
        nodes = path_nodes(path, i, t)
        for j in range(hk):
            n = min(max(int(length[i, j]), 0), c)
            kc, kn, vn = _head(k_cache, i, j)[:n], _head(k, i, j), _head(v, i, j)
            for at, u in enumerate(nodes):
                w = math.exp(recency_decay * (at - (len(nodes) - 1)))
                for h in range(j * g, (j + 1) * g):
                    z = float(lse[i, h, u])
                    if z == -math.inf:
                        continue
                    row = _head(q, i, h, u)
                    own = kn[nodes[:at + 1]]
                    added[i, j, :n] += w * torch.exp(scale * (kc @ row) - z)
                    new[i, j, :at + 1] += w * torch.exp(scale * (own @ row) - z)
                    dots = max(dots, float((torch.cat((kc, own)).abs() @ row.abs()).max()) * abs(scale))
            if value_norm is not None:
                added[i, j, :n] *= _head(value_norm, i, j)[:n]
                new[i, j, :len(nodes)] *= vn[nodes].abs().sum(1)
            out[i, j, :n] = out[i, j, :n] * math.exp(-recency_decay * len(nodes)) + added[i, j, :n]
    return {"importance": out, "new_importance": new, "added": added, "dots": dots}


def insert(cache, k, v, budget, recent=0, new_importance=None, path=None):
    """The rule on a dict of CPU tensors (k, v, importance, position, value_norm or None, length,
    seen), in place: rank, cut, fill."""
    hk, c = cache["k"].shape[1:3]
    for i in range(cache["k"].shape[0]):
        nodes = [] if k is None else path_nodes(path, i, k.shape[2])
        for j in range(hk):
            n, first = min(max(int(cache["length"][i, j]), 0), c), int(cache["seen"][i, j])
            weight = cache["importance"][i, j, :n].tolist()
            weight += [0.] * len(nodes) if new_importance is None else new_importance[i, j, :len(nodes)].tolist()
            place = cache["position"][i, j, :n].tolist() + [first + x for x in range(len(nodes))]
            final = min(n + len(nodes), budget)
            held = first + len(nodes) - recent

            def rank(x):
                w = weight[x]
                if place[x] >= held:
                    return (0, 0., x)                 # protected: by slot alone
                return (1, 0., x) if math.isnan(w) else (2, -w, x)

            kept = set(sorted(range(len(weight)), key=rank)[:final])
            holes = [x for x in range(final) if x not in kept]
            movers = [x for x in sorted(kept) if x >= final]
            assert len(holes) == len(movers)
            for src, dst in list(zip(movers, holes)) + [(x, x) for x in sorted(kept) if n <= x < final]:
                for name, new in (("k", k), ("v", v)):
                    cache[name][i, j, dst] = new[i, j, nodes[src - n]] if src >= n else cache[name][i, j, src].clone()
                if cache["value_norm"] is not None:
                    cache["value_norm"][i, j, dst] = (v[i, j, nodes[src - n]].double().abs().sum() if src >= n
                                                      else cache["value_norm"][i, j, src].clone())
                cache["importance"][i, j, dst] = weight[src]
                cache["position"][i, j, dst] = place[src]
            cache["length"][i, j], cache["seen"][i, j] = final, first + len(nodes)
    return cache
