"""Decoding over a bounded KV cache: the operators' cases, their plain forms and their values in 64 bits.

Three operators of flash_evict, which a serving loop runs one after the other on each layer:

  attend   decode_attention: T new tokens (one token, a causal chunk, or a tree of drafted tokens) attend over
           a cache of `length` rows and over each other; for tokens that stay, the attention weight each cache
           row received is added to its importance
  replay   replay_path: the accepted path of a drafted tree, whose rows' weights reach the importance after the
           verification (the rejected rows' do not)
  insert   insert_tokens: new tokens enter a cache of bounded size; the rows of least importance leave it

A case is a dict of sizes; `prepare` makes its tensors, `run` one pass. With `own` false a pass is computed in
elementary torch operations in 32 bits, with `own` true by the package's calls.
"""
import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-evict-prefill_amd")
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
RECENT = 64        # newest tokens an insertion never evicts, where the cache is large enough
DECAY = 0.1        # recency decay of the importance


def _calls():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import flash_evict
    return flash_evict


# ---------------------------------------------------------------------------------------------- cases

def _case(name, op, batch, heads, kv_heads, dim, cache, tokens, dtype="bf16", **more):
    return dict(name=name, op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, tokens=tokens,
                dtype=dtype, **more)


def listed():
    return [
        # one request, a cache evicted to 1024 tokens: the latency of a decode step
        _case("step 1024", "attend", 1, 32, 8, 128, 1024, 1, branch=0, ragged=False),
        # a serving batch whose requests are at different points of their generation
        _case("step batch 32", "attend", 32, 28, 4, 128, 8192, 1, branch=0, ragged=True),
        # one request over a long prompt whose cache was kept whole
        _case("step 131072", "attend", 1, 32, 8, 128, 131072, 1, branch=0, ragged=False),
        # a turn of a conversation appended as one causal chunk: odd sizes, a head dim below its tile
        _case("chunk 33", "attend", 3, 8, 2, 80, 5000, 33, "fp16", branch=0, ragged=True),
        # verification of a drafted binary tree over an evicted cache
        _case("tree 64 over 4096", "attend", 8, 32, 8, 128, 4096, 64, branch=2, ragged=True),
        # the same over a long cache, seven query heads to a KV head, a tree that fills no tile
        _case("tree 61 over 32768", "attend", 2, 28, 4, 128, 32768, 61, "fp16", branch=3, ragged=True),
        # four accepted tokens of a small tree, one request
        _case("accept 4 of 16", "replay", 1, 32, 8, 128, 1024, 16, branch=2, accepted=4, ragged=False),
        # up to six accepted tokens of a larger tree over long caches
        _case("accept 6 of 64", "replay", 8, 28, 4, 128, 32768, 64, branch=2, accepted=6, ragged=True),
        # the steady state of a decode loop: one token in, one out of each head's cache
        _case("insert 1 in 1024", "insert", 1, 32, 8, 128, 1024, 1, branch=0, accepted=1),
        # the same for a serving batch
        _case("insert 1 in 8192", "insert", 32, 28, 4, 128, 8192, 1, branch=0, accepted=1),
        # an accepted path enters caches of a tenth of a long prompt
        _case("insert 6 of 64", "insert", 4, 32, 8, 128, 13107, 64, branch=2, accepted=6),
        # a chunk replaces an eighth of small caches of an odd size
        _case("insert 250 in 2000", "insert", 8, 8, 2, 80, 2000, 250, "fp16", branch=0, accepted=250),
    ]


_LARGEST_BYTES = 500e6     # K and V of a cache that a pass reads
_LARGEST_FLOPS = 50e9      # of a pass, narrow heads counted as wide ones


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "replay", "insert"])
    heads, kv_heads = rng.choice([(32, 8), (28, 4), (8, 2), (4, 2), (16, 16), (7, 1)])
    dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
    dtype = rng.choice(["bf16", "fp16"])
    batch = _log(rng, 1, 32)
    if op == "insert":
        cache = _log(rng, 256, 32768)
        while batch > 1 and 4 * batch * kv_heads * cache * dim > _LARGEST_BYTES:
            batch //= 2
        while 4 * batch * kv_heads * cache * dim > _LARGEST_BYTES:
            cache //= 2
        branch = rng.choice([0, 0, 2, 3])
        tokens = _log(rng, 2, 64) if branch else _log(rng, 1, min(256, cache // 2))
        accepted = rng.randint(1, _depth(tokens, branch)) if branch else tokens
        return dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, tokens=tokens, dtype=dtype,
                    branch=branch, accepted=accepted, ragged=rng.random() < 0.3)
    cache = _log(rng, 64, 131072)
    branch = rng.choice([0, 1, 2, 3]) if op == "attend" else rng.choice([1, 2, 3])
    tokens = rng.choice([1, 1, _log(rng, 2, 128)]) if branch == 0 else _log(rng, 2, 128)

    def too_large():
        return (4 * batch * kv_heads * cache * dim > _LARGEST_BYTES
                or 4 * batch * heads * tokens * cache * max(dim, 128) > _LARGEST_FLOPS)

    while batch > 1 and too_large():
        batch //= 2
    while too_large():
        cache //= 2
    case = dict(op=op, batch=batch, heads=heads, kv_heads=kv_heads, dim=dim, cache=cache, tokens=tokens, dtype=dtype,
                branch=branch, ragged=rng.random() < 0.5)
    if op == "replay":
        case["accepted"] = rng.randint(1, min(16, _depth(tokens, branch)))
    return case


# A drafted tree: node 0 is the root, node i's parent is (i - 1) // branch. branch 0: a causal chunk, no tree.
def _ancestors(node, branch):
    """The path from the root to `node`."""
    path = [node]
    while path[-1] > 0:
        path.append((path[-1] - 1) // branch)
    return path[::-1]


def _depth(tokens, branch):
    return len(_ancestors(tokens - 1, branch))


def _tree(case):
    t, branch = case["tokens"], case["branch"]
    mask = torch.zeros((t, t), dtype=torch.bool)
    for i in range(t):
        mask[i, _ancestors(i, branch)] = True
    return mask


def _lengths(case):
    """Rows in each request's cache: all of it, or between half and all of it."""
    c, b = case["cache"], case["batch"]
    return [max(1, c - (i * c) // (2 * b)) if case.get("ragged") else c for i in range(b)]


def _accepted(case):
    """Accepted tokens of each request: all the path has room for, or about half of that."""
    a = case["accepted"]
    if not case["branch"]:
        return [a] * case["batch"]
    return [a if i % 2 == 0 else max(1, a // 2) for i in range(case["batch"])]


# ---------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    b, hq, hk, d, c, t = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "cache", "tokens"))

    def normal(*shape, to=None, std=1.0):
        x = torch.randn(shape, generator=gen, device=dev, dtype=torch.float32)
        return (x if std == 1.0 else x * std).to(to or dtype)

    def cached():      # one batch row at a time: no float copy of a whole cache
        x = torch.empty((b, hk, c, d), dtype=dtype, device=dev)
        for i in range(b):
            x[i] = normal(hk, c, d)
        return x

    s = {"case": dict(case)}
    # projections give [B, T, H, D]; attention takes the transposed view
    s["q"] = normal(b, t, hq, d, std=1.5).transpose(1, 2)
    s["k"] = normal(b, t, hk, d).transpose(1, 2)
    s["v"] = normal(b, t, hk, d).transpose(1, 2)
    s["k_cache"], s["v_cache"] = cached(), cached()
    # a few rows hold most of the accumulated weight, as after a prompt
    s["importance"] = torch.exp(1.5 * normal(b, hk, c, to=torch.float32))
    s["length"] = torch.tensor(_lengths(case), dtype=torch.int32).to(dev)[:, None].expand(b, hk).contiguous()
    if case["op"] == "insert":
        s["seen"] = torch.full((b, hk), 4 * c, dtype=torch.int32, device=dev)
        # the kept positions of a prompt of 4 * c tokens: distinct, in no order after many insertions
        s["position"] = (4 * torch.argsort(torch.rand((b, hk, c), generator=gen, device=dev), dim=-1)
                         + torch.randint(0, 4, (b, hk, c), generator=gen, device=dev)).to(torch.int32)
        s["new_importance"] = torch.exp(1.5 * normal(b, hk, case["accepted"], to=torch.float32))
    s["value_norm"] = torch.stack([s["v_cache"][i].float().abs().sum(-1) for i in range(b)])
    s["tree"] = _tree(case).to(dev) if case["branch"] else None
    if case["op"] == "attend":
        # a tree's weights wait for the verification
        s["importance_out"] = None if case["branch"] else torch.zeros_like(s["importance"])
    else:
        s["path"] = None
        if case["branch"]:
            counts = _accepted(case)
            path = torch.full((b, case["accepted"]), -1, dtype=torch.int32)
            pick = torch.randint(0, 1 << 30, (b,), generator=torch.Generator().manual_seed(seed)).tolist()
            trails = [_ancestors(x, case["branch"]) for x in range(t)]
            for i in range(b):
                ends = [x for x in trails if len(x) == counts[i]]
                path[i, :counts[i]] = torch.tensor(ends[pick[i] % len(ends)], dtype=torch.int32)
            s["path"] = path.to(dev)
    if case["op"] == "replay":
        # log-sum-exp of rows of about normal logits of standard deviation 1.5
        n = s["length"].repeat_interleave(hq // hk, 1)[:, :, None]
        s["lse"] = torch.log(n + 0.5 * t) + 1.125 + 0.1 * normal(b, hq, t, to=torch.float32)
        s["importance_out"] = torch.zeros_like(s["importance"])
    return s


# ---------------------------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if op == "attend":
        return _attend_own(s) if own else _attend_plain(s)
    if op == "replay":
        return _replay_own(s) if own else _replay_plain(s)
    return _insert_own(s) if own else _insert_plain(s)


def _attend_own(s):
    out, lse, imp, new = _calls().decode_attention(
        s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["length"], tree=s["tree"],
        importance=s["importance"] if s["importance_out"] is not None else None,
        value_norm=s["value_norm"] if s["importance_out"] is not None else None,
        recency_decay=DECAY, importance_out=s["importance_out"])
    return {"out": out, "lse": lse} if imp is None else {"out": out, "lse": lse, "importance": imp, "new_importance": new}


def _replay_own(s):
    imp, new = _calls().replay_path(
        s["q"], s["k"], s["v"], s["k_cache"], s["length"], s["lse"], s["path"], s["importance"],
        value_norm=s["value_norm"], recency_decay=DECAY, importance_out=s["importance_out"])
    return {"importance": imp, "new_importance": new}


def _insert_own(s):
    _calls().insert_tokens(
        s["k"], s["v"], s["k_cache"], s["v_cache"], s["importance"], s["position"], s["length"], s["seen"],
        s["case"]["cache"], recent=min(RECENT, s["case"]["cache"] // 4), new_importance=s["new_importance"],
        value_norm=s["value_norm"], path=s["path"])
    return {x: s[x] for x in ("k_cache", "v_cache", "importance", "position", "value_norm", "length", "seen")}


def _attend_plain(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    b, hq, t, d = q.shape
    hk, c = s["k_cache"].shape[1:3]
    g = hq // hk
    keys = torch.cat((s["k_cache"].float(), k), 2)
    values = torch.cat((s["v_cache"].float(), v), 2)
    x = torch.matmul(q.reshape(b, hk, g * t, d), keys.transpose(2, 3)) * d ** -0.5
    tree = s["tree"] if s["tree"] is not None else torch.ones((t, t), dtype=torch.bool, device=q.device).tril()
    there = torch.arange(c, device=q.device) < s["length"][:, :, None]
    seen = torch.cat((there[:, :, None, :].expand(b, hk, t, c), tree.expand(b, hk, t, t)), 3)
    x = x.view(b, hk, g, t, c + t).masked_fill_(~seen[:, :, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x.sub_(m))
    total = p.sum(-1, keepdim=True)
    p /= total
    out = torch.matmul(p.view(b, hk, g * t, c + t), values).view(b, hq, t, d).to(s["q"].dtype)
    lse = (m + torch.log(total)).view(b, hq, t)
    if s["importance_out"] is None:
        return {"out": out, "lse": lse}
    w = torch.exp(-DECAY * torch.arange(t - 1, -1, -1, device=q.device, dtype=torch.float32))
    mass = (p * w[:, None]).sum((2, 3))
    updated = s["importance"] * math.exp(-DECAY * t) + s["value_norm"] * mass[..., :c]
    s["importance_out"].copy_(torch.where(there, updated, s["importance_out"]))
    return {"out": out, "lse": lse, "importance": s["importance_out"],
            "new_importance": v.abs().sum(-1) * mass[..., c:]}


def _replay_plain(s):
    path = s["path"]
    b, hq, t, d = s["q"].shape
    hk, c = s["k_cache"].shape[1:3]
    g, a = hq // hk, path.shape[1]
    taken = path >= 0
    at = path.clamp(min=0).long()
    q = torch.gather(s["q"].float(), 2, at[:, None, :, None].expand(b, hq, a, d))
    lse = torch.gather(s["lse"], 2, at[:, None, :].expand(b, hq, a))
    k = torch.gather(s["k"].float(), 2, at[:, None, :, None].expand(b, hk, a, d))
    v = torch.gather(s["v"].float(), 2, at[:, None, :, None].expand(b, hk, a, d))
    count = taken.sum(1)
    keys = torch.cat((s["k_cache"].float(), k), 2)
    x = torch.matmul(q.reshape(b, hk, g * a, d), keys.transpose(2, 3)).view(b, hk, g, a, c + a) * d ** -0.5
    there = torch.arange(c, device=x.device) < s["length"][:, :, None]
    rows = torch.arange(a, device=x.device)
    before = (rows[None, :] <= rows[:, None])[None] & taken[:, None, :]
    seen = torch.cat((there[:, :, None, :].expand(b, hk, a, c), before[:, None].expand(b, hk, a, a)), 3) & taken[:, None, :, None]
    p = torch.exp(x - lse.view(b, hk, g, a, 1)) * seen[:, :, None]
    w = torch.exp(-DECAY * (count[:, None] - 1 - rows).clamp(min=0).float())
    mass = (p * w[:, None, None, :, None]).sum((2, 3))
    updated = s["importance"] * torch.exp(-DECAY * count.float())[:, None, None] + s["value_norm"] * mass[..., :c]
    s["importance_out"].copy_(torch.where(there, updated, s["importance_out"]))
    return {"importance": s["importance_out"], "new_importance": v.abs().sum(-1) * mass[..., c:]}


def _insert_plain(s):
    b, hk, c, d = s["k_cache"].shape
    a = s["new_importance"].shape[2]
    recent = min(RECENT, c // 4)
    dev = s["length"].device
    n, seen = s["length"][:, :, None].long(), s["seen"][:, :, None].long()
    count = (s["path"] >= 0).sum(1)[:, None, None] if s["path"] is not None else torch.full((b, 1, 1), a, device=dev)
    final = (n + count).clamp(max=c)
    slots = torch.arange(c + a, device=dev)
    # candidates: the cache's slots, then the new rows (slot n + i is new row i)
    new = slots - n
    is_new = (new >= 0) & (new < count)
    there = slots < n + count
    of_new = new.clamp(0, a - 1)
    of_old = slots.clamp(max=c - 1).expand(b, hk, c + a)
    weight = torch.where(is_new, torch.gather(s["new_importance"], 2, of_new), torch.gather(s["importance"], 2, of_old))
    place = torch.where(is_new, seen + new, torch.gather(s["position"], 2, of_old).long())
    held = there & (place >= seen + count - recent)
    # kept: the protected ones, then by importance; equal ones by slot
    weight = torch.where(there, torch.where(held, math.inf, weight), -math.inf)
    order = torch.argsort(weight, dim=-1, descending=True, stable=True)
    rank = torch.empty_like(order).scatter_(2, order, slots.expand(b, hk, c + a))
    keep = there & (rank < final)
    # the i-th kept candidate at or past `final` goes to the i-th vacated slot below it
    hole = ~keep & (slots < final)
    mover = keep & (slots >= final)
    holes = torch.argsort((~hole).to(torch.int8), dim=-1, stable=True)[..., :a]
    movers = torch.argsort((~mover).to(torch.int8), dim=-1, stable=True)[..., :a]
    live = torch.arange(a, device=dev) < mover.sum(-1, keepdim=True)
    # new rows that stay where they were appended
    own_slot = n + torch.arange(a, device=dev)
    stay = torch.gather(keep & is_new & (slots < final), 2, own_slot)
    source, target = torch.cat((movers, own_slot), -1), torch.cat((holes, own_slot), -1)
    which = torch.cat((live, stay), -1)
    bi, hi, ai = torch.nonzero(which, as_tuple=True)
    src, dst = source[bi, hi, ai], target[bi, hi, ai]
    row = src - s["length"][bi, hi].long()
    fresh = row >= 0
    row = row.clamp(min=0)
    token = s["path"][bi, row].long() if s["path"] is not None else row
    old = src.clamp(max=c - 1)
    k_rows = torch.where(fresh[:, None], s["k"][bi, hi, token], s["k_cache"][bi, hi, old])
    v_rows = torch.where(fresh[:, None], s["v"][bi, hi, token], s["v_cache"][bi, hi, old])
    norms = torch.where(fresh, s["v"][bi, hi, token].float().abs().sum(-1), s["value_norm"][bi, hi, old])
    weights = torch.where(fresh, s["new_importance"][bi, hi, row], s["importance"][bi, hi, old])
    places = torch.where(fresh, s["seen"][bi, hi] + row.to(torch.int32), s["position"][bi, hi, old])
    s["k_cache"][bi, hi, dst] = k_rows
    s["v_cache"][bi, hi, dst] = v_rows
    s["value_norm"][bi, hi, dst] = norms
    s["importance"][bi, hi, dst] = weights
    s["position"][bi, hi, dst] = places
    s["length"].copy_(final[..., 0].expand(b, hk))
    s["seen"] += count[..., 0].to(torch.int32)
    return {x: s[x] for x in ("k_cache", "v_cache", "importance", "position", "value_norm", "length", "seen")}


# ---------------------------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _attend_exact(s)
    if case["op"] == "replay":
        return _replay_exact(s)
    return _insert_exact(s)


def _attend_exact(s):
    b, hq, t, d = s["q"].shape
    hk, c = s["k_cache"].shape[1:3]
    g = hq // hk
    weighted = s["importance_out"] is not None
    out = torch.zeros((b, hq, t, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((b, hq, t), dtype=torch.float64, device="cuda")
    imp = torch.zeros((b, hk, c), dtype=torch.float64, device="cuda")
    new = torch.zeros((b, hk, t), dtype=torch.float64, device="cuda")
    tree = s["tree"]
    w = [math.exp(-DECAY * (t - 1 - i)) for i in range(t)]
    for i in range(b):
        for j in range(hk):
            n = int(s["length"][i, j])
            kc, vc = s["k_cache"][i, j, :n].double(), s["v_cache"][i, j, :n].double()
            kn, vn = s["k"][i, j].double(), s["v"][i, j].double()
            for h in range(j * g, (j + 1) * g):
                qh = s["q"][i, h].double() / math.sqrt(d)
                old, fresh = qh @ kc.T, qh @ kn.T
                for u in range(t):
                    hidden = ~tree[u] if tree is not None else torch.arange(t, device="cuda") > u
                    fresh[u][hidden] = -math.inf
                x = torch.cat((old, fresh), 1)
                z = torch.logsumexp(x, 1)
                p = torch.exp(x - z[:, None])
                out[i, h] = p[:, :n] @ vc + p[:, n:] @ vn
                lse[i, h] = z
                if weighted:
                    mass = torch.tensor(w, dtype=torch.float64, device="cuda") @ p
                    imp[i, j, :n] += mass[:n]
                    new[i, j] += mass[n:]
            if weighted:
                imp[i, j, :n] = imp[i, j, :n] * vc.abs().sum(1) + s["importance"][i, j, :n].double() * math.exp(-DECAY * t)
                new[i, j] *= vn.abs().sum(1)
    return {"out": out, "lse": lse, "importance": imp, "new_importance": new} if weighted else {"out": out, "lse": lse}


def _replay_exact(s):
    b, hq, t, d = s["q"].shape
    hk, c = s["k_cache"].shape[1:3]
    g, a = hq // hk, s["path"].shape[1]
    imp = torch.zeros((b, hk, c), dtype=torch.float64, device="cuda")
    new = torch.zeros((b, hk, a), dtype=torch.float64, device="cuda")
    for i in range(b):
        nodes = [x for x in s["path"][i].tolist() if x >= 0]
        w = torch.tensor([math.exp(-DECAY * (len(nodes) - 1 - r)) for r in range(len(nodes))], dtype=torch.float64, device="cuda")
        for j in range(hk):
            n = int(s["length"][i, j])
            kc, kn = s["k_cache"][i, j, :n].double(), s["k"][i, j, nodes].double()
            for h in range(j * g, (j + 1) * g):
                q = s["q"][i, h, nodes].double() / math.sqrt(d)
                z = s["lse"][i, h, nodes].double()[:, None]
                imp[i, j, :n] += w @ torch.exp(q @ kc.T - z)
                new[i, j, :len(nodes)] += w @ torch.exp(q @ kn.T - z).tril()
            imp[i, j, :n] *= s["v_cache"][i, j, :n].double().abs().sum(1)
            imp[i, j, :n] += s["importance"][i, j, :n].double() * math.exp(-DECAY * len(nodes))
            new[i, j, :len(nodes)] *= s["v"][i, j, nodes].double().abs().sum(1)
    return {"importance": imp, "new_importance": new}


def _insert_exact(s):
    """The rule taken literally, one head at a time on the host: sort, cut, fill."""
    b, hk, c, d = s["k_cache"].shape
    recent = min(RECENT, c // 4)
    r = {x: s[x].double().cpu() for x in ("k_cache", "v_cache", "importance", "value_norm")}
    r.update({x: s[x].cpu().clone() for x in ("position", "length", "seen")})
    k, v, fresh = s["k"].double().cpu(), s["v"].double().cpu(), s["new_importance"].double().cpu()
    for i in range(b):
        nodes = [x for x in s["path"][i].tolist() if x >= 0] if s["path"] is not None else list(range(k.shape[2]))
        for j in range(hk):
            n, first = int(r["length"][i, j]), int(r["seen"][i, j])
            weights = r["importance"][i, j, :n].tolist() + fresh[i, j, :len(nodes)].tolist()
            places = r["position"][i, j, :n].tolist() + [first + x for x in range(len(nodes))]
            held = first + len(nodes) - recent
            final = min(n + len(nodes), c)
            ranked = sorted(range(len(weights)), key=lambda x: (places[x] < held, -weights[x], x))
            kept = set(ranked[:final])
            holes = [x for x in range(final) if x not in kept]
            movers = sorted(x for x in kept if x >= final)
            pairs = list(zip(movers, holes)) + [(x, x) for x in range(n, final) if x in kept]
            for src, dst in pairs:
                if src >= n:
                    r["k_cache"][i, j, dst], r["v_cache"][i, j, dst] = k[i, j, nodes[src - n]], v[i, j, nodes[src - n]]
                    r["value_norm"][i, j, dst] = v[i, j, nodes[src - n]].abs().sum()
                else:
                    for x in ("k_cache", "v_cache", "value_norm"):
                        r[x][i, j, dst] = r[x][i, j, src]
                r["importance"][i, j, dst], r["position"][i, j, dst] = weights[src], places[src]
            r["length"][i, j], r["seen"][i, j] = final, first + len(nodes)
    return r


# ---------------------------------------------------------------------------------------------- work

def work(case):
    """Each input read once, each output written once; the products' multiplications and additions."""
    b, hq, hk, d, c, t = (case[x] for x in ("batch", "heads", "kv_heads", "dim", "cache", "tokens"))
    if case["op"] == "insert":
        rows = sum(_accepted(case)) * hk
        # importance and position of every slot; the new rows in, as many rows out with their four numbers
        return {"bytes": 8 * hk * sum(_lengths(case)) + rows * (8 * d + 4 + 12), "flops": rows * d}
    keys = sum(_lengths(case))
    if case["op"] == "replay":
        counts = _accepted(case)
        pairs = sum(n * a + a * (a + 1) // 2 for n, a in zip(_lengths(case), counts))
        return {"bytes": 2 * d * (hk * keys + sum(counts) * (hq + 2 * hk)) + 4 * hq * sum(counts) + 12 * hk * keys
                + 4 * hk * sum(counts), "flops": 2 * d * hq * pairs}
    inner = int(_tree(case).sum()) if case["branch"] else t * (t + 1) // 2
    extra = 0 if case["branch"] else 12 * hk * keys + 4 * b * hk * t
    return {"bytes": 4 * d * (hk * keys + b * t * (hq + hk)) + 4 * b * hq * t + extra,
            "flops": 4 * d * hq * (t * keys + b * inner)}
