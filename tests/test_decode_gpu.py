"""Attention of new tokens over a bounded cache, replay of a path and insertion, against float64 on the CPU."""
import math

import pytest
import torch

from flash_evict import DecodeCache, decode_attention, gather_tokens, insert_tokens, prefill, replay_path, select_tokens
from oracle import decode as odec

from _decode import E24, check_attention, check_importance, make, random_tree, trail
from _helpers import seeded_randn

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _lengths(b, hk, c, seed):
    """Per-head lengths with 0, 1 and c among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(0, c + 1, (b, hk), generator=g).to(torch.int32)
    flat = x.flatten()
    for i, n in enumerate((c, 0, 1, max(c - 1, 0))):
        if i < flat.numel():
            flat[i] = n
    return x.cuda()


def _scores(b, hk, c, vc, seed):
    imp = seeded_randn((b, hk, c), torch.float32, seed).abs()
    return imp, vc.float().abs().sum(-1)


def _attend_and_check(q, k, v, kc, vc, length, **kw):
    out, lse, imp, new = decode_attention(q, k, v, kc, vc, length, **kw)
    ref_kw = {x: kw[x] for x in ("tree", "scale", "importance", "value_norm", "recency_decay") if x in kw}
    ref = odec.attend(q, k, v, kc, vc, length, **ref_kw)
    c, d = kc.shape[2:]
    check_attention(out, lse, ref, q.dtype, c, d)
    if "importance" in kw:
        finite = ref["lse"][ref["lse"] != -math.inf]
        check_importance(imp, new, ref, kw["importance"], float(finite.abs().max()) if finite.numel() else 0., float(ref["dots"].max()),
                         q.shape[1] // kc.shape[1] * q.shape[2], c, d, False)
    else:
        assert imp is None and new is None
    return out, lse, imp, new, ref


CASES = [
    # b, hq, hk, t, c, d, dtype, layout
    (1, 1, 1, 1, 1, 8, BF, "contiguous"),
    (1, 8, 2, 1, 33, 64, FP, "transposed"),
    (2, 4, 4, 1, 100, 128, BF, "transposed"),          # one query head a KV head
    (3, 14, 2, 1, 257, 128, BF, "contiguous"),         # seven
    (1, 32, 8, 1, 1024, 128, BF, "transposed"),
    (1, 64, 1, 1, 500, 128, FP, "contiguous"),         # all on one KV head
    (2, 8, 2, 2, 31, 80, FP, "padded"),
    (1, 8, 2, 4, 64, 96, BF, "transposed"),
    (1, 4, 2, 8, 65, 256, BF, "transposed"),
    (2, 4, 2, 7, 200, 192, FP, "contiguous"),
    (1, 6, 2, 33, 129, 40, BF, "contiguous"),
    (1, 28, 4, 5, 700, 128, FP, "transposed"),         # 35 rows a KV head
    (1, 4, 2, 64, 300, 64, BF, "padded"),
    (1, 2, 1, 256, 90, 128, FP, "transposed"),
    (1, 4, 4, 100, 1, 32, BF, "contiguous"),
    (2, 4, 2, 3, 70, 100, BF, "contiguous"),           # head dims that are no multiple of 8
    (1, 4, 2, 9, 40, 7, FP, "transposed"),
    (1, 2, 2, 5, 66, 250, BF, "contiguous"),
    (1, 4, 2, 6, 50, 64, BF, "strided"),
    (2, 4, 1, 3, 77, 128, FP, "odd_rows"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
def test_chunk(case):
    b, hq, hk, t, c, d, dtype, layout = case
    q, k, v, kc, vc = make(b, hq, hk, t, c, d, dtype, 11, layout)
    length = _lengths(b, hk, c, 3)
    imp, norm = _scores(b, hk, c, vc, 5)
    before = imp.clone()
    out, lse, got, new, _ = _attend_and_check(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.1)
    assert torch.equal(imp, before) and got is not imp
    for i in range(b):                                  # slots past the length
        for j in range(hk):
            assert torch.equal(got[i, j, int(length[i, j]):], before[i, j, int(length[i, j]):])
    # without weights: the same attention; unweighted and in place
    again = decode_attention(q, k, v, kc, vc, length)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse) and again[2] is None
    _, _, same, _ = decode_attention(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.1, importance_out=imp)
    assert same is imp and torch.equal(imp, got)
    _attend_and_check(q, k, v, kc, vc, length, importance=before)


@pytest.mark.parametrize("rows", [(16, 1), (17, 1), (1, 24), (4, 8)], ids=str)
@pytest.mark.parametrize("d", [64, 72, 96, 128, 192, 250, 256])
def test_rows_about_a_tile_of_queries(rows, d):
    """16, 17, 24 and 32 query rows to a KV head in every tile dim, with a length that ends inside a tile."""
    g, t = rows
    q, k, v, kc, vc = make(1, 2 * g, 2, t, 300, d, BF if d % 128 else FP, 12, "contiguous")
    length = torch.tensor([[300, 141]], dtype=torch.int32).cuda()
    imp, norm = _scores(1, 2, 300, vc, 5)
    _attend_and_check(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.05)
    _attend_and_check(q, k, v, kc, vc, length, scale=-0.3)


@pytest.mark.parametrize("b,hk,g,t,c,d", [(9, 8, 8, 5, 150, 64), (17, 8, 9, 4, 70, 64), (1, 2, 5, 120, 900, 64), (2, 1, 3, 256, 257, 192),
                                          (3, 2, 4, 33, 2500, 80)])
def test_heads_of_different_lengths_share_the_blocks(b, hk, g, t, c, d):
    """More than 32 rows a KV head: up to and over 128 heads, several row blocks, few and many tiles a head."""
    q, k, v, kc, vc = make(b, g * hk, hk, t, c, d, BF, 13)
    length = _lengths(b, hk, c, 14)
    imp, norm = _scores(b, hk, c, vc, 15)
    _attend_and_check(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.01)


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, FP), (192, BF)])
@pytest.mark.parametrize("alike", [False, True])
def test_batches_of_many_heads(d, dtype, alike):
    """Few rows of 64 and 128 heads, more tiles than blocks: steps, a chunk and a path, lengths from 0 to all or alike."""
    b, hk, c, t = 16 if d > 128 else 32, 4, 1100, 3
    q, k, v, kc, vc = make(b, 2 * hk, hk, t, c, d, dtype, 16)
    length = torch.full((b, hk), c, dtype=torch.int32).cuda() if alike else _lengths(b, hk, c, 17)
    imp, norm = _scores(b, hk, c, vc, 18)
    _attend_and_check(q[:, :, :1], k[:, :, :1], v[:, :, :1], kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.1)
    tree = torch.tensor([[1, 0, 0], [1, 1, 0], [1, 0, 1]], dtype=torch.bool).cuda()
    _, lse, _, _, _ = _attend_and_check(q, k, v, kc, vc, length, tree=tree)
    path = torch.tensor([[0, 2], [0, -1]], dtype=torch.int32).repeat(b // 2, 1).cuda()
    got, new = replay_path(q, k, v, kc, length, lse, path, imp, value_norm=norm, recency_decay=0.2)
    ref = odec.replay(q, k, v, kc, length, lse, path, imp, value_norm=norm, recency_decay=0.2)
    check_importance(got, new, ref, imp, float(lse[lse != -math.inf].abs().max()), ref["dots"], 4, c, d, True)


TREES = [(1, 8, 2, 2, 40, 64, BF), (2, 8, 2, 13, 100, 128, FP), (1, 28, 4, 64, 333, 128, BF), (2, 4, 2, 61, 64, 80, FP),
         (1, 4, 1, 128, 200, 128, BF), (1, 2, 2, 250, 31, 256, FP), (1, 4, 2, 33, 50, 100, BF)]


@pytest.mark.parametrize("case", TREES, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
@pytest.mark.parametrize("each", [False, True], ids=["shared", "each"])
def test_tree(case, each):
    b, hq, hk, t, c, d, dtype = case
    q, k, v, kc, vc = make(b, hq, hk, t, c, d, dtype, 21)
    length = _lengths(b, hk, c, 4)
    masks = [random_tree(t, 7 + i, empty=(t // 2,) if t > 2 else ()) for i in range(b)]
    tree = torch.stack([m for m, _ in masks]).cuda() if each else masks[0][0].cuda()
    out, lse, _, _, _ = _attend_and_check(q, k, v, kc, vc, length, tree=tree)
    # the accepted path: a trail of each row's tree, of its own length (one of them empty)
    parents = [masks[i if each else 0][1] for i in range(b)]
    trails = [trail(p, t - 1 - i) for i, p in enumerate(parents)]
    trails = [[x for x in tr if x != t // 2 or t <= 2] for tr in trails]
    a = max(map(len, trails))
    path = torch.full((b, a), -1, dtype=torch.int32)
    for i, tr in enumerate(trails):
        if not (i == 1 and each):
            path[i, :len(tr)] = torch.tensor(tr, dtype=torch.int32)
    imp, norm = _scores(b, hk, c, vc, 6)
    path = path.cuda()
    for w in (norm, None):
        got, new = replay_path(q, k, v, kc, length, lse, path, imp, value_norm=w, recency_decay=0.2)
        ref = odec.replay(q, k, v, kc, length, lse, path, imp, value_norm=w, recency_decay=0.2)
        finite = lse[lse != -math.inf]
        check_importance(got, new, ref, imp, float(finite.abs().max()), ref["dots"], hq // hk * a, c, d, True)
        for i in range(b):
            assert torch.equal(new[i, :, len(odec.path_nodes(path, i, t)):], torch.zeros_like(new[i, :, len(odec.path_nodes(path, i, t)):]))


def test_replay_of_the_whole_chunk_and_of_odd_paths():
    """None is every token in order; a path may end at any entry outside the tokens, and name a node again."""
    b, hq, hk, t, c, d = 2, 8, 2, 10, 90, 64
    q, k, v, kc, vc = make(b, hq, hk, t, c, d, BF, 31)
    length = _lengths(b, hk, c, 5)
    imp, norm = _scores(b, hk, c, vc, 7)
    _, lse, whole, fresh = decode_attention(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.1)
    got, new = replay_path(q, k, v, kc, length, lse, None, imp, value_norm=norm, recency_decay=0.1)
    torch.testing.assert_close(got, whole, rtol=1e-5, atol=0)
    torch.testing.assert_close(new, fresh, rtol=1e-5, atol=0)
    for path in ([[0, 3, 99, 1], [-1, 2, 3, 4]], [[4, 4, 4, 2], [9, 0, -5, 0]], [[-1], [10]]):
        path = torch.tensor(path, dtype=torch.int32).cuda()
        ref = odec.replay(q, k, v, kc, length, lse, path, imp, value_norm=norm, recency_decay=0.1)
        got, new = replay_path(q, k, v, kc, length, lse, path, imp, value_norm=norm, recency_decay=0.1)
        check_importance(got, new, ref, imp, float(lse.abs().max()), ref["dots"], hq // hk * 4, c, d, True)


@pytest.mark.parametrize("scale", [0., -0.2, 1.5])
def test_scales(scale):
    q, k, v, kc, vc = make(1, 8, 2, 5, 150, 64, BF, 41)
    length = _lengths(1, 2, 150, 6)
    imp, norm = _scores(1, 2, 150, vc, 8)
    _attend_and_check(q, k, v, kc, vc, length, scale=scale, importance=imp, value_norm=norm, recency_decay=0.05)


@pytest.mark.parametrize("d,layout", [(64, "contiguous"), (128, "transposed"), (20, "contiguous")])
def test_what_is_hidden_does_not_matter(d, layout):
    """Cache rows past the length and new tokens a query does not see may hold anything, infinities and NaN too."""
    b, hq, hk, t, c = 2, 4, 2, 40, 70
    q, k, v, kc, vc = make(b, hq, hk, t, c, d, BF, 51, layout)
    length = torch.tensor([[70, 33], [0, 31]], dtype=torch.int32).cuda()
    tree, _ = random_tree(t, 3)
    poison = [5, 17, 33]
    tree[:, poison] = False
    tree = tree.cuda()
    tree[5, 17] = True                                  # a query that does see one
    clean = decode_attention(q, k, v, kc, vc, length, tree=tree)
    kc, vc, k, v = (x.clone() for x in (kc, vc, k, v))
    for i in range(b):
        for j in range(hk):
            kc[i, j, int(length[i, j]):], vc[i, j, int(length[i, j]):] = math.nan, math.inf
    k[:, :, poison], v[:, :, poison] = math.nan, math.inf
    v[:, :, 33, 0] = -math.inf
    out, lse = decode_attention(q, k, v, kc, vc, length, tree=tree)[:2]
    rows = [i for i in range(t) if i != 5]
    assert torch.equal(out[:, :, rows], clean[0][:, :, rows]) and torch.equal(lse[:, :, rows], clean[1][:, :, rows])
    assert bool(torch.isnan(lse[:, :, 5]).all())
    # an infinite value reaches the queries that see it, as what it is
    k2, v2 = k.clone(), v.clone()
    k2[:, :, poison] = 0.
    out = decode_attention(q, k2, v2, kc, vc, length, tree=tree)[0]
    assert bool((out[:, :, 5] == math.inf).all()) and bool(torch.isfinite(out[:, :, rows]).all())


def test_empty_cache_and_rows_that_see_nothing():
    q, k, v, kc, vc = make(1, 4, 2, 3, 20, 64, FP, 61)
    length = torch.zeros((1, 2), dtype=torch.int32).cuda()
    tree = torch.zeros((3, 3), dtype=torch.bool).cuda()
    tree[2, 0] = True
    out, lse, imp, new = decode_attention(q, k, v, kc, vc, length, tree=tree, importance=torch.ones((1, 2, 20)).cuda())
    assert torch.equal(out[:, :, :2], torch.zeros_like(out[:, :, :2])) and bool((lse[:, :, :2] == -math.inf).all())
    assert torch.equal(out[0, :, 2], v[0, :, 0].repeat_interleave(2, 0))
    assert torch.equal(imp, torch.ones_like(imp))
    # replaying rows that saw nothing gives no weight
    got, fresh = replay_path(q, k, v, kc, length, lse, torch.tensor([[0, 1]], dtype=torch.int32).cuda(), imp)
    assert torch.equal(got, imp) and torch.equal(fresh, torch.zeros_like(fresh))


def test_lengths_outside_the_cache_are_clamped():
    q, k, v, kc, vc = make(1, 4, 2, 2, 40, 64, BF, 71)
    a = decode_attention(q, k, v, kc, vc, torch.tensor([[40, 0]], dtype=torch.int32).cuda())
    b = decode_attention(q, k, v, kc, vc, torch.tensor([[1 << 30, -7]], dtype=torch.int32).cuda())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("t", [1, 8])
def test_rows_past_two_to_the_31(t):
    """A head's rows more than 2^31 elements apart from each other, and from the next head's."""
    c, d, wide = 300, 128, 1 << 23
    store = torch.zeros((c - 1) * wide + 4 * d, dtype=BF, device="cuda")      # 5 GB
    cache = torch.as_strided(store, (1, 2, c, d), (0, d, wide, 1))
    src = seeded_randn((1, 2, c, d), BF, 81)
    cache.copy_(src)
    vcache = torch.as_strided(store, (1, 2, c, d), (0, d, wide, 1), 2 * d)
    vsrc = seeded_randn((1, 2, c, d), BF, 82)
    vcache.copy_(vsrc)
    q, k, v, _, _ = make(1, 8, 2, t, 1, d, BF, 83)
    length = torch.tensor([[c, c - 3]], dtype=torch.int32).cuda()
    imp = torch.ones((1, 2, c), device="cuda")
    a = decode_attention(q, k, v, cache, vcache, length, importance=imp)
    b = decode_attention(q, k, v, src, vsrc, length, importance=imp)
    for x, y in zip(a, b):
        assert torch.equal(x, y)


# ---------------------------------------------------------------------------------------------- insertion

def _state(b, hk, c, d, dtype, seed, length, layout="contiguous", ties=False):
    kc, vc = make(b, hk, hk, 1, c, d, dtype, seed, layout)[3:]
    g = torch.Generator().manual_seed(seed)
    imp = torch.randint(0, 4, (b, hk, c), generator=g).float() if ties else torch.rand((b, hk, c), generator=g)
    pos = torch.stack([torch.randperm(3 * c, generator=g)[:c] for _ in range(b * hk)]).view(b, hk, c).to(torch.int32)
    return {"k": kc.clone(memory_format=torch.preserve_format) if layout != "padded" else kc,
            "v": vc.clone(memory_format=torch.preserve_format) if layout != "padded" else vc, "importance": imp.cuda(),
            "position": pos.cuda(), "value_norm": vc.float().abs().sum(-1), "length": length.clone(),
            "seen": torch.full((b, hk), 3 * c, dtype=torch.int32).cuda()}


def _insert_and_check(s, k, v, budget, **kw):
    host = {x: None if y is None else y.detach().cpu().clone() for x, y in s.items()}
    host["value_norm"] = None if s["value_norm"] is None else host["value_norm"].double()
    ref = odec.insert(host, None if k is None else k.cpu(), None if v is None else v.cpu(), budget, kw.get("recent", 0),
                      None if kw.get("new_importance") is None else kw["new_importance"].cpu(),
                      None if kw.get("path") is None else kw["path"].cpu())
    insert_tokens(k, v, s["k"], s["v"], s["importance"], s["position"], s["length"], s["seen"], budget,
                  value_norm=s["value_norm"], **kw)
    for x in ("length", "seen", "position"):
        assert torch.equal(s[x].cpu(), ref[x]), x
    for x in ("k", "v", "importance"):
        assert torch.equal(torch.nan_to_num(s[x].cpu(), nan=77.), torch.nan_to_num(ref[x], nan=77.)), x
    if s["value_norm"] is not None:
        d = s["v"].shape[3]
        err = (s["value_norm"].cpu().double() - ref["value_norm"]).abs()
        assert bool((err <= d * E24 * ref["value_norm"]).all())


INSERTS = [
    # b, hk, c, d, t, budget, recent, dtype, layout
    (1, 1, 1, 8, 1, 1, 0, BF, "contiguous"),
    (1, 8, 128, 128, 1, 128, 16, BF, "transposed"),
    (2, 2, 100, 64, 1, 90, 10, FP, "contiguous"),
    (2, 3, 257, 80, 7, 200, 20, BF, "padded"),
    (1, 2, 1024, 128, 64, 1000, 64, BF, "transposed"),
    (1, 2, 50, 256, 49, 50, 50, FP, "contiguous"),
    (2, 2, 40, 64, 100, 40, 8, BF, "contiguous"),       # more new rows than the cache holds
    (1, 2, 64, 100, 5, 60, 3, BF, "contiguous"),        # element copies
    (1, 2, 30, 64, 5, 30, 3, FP, "strided"),
    (1, 1, 5000, 32, 300, 4000, 128, BF, "contiguous"),
    (1, 2, 2500, 16, 1200, 2500, 0, FP, "contiguous"),
]


@pytest.mark.parametrize("case", INSERTS, ids=lambda c: "-".join(map(str, c)).replace("torch.", ""))
@pytest.mark.parametrize("ties", [False, True], ids=["", "ties"])
def test_insert(case, ties):
    b, hk, c, d, t, budget, recent, dtype, layout = case
    length = _lengths(b, hk, c, 9)
    s = _state(b, hk, c, d, dtype, 91, length, layout, ties)
    for step in range(3):
        k = seeded_randn((b, t, hk, d), dtype, 92 + step).transpose(1, 2)
        v = seeded_randn((b, t, hk, d), dtype, 95 + step).transpose(1, 2)
        g = torch.Generator().manual_seed(step)
        new = torch.randint(0, 4, (b, hk, t), generator=g).float() if ties else torch.rand((b, hk, t), generator=g)
        _insert_and_check(s, k, v, budget, recent=recent, new_importance=new.cuda() if step else None)


@pytest.mark.parametrize("t", [9, 31, 32, 33, 47])
@pytest.mark.parametrize("room", [0, 3])
def test_insert_as_many_as_are_drawn_one_by_one(t, room):
    """Up to 32 evictions, and more; from a full cache and from one with room for some of the rows; ties."""
    s = _state(2, 2, 1500, 48, BF, 99, torch.tensor([[1500 - room, 1500], [1490, 700]], dtype=torch.int32).cuda(), ties=True)
    for step in range(2):
        k, v = seeded_randn((2, 2, t, 48), BF, 92 + step), seeded_randn((2, 2, t, 48), BF, 95 + step)
        new = torch.randint(0, 4, (2, 2, t), generator=torch.Generator().manual_seed(step)).float()
        _insert_and_check(s, k, v, 1500, recent=5, new_importance=new.cuda())


@pytest.mark.parametrize("ties", [False, True], ids=["", "ties"])
def test_insert_a_path(ties):
    b, hk, c, d, t = 3, 2, 200, 64, 30
    s = _state(b, hk, c, d, BF, 101, torch.tensor([[200, 199], [150, 0], [200, 200]], dtype=torch.int32).cuda(), ties=ties)
    for path in ([[0, 3, 29, 4], [1, -1, 5, 6], [-1, 0, 0, 0]], [[7, 7, 7, 7], [30, 0, 0, 0], [29, 28, 27, 26]]):
        k, v = seeded_randn((b, hk, t, d), BF, 102), seeded_randn((b, hk, t, d), BF, 103)
        new = torch.randint(0, 4, (b, hk, 4), generator=torch.Generator().manual_seed(1)).float().cuda()
        _insert_and_check(s, k, v, c, recent=2, new_importance=new, path=torch.tensor(path, dtype=torch.int32).cuda())


@pytest.mark.parametrize("c,budget,recent", [(300, 100, 10), (5000, 1, 0), (5000, 4999, 64), (70000, 7000, 64), (200, 200, 0)])
def test_evict(c, budget, recent):
    length = torch.tensor([[c, c - 1, min(budget, c)], [c // 2, 0, 1]], dtype=torch.int32).cuda()
    s = _state(2, 3, c, 32, BF, 111, length, ties=c == 5000)
    s["importance"][0, 0, ::7] = math.nan
    s["importance"][0, 1, ::5] = -0.
    s["importance"][1, 0, ::3] = math.inf
    _insert_and_check(s, None, None, budget, recent=recent)


def test_insert_without_norms_and_with_many_protected_rows():
    """Rows that claim newer positions than `recent` allows: ties among the protected ones keep the lower slot."""
    s = _state(1, 2, 60, 64, BF, 121, torch.full((1, 2), 60, dtype=torch.int32).cuda())
    s["position"][:, 0] += 1000
    s["value_norm"] = None
    k = seeded_randn((1, 2, 9, 64), BF, 122)
    _insert_and_check(s, k, k.clone(), 50, recent=5)


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("decay,weighted", [(0., True), (0.1, False), (0.02, True)])
def test_decoding_continues_prefill(decay, weighted):
    """With room for everything: prefill of 200 tokens, then chunks, one by one and a drafted path, give the output
    and importance of a prefill of all of them. Tolerances: both sides round P and the output (2 + 2 + 2 half steps
    of values of order 1), and importance sums of FP32 probabilities, 1e-4 relative as in the prefill tests."""
    b, hq, hk, n, d = 1, 8, 2, 263, 64
    q, k, v = (seeded_randn((b, n, h, d), BF, 131 + i).transpose(1, 2) for i, h in enumerate((hq, hk, hk)))
    ref_out, ref_imp = prefill(q, k, v, recency_decay=decay, value_weighted=weighted)
    cut = 200
    out, imp = prefill(q[:, :, :cut], k[:, :, :cut], v[:, :, :cut], recency_decay=decay, value_weighted=weighted)
    cache = DecodeCache(b, hk, d, 300, dtype=BF, device="cuda", recency_decay=decay, value_weighted=weighted)
    cache.load(k[:, :, :cut], v[:, :, :cut], imp)
    outs = [out]
    for t in (1, 1, 33, 20):
        end = cut + t
        outs.append(cache.decode(q[:, :, cut:end], k[:, :, cut:end], v[:, :, cut:end]))
        cut = end
    # the last 8 as the even nodes of a drafted chain whose odd nodes are rejected
    t = n - cut
    take = torch.arange(0, 2 * t, 2)
    dq, dk, dv = (seeded_randn((b, x.shape[1], 2 * t, d), BF, 141) for x in (q, k, v))
    for x, y in ((dq, q), (dk, k), (dv, v)):
        x[:, :, take.cuda()] = y[:, :, cut:]
    tree = torch.eye(2 * t, dtype=torch.bool)
    for i in range(0, 2 * t, 2):
        tree[i, :i + 1:2] = True
    o, lse = cache.draft(dq, dk, dv, tree.cuda())
    outs.append(o[:, :, ::2])
    cache.accept(dq, dk, dv, lse, take.to(torch.int32).view(1, -1).cuda())
    got = torch.cat(outs, 2).float()
    torch.testing.assert_close(got, ref_out.float(), atol=6 * 2. ** -9, rtol=6 * 2. ** -9)
    assert cache.length.tolist() == [[n] * hk] and cache.seen.tolist() == [[n] * hk]
    assert torch.equal(cache.position[0, 0, :n].cpu(), torch.arange(n, dtype=torch.int32))
    assert torch.equal(cache.k[:, :, :n], k) and torch.equal(cache.v[:, :, :n], v)
    torch.testing.assert_close(cache.importance[:, :, :n], ref_imp, rtol=1e-4, atol=1e-6)


def test_a_bounded_loop_follows_the_oracle():
    """Prefill, eviction to a budget, steps and drafts, each step's result fed on: attention against float64 over the
    cache's own rows, the moves against the rule on the kernel's own importance."""
    b, hq, hk, n, d, budget = 1, 8, 2, 150, 64, 60
    q, k, v = (seeded_randn((b, h, n, d), BF, 151 + i) for i, h in enumerate((hq, hk, hk)))
    out, imp = prefill(q, k, v, recency_decay=0.1)
    cache = DecodeCache(b, hk, d, budget, dtype=BF, device="cuda", recent=8, recency_decay=0.1)
    cache.load(k, v, imp)
    kept, _ = select_tokens(imp, budget, recent=8)
    assert torch.equal(cache.position.sort(-1).values.long(), kept)
    order = cache.position.sort(-1).indices
    assert torch.equal(cache.k.gather(2, order[..., None].expand(b, hk, budget, d)), gather_tokens(k, kept))
    for step in range(12):
        t = (1, 1, 6)[step % 3]
        q, k, v = (seeded_randn((b, h, t, d), BF, 161 + 3 * step + i) for i, h in enumerate((hq, hk, hk)))
        s = {x: getattr(cache, x).cpu().clone() for x in ("k", "v", "importance", "position", "value_norm", "length", "seen")}
        if t == 1:
            path = None
            ref = odec.attend(q, k, v, s["k"], s["v"], s["length"])
            out = cache.decode(q, k, v)
            lse = None
        else:
            tree, parent = random_tree(t, step)
            ref = odec.attend(q, k, v, s["k"], s["v"], s["length"], tree=tree)
            out, lse = cache.draft(q, k, v, tree.cuda())
            path = torch.tensor([trail(parent, t - 1)], dtype=torch.int32).cuda()
            cache.accept(q, k, v, lse, path)
        err = (out.cpu().double() - ref["out"]).abs()
        assert bool((err <= 4 * 2. ** -8 * ref["mass_v"] + 1e-5).all())
        # what stayed is what the importance before the moves ranks highest: redo the step's weights from the kernel
        s2 = {x: y.cuda() for x, y in s.items()}
        if path is None:
            _, _, _, new = decode_attention(q, k, v, s2["k"], s2["v"], s2["length"], importance=s2["importance"],
                                            value_norm=s2["value_norm"], recency_decay=0.1, importance_out=s2["importance"])
        else:
            _, new = replay_path(q, k, v, s2["k"], s2["length"], lse, path, s2["importance"], value_norm=s2["value_norm"],
                                 recency_decay=0.1, importance_out=s2["importance"])
        host = {x: y.cpu() for x, y in s2.items()}
        odec.insert(host, k.cpu(), v.cpu(), budget, 8, new.cpu(), None if path is None else path.cpu())
        for x in ("k", "v", "importance", "position", "length", "seen"):
            assert torch.equal(getattr(cache, x).cpu(), host[x]), (step, x)
    cache.evict(20)
    assert cache.length.tolist() == [[20, 20]]
    assert bool((cache.position[:, :, :20] >= cache.seen[..., None] - 8).sum(-1).eq(8).all())


# ---------------------------------------------------------------------------------------------- calls

def test_calls_are_repeatable_and_independent_of_the_stream():
    q, k, v, kc, vc = make(2, 8, 2, 3, 500, 128, BF, 171)
    length = _lengths(2, 2, 500, 10)
    imp, norm = _scores(2, 2, 500, vc, 11)
    kw = dict(importance=imp, value_norm=norm, recency_decay=0.1)
    first = decode_attention(q, k, v, kc, vc, length, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = decode_attention(q, k, v, kc, vc, length, **kw)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(first, other):
        assert torch.equal(x, y)


def test_a_captured_step_replays_as_eager():
    """A decode step in a graph, replayed with eager work between: lengths, moves and importance go on as eagerly."""
    b, hq, hk, d, budget = 2, 8, 2, 64, 48

    def tokens(i):
        return (seeded_randn((b, h, 1, d), BF, 181 + 3 * i + j) for j, h in enumerate((hq, hk, hk)))

    def cache():
        c = DecodeCache(b, hk, d, budget, dtype=BF, device="cuda", recent=4, recency_decay=0.1)
        c.load(seeded_randn((b, hk, 45, d), BF, 1), seeded_randn((b, hk, 45, d), BF, 2), seeded_randn((b, hk, 45), torch.float32, 3).abs())
        return c

    eager, graphed = cache(), cache()
    held = [x.clone() for x in tokens(0)]
    warm = cache()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm.decode(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.decode(*held)
    for i in range(8):
        for x, y in zip(held, tokens(i)):
            x.copy_(y)
        graph.replay()
        want = eager.decode(*tokens(i))
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("k", "v", "importance", "position", "value_norm", "length", "seen"):
            assert torch.equal(getattr(eager, name), getattr(graphed, name)), (i, name)


def test_refusals_on_the_gpu():
    q, k, v, kc, vc = make(2, 4, 2, 3, 20, 64, BF, 191)
    length = torch.full((2, 2), 20, dtype=torch.int32, device="cuda")
    imp = torch.ones((2, 2, 20), device="cuda")
    eye = torch.eye(3, dtype=torch.bool, device="cuda")
    path = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    lse = torch.zeros((2, 4, 3), device="cuda")
    for bad in (length.long(), length[:1], length.cpu(), length.t()[:, :].t().expand(2, 2).t()[:, :1]):
        with pytest.raises(ValueError, match="length"):
            decode_attention(q, k, v, kc, vc, bad)
    for bad in (eye.int(), eye[:2], eye.cpu(), eye.expand(3, 3, 3)):
        with pytest.raises(ValueError, match="tree"):
            decode_attention(q, k, v, kc, vc, length, tree=bad)
    with pytest.raises(ValueError, match="k_cache and v_cache"):
        decode_attention(q, k, v, kc, vc[:, :, :10], length)
    with pytest.raises(ValueError, match="same device and dtype"):
        decode_attention(q, k.half(), v, kc, vc, length)
    with pytest.raises(ValueError, match="scale"):
        decode_attention(q, k, v, kc, vc, length, scale=math.nan)
    with pytest.raises(ValueError, match="recency_decay"):
        decode_attention(q, k, v, kc, vc, length, recency_decay=-0.1)
    with pytest.raises(ValueError, match="go with importance"):
        decode_attention(q, k, v, kc, vc, length, value_norm=imp)
    with pytest.raises(ValueError, match="importance must be"):
        decode_attention(q, k, v, kc, vc, length, importance=imp.double())
    with pytest.raises(ValueError, match="importance_out is written"):
        decode_attention(q, k, v, kc, vc, length, importance=imp, importance_out=imp[:, :, :1].expand(2, 2, 20))
    with pytest.raises(ValueError, match="Inference only"):
        decode_attention(q.clone().requires_grad_(), k, v, kc, vc, length)
    for bad in (path.long(), path[:1], path.cpu(), torch.zeros((2, 4), dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError, match="path"):
            replay_path(q, k, v, kc, length, lse, bad, imp)
    with pytest.raises(ValueError, match="lse"):
        replay_path(q, k, v, kc, length, lse[:, :2], path, imp)
    pos, seen = torch.zeros((2, 2, 20), dtype=torch.int32, device="cuda"), length.clone()
    kc, vc = kc.contiguous(), vc.contiguous()
    for kw, match in ((dict(budget=0), "budget"), (dict(budget=21), "budget"), (dict(recent=21), "recent"),
                      (dict(new_importance=imp), "new_importance"), (dict(path=path.long()), "path")):
        kw = dict(dict(budget=20), **kw)
        with pytest.raises(ValueError, match=match):
            insert_tokens(k, v, kc, vc, imp, pos, length, seen, kw.pop("budget"), **kw)
    with pytest.raises(ValueError, match="come together"):
        insert_tokens(k, None, kc, vc, imp, pos, length, seen, 20)
    with pytest.raises(ValueError, match="share the cache's memory"):
        insert_tokens(kc[:, :, :3], v, kc, vc, imp, pos, length, seen, 20)
    with pytest.raises(ValueError, match="expanded"):
        insert_tokens(k, v, kc[:, :, :1].expand(2, 2, 20, 64), vc, imp, pos, length, seen, 20)
    with pytest.raises(ValueError, match="importance is written"):
        insert_tokens(k, v, kc, vc, imp[:, :, ::2].repeat(1, 1, 2)[:, :, :20].transpose(0, 1), pos, length, seen, 20)
    with pytest.raises(ValueError, match="seen"):
        insert_tokens(k, v, kc, vc, imp, pos, length, seen.cpu(), 20)
