"""Inputs and tolerances of the decoding tests.

Tolerances. u is half a step of the input type, e = 2^-24. The kernels multiply the exact products of the inputs,
accumulated in FP32, by scale * log2 e, so a logit is off by at most (D + 4) e times dots, the largest sum of
absolute products of its row (scaled); exp2's argument (a difference of two values of at most that size) and exp2
itself add 4 e (dots + 1) log2 e and 2 e. Call the sum EL. A probability is off by EL relative, its sum by EL and by
the additions: a lane adds 16 values for each of its tiles, the tiles' sums go through at most C / 32 steps and 512
splits, each with a rescale: 3 e (C / 32 + 528).

  out         P is rounded to the input type (u relative; in fp16 half a subnormal step, 2^-25, absolute, where the
              sum of the rounded P is at least 1/2) and normalised by the sum of the rounded values: 2 u of mass_v,
              2^-24 of sum_v in fp16; FP32 effects twice EL and the additions' bound of mass_v; the result's own
              rounding u |out|, and in fp16 half a subnormal step.
  lse         EL, the additions, and rounding: 4 e (|lse| + 1)
  importance  EL and the rounding of lse in the bias, 4 e (|lse| + dots + 1) log2 e, and the additions over rows
              and of a norm, e (G T + D + 8), of the added part; 4 e of the result and 8 e of what decays.
"""
import math

import torch

from _helpers import seeded_randn

E24 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def logit_error(dots, d):
    return (d + 4) * E24 * dots + 4 * E24 * (dots + 1) * 1.5 + 2 * E24


def sum_error(c):
    return 3 * E24 * (c / 32 + 528)


def make(b, hq, hk, t, c, d, dtype, seed, layout="transposed", device="cuda", std=1.0):
    """q, k, v, k_cache, v_cache in a layout; lengths and scores come from the test."""
    if layout == "transposed":      # projections' [B, T, H, D], cache [B, C, Hkv, D]
        q, k, v = (seeded_randn((b, t, h, d), dtype, seed + i, std if i == 0 else 1., device).transpose(1, 2) for i, h in enumerate((hq, hk, hk)))
        kc, vc = (seeded_randn((b, c, hk, d), dtype, seed + 3 + i, 1., device).transpose(1, 2) for i in range(2))
    elif layout == "contiguous":
        q, k, v = (seeded_randn((b, h, t, d), dtype, seed + i, std if i == 0 else 1., device) for i, h in enumerate((hq, hk, hk)))
        kc, vc = (seeded_randn((b, hk, c, d), dtype, seed + 3 + i, 1., device) for i in range(2))
    elif layout == "strided":       # every other channel
        q, k, v = (seeded_randn((b, h, t, 2 * d), dtype, seed + i, 1., device)[..., ::2] for i, h in enumerate((hq, hk, hk)))
        kc, vc = (seeded_randn((b, hk, c, 2 * d), dtype, seed + 3 + i, 1., device)[..., ::2] for i in range(2))
    elif layout == "odd_rows":      # rows two bytes off a 16-byte boundary
        q, k, v = (seeded_randn((b, h, t, d + 1), dtype, seed + i, 1., device)[..., 1:] for i, h in enumerate((hq, hk, hk)))
        kc, vc = (seeded_randn((b, hk, c, d + 1), dtype, seed + 3 + i, 1., device)[..., 1:] for i in range(2))
    else:                           # "padded": rows and heads apart, a slice of a larger cache
        q, k, v = (seeded_randn((b, h, t, d), dtype, seed + i, 1., device) for i, h in enumerate((hq, hk, hk)))
        kc, vc = (seeded_randn((b, hk, c + 5, d + 8), dtype, seed + 3 + i, 1., device)[:, :, 2:c + 2, :d] for i in range(2))
    return q, k, v, kc, vc


def random_tree(t, seed, empty=()):
    """Ancestor mask of a random tree, itself included; rows in `empty` see nothing."""
    g = torch.Generator().manual_seed(seed)
    mask = torch.zeros((t, t), dtype=torch.bool)
    parent = [-1] + [int(torch.randint(0, i, (1,), generator=g)) for i in range(1, t)]
    for i in range(t):
        if parent[i] >= 0:
            mask[i] = mask[parent[i]]
        mask[i, i] = True
    for i in empty:
        mask[i] = False
    return mask, parent


def trail(parent, node):
    nodes = [node]
    while parent[nodes[-1]] >= 0:
        nodes.append(parent[nodes[-1]])
    return nodes[::-1]


def check_attention(out, lse, ref, dtype, c, d):
    out, lse = out.detach().cpu().double(), lse.detach().cpu().double()
    u = half_step(dtype)
    nothing = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, nothing) and torch.equal(out[nothing], torch.zeros_like(out[nothing]))
    el = logit_error(ref["dots"], d)
    tiny = 2. ** -25 if dtype == torch.float16 else 0.
    bound = ((2 * u + 2 * (el + sum_error(c)))[..., None] * ref["mass_v"] + 2 * tiny * ref["sum_v"] + u * ref["out"].abs() + tiny)
    err = (out - ref["out"]).abs()
    assert bool((err <= bound).all()), ("out", float((err / bound.clamp(min=1e-30)).max()))
    some = ~nothing
    err, bound = (lse - ref["lse"]).abs()[some], (el + sum_error(c) + 4 * E24 * (ref["lse"].abs() + 1))[some]
    assert bool((err <= bound).all()), ("lse", float((err / bound).max()))


def check_importance(got, new, ref, before, lse_size, dots, rows, c, d, exact_lse):
    """`exact_lse`: the call was given its lse (a replay); otherwise lse has its own error."""
    rel = logit_error(dots, d) + 4 * E24 * (lse_size + dots + 1) * 1.5 + E24 * (rows + d + 8)
    if not exact_lse:
        rel += logit_error(dots, d) + sum_error(c)
    got, new = got.detach().cpu().double(), new.detach().cpu().double()
    bound = rel * ref["added"] + 4 * E24 * ref["importance"].abs() + 8 * E24 * before.detach().cpu().double().abs() + 1e-37
    err = (got - ref["importance"]).abs()
    assert bool((err <= bound).all()), ("importance", float((err / bound).max()))
    err, bound = (new - ref["new_importance"]).abs(), (rel + 4 * E24) * ref["new_importance"] + 1e-37
    assert bool((err <= bound).all()), ("new_importance", float((err / bound).max()))
