"""The controllers' bounded decoding (`decode_budget`) on a tiny random-init Qwen2 (bf16): the prompt's kept tokens and
importance go on as a DecodeCache in every layer."""
import pytest
import torch

from _decode import check_attention
from flash_evict.decode import DecodeCache
from flash_evict.kv_distill_adapter import FusedController
from flash_evict.prefill import select_tokens
from flash_evict.streaming_adapter import StreamingController
from oracle import decode as odec
from test_adapters_gpu import tiny_model

pytestmark = pytest.mark.gpu
PROMPT, KEPT, LAYERS = 137, 24, 2
SCORING = {"recency_decay": .1, "value_weighted": True}


def record(ctl):
    """Every decoding call's (layer, q, k, v, scaling, output [B, Hq, T, D])."""
    calls, inner = [], ctl._decode_layer

    def layer(index, q, k, v, scaling):
        out = inner(index, q, k, v, scaling)
        calls.append((index, q, k, v, scaling, out.transpose(1, 2)))
        return out
    ctl._decode_layer = layer
    return calls


def prompt(ctl, ids):
    """The prompt forward; each layer's K, V and importance."""
    ctl.reset()
    ctl.model.model(ids[:, :PROMPT], position_ids=torch.arange(PROMPT, device="cuda")[None], use_cache=False)
    return {i: {x: s[x].clone() for x in ("k", "v", "importance") if x in s} for i, s in ctl.states.items()}


def forward(ctl, ids, start, t):
    pos = torch.arange(start, start + t, device="cuda")[None]
    return ctl.model.model(ids[:, start:start + t], position_ids=pos, use_cache=False).last_hidden_state


@torch.inference_mode()
def test_with_room_for_all_it_is_attention_over_the_kept_and_the_new_tokens():
    torch.manual_seed(301)
    model = tiny_model(LAYERS)
    ids = torch.randint(0, 257, (1, 500), device="cuda")
    ctl = FusedController(model)
    ctl.prefill_backend, ctl.scoring, ctl.decode_budget = "fused", SCORING, 400
    prompt(ctl, ids)
    ctl.compress("fused_%d" % KEPT, PROMPT)
    rows = {i: (s["k"].clone(), s["v"].clone()) for i, s in ctl.states.items()}
    calls = record(ctl)
    at = PROMPT
    for t in (5, 1, 1, 300):                # the last one is more than a call's tokens
        forward(ctl, ids, at, t)
        at += t
    for layer, q, k, v, scaling, out in calls:
        kc, vc = rows[layer]
        ref = odec.attend(q, k, v, kc, vc, torch.full((1, 2), kc.shape[2], dtype=torch.int32), scale=scaling)
        check_attention(out, ref["lse"], ref, q.dtype, 400, q.shape[3])
        rows[layer] = torch.cat((kc, k), 2), torch.cat((vc, v), 2)
    for i, s in ctl.states.items():
        assert torch.equal(s["k"], rows[i][0]) and torch.equal(s["v"], rows[i][1])
    ctl.close()


@torch.inference_mode()
@pytest.mark.parametrize("streaming", [False, True])
def test_layers_follow_a_cache_of_their_own(streaming):
    """Every layer's outputs and rows are those of a DecodeCache that starts from the prompt's kept tokens, their
    importance and positions, and is fed the layer's q, k, v."""
    torch.manual_seed(302)
    model = tiny_model(LAYERS)
    ids = torch.randint(0, 257, (1, 200), device="cuda")
    plain = FusedController(model)
    plain.prefill_backend, plain.scoring = "fused", SCORING
    whole = prompt(plain, ids)
    plain.close()
    if streaming:
        ctl = StreamingController(model, budget=KEPT, scoring=SCORING, reserved_recent=4)
    else:
        ctl = FusedController(model)
        ctl.prefill_backend, ctl.scoring, ctl.reserved_recent = "fused", SCORING, 4
    ctl.decode_budget, ctl.decode_recent = 30, 4
    whole_again = prompt(ctl, ids)
    if streaming:
        ctl.finish_prefill()
    else:
        whole = whole_again                 # the very importance, whose sums' order may differ between runs
        ctl.compress("fused_%d" % KEPT, PROMPT)
    caches = {}
    for i, s in ctl.states.items():
        keep = s["position"].long()
        if not streaming:
            assert torch.equal(keep, select_tokens(whole[i]["importance"], KEPT, recent=4)[0])
        index = keep[..., None].expand(-1, -1, -1, s["k"].shape[3])
        assert torch.equal(s["k"], whole[i]["k"].gather(2, index)) and torch.equal(s["v"], whole[i]["v"].gather(2, index))
        torch.testing.assert_close(s["importance"], whole[i]["importance"].gather(2, keep), rtol=1e-4, atol=1e-6)
        caches[i] = DecodeCache(1, 2, s["k"].shape[3], 30, dtype=torch.bfloat16, device="cuda", recent=4, recency_decay=.1)
        caches[i].load(s["k"], s["v"], s["importance"], position=s["position"], seen=PROMPT)
    calls = record(ctl)
    at = PROMPT
    for t in (1, 7, 1, 1, 20):
        forward(ctl, ids, at, t)
        at += t
    for layer, q, k, v, scaling, out in calls:
        assert torch.equal(caches[layer].decode(q, k, v, scale=scaling), out)
    for i, s in ctl.states.items():
        assert s["k"].shape[2] == 30 and caches[i].length.tolist() == [[30, 30]]
        assert torch.equal(s["k"], caches[i].k) and torch.equal(s["v"], caches[i].v)
        newest = caches[i].position >= at - 4
        assert caches[i].seen.tolist() == [[at, at]] and bool((newest.sum(-1) == 4).all())
    handed = ctl.dynamic_cache()
    assert handed.get_seq_length() == 30
    ctl.close()


@torch.inference_mode()
def test_refusals():
    torch.manual_seed(303)
    model = tiny_model(1)
    ids = torch.randint(0, 257, (1, 140), device="cuda")
    ctl = FusedController(model)
    ctl.prefill_backend, ctl.decode_budget = "fused", 16
    prompt(ctl, ids)
    ctl.compress("fused_24", PROMPT)
    with pytest.raises(ValueError, match="less than the compressed"):
        forward(ctl, ids, PROMPT, 1)
    ctl.decode_budget = 64
    forward(ctl, ids, PROMPT, 1)
    ctl.prefill_backend = "baseline"
    prompt(ctl, ids)
    ctl.compress("snap_40", PROMPT)
    with pytest.raises(ValueError, match="fused"):
        forward(ctl, ids, PROMPT, 1)
    ctl.decode_budget = None
    assert bool(torch.isfinite(forward(ctl, ids, PROMPT, 1)).all())
    ctl.close()
