"""Decoding over a bounded cache, what needs no GPU: the oracle against loops and against the prefill oracle, and
the refusals of the Python and C entry points (all before anything is launched)."""
import ctypes
import math

import pytest
import torch

import flash_evict
from flash_evict import DecodeCache, _lib, decode_attention, insert_tokens, replay_path
from oracle import decode as odec
from oracle.attention import materialized

INVALID, WORKSPACE, UNSUPPORTED = -1, -3, -4


def _rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


@pytest.mark.parametrize("decay,weighted", [(0., True), (0.1, True), (0.3, False)])
def test_chunks_continue_the_prefill_oracle(decay, weighted):
    """A prompt of 12 continued by chunks of 1, 5 and 3 has the output and importance of a prompt of 21."""
    n, d, hq, hk = 21, 16, 4, 2
    q, k, v = (_rand(1, h, n, d, seed=s).float() for s, h in enumerate((hq, hk, hk)))
    ref_out, ref_imp = materialized(q, k, v, recency_decay=decay, value_weighted=weighted)
    cut = 12
    out, imp = materialized(q[:, :, :cut], k[:, :, :cut], v[:, :, :cut], recency_decay=decay, value_weighted=weighted)
    outs, imp = [out.double()], imp.double()
    for t in (1, 5, 3):
        end = cut + t
        norm = v[:, :, :cut].double().abs().sum(-1) if weighted else None
        r = odec.attend(q[:, :, cut:end], k[:, :, cut:end], v[:, :, cut:end], k[:, :, :cut], v[:, :, :cut],
                        torch.full((1, hk), cut), importance=imp, value_norm=norm, recency_decay=decay)
        outs.append(r["out"])
        imp = torch.cat((r["importance"], r["new_importance"]), 2)
        cut = end
    # FP32 oracle: 21 terms of order 1
    torch.testing.assert_close(torch.cat(outs, 2), ref_out.double(), atol=1e-5, rtol=1e-5)
    torch.testing.assert_close(imp, ref_imp.double(), atol=1e-5, rtol=1e-5)


def test_replay_of_a_whole_chunk_is_the_chunks_importance():
    q, k, v, kc, vc = _rand(2, 4, 5, 8, seed=1), _rand(2, 2, 5, 8, seed=2), _rand(2, 2, 5, 8, seed=3), _rand(2, 2, 9, 8, seed=4), _rand(2, 2, 9, 8, seed=5)
    length = torch.tensor([[9, 4], [0, 1]])
    imp = _rand(2, 2, 9, seed=6).abs()
    norm = vc.abs().sum(-1)
    a = odec.attend(q, k, v, kc, vc, length, importance=imp, value_norm=norm, recency_decay=0.2)
    for path in (None, torch.arange(5).expand(2, 5)):
        r = odec.replay(q, k, v, kc, length, a["lse"], path, imp, value_norm=norm, recency_decay=0.2)
        torch.testing.assert_close(r["importance"], a["importance"])
        torch.testing.assert_close(r["new_importance"], a["new_importance"])
    # weights of a query sum to 1 over what it sees
    s = odec.attend(q, k, v, kc, vc, length, importance=torch.zeros_like(imp))
    torch.testing.assert_close(s["importance"].sum(-1) + s["new_importance"].sum(-1), torch.full((2, 2), 10., dtype=torch.float64))


def test_insert_oracle_on_known_answers():
    def cache(importance, position, length, seen):
        n = len(importance)
        k = torch.arange(n, dtype=torch.float64).view(1, 1, n, 1)
        return {"k": k.clone(), "v": -k, "importance": torch.tensor([[importance]], dtype=torch.float64),
                "position": torch.tensor([[position]]), "value_norm": k[..., 0].clone(), "length": torch.tensor([[length]]),
                "seen": torch.tensor([[seen]])}

    new = torch.tensor([100., 101.], dtype=torch.float64).view(1, 1, 2, 1)
    # full cache of 4: slots 1 and 3 hold the least, the new rows take them in order
    c = odec.insert(cache([5., 1., 4., 2.], [0, 1, 2, 3], 4, 4), new, -new, 4, recent=2)
    assert c["k"].flatten().tolist() == [0., 100., 2., 101.] and c["position"].flatten().tolist() == [0, 4, 2, 5]
    assert c["importance"].flatten().tolist() == [5., 0., 4., 0.] and c["length"].item() == 4 and c["seen"].item() == 6
    assert c["value_norm"].flatten().tolist() == [0., 100., 2., 101.]
    # unprotected new rows of importance 0 leave at once; equal ones keep the lower slot
    c = odec.insert(cache([0., 1., 4., 0.], [0, 1, 2, 3], 4, 4), new, -new, 4)
    assert c["k"].flatten().tolist() == [0., 1., 2., 3.] and c["seen"].item() == 6
    # room for one: the first new row is appended, the second finds everything above it
    c = odec.insert(cache([3., 1., 4., 7.], [0, 1, 2, 9], 3, 3), new, -new, 4)
    assert c["k"].flatten().tolist() == [0., 1., 2., 100.] and c["length"].item() == 4
    # eviction alone: NaN above everything, then 4; both move, and slots from the new length on stay as they were
    c = odec.insert(cache([3., 1., 4., math.nan], [0, 1, 2, 3], 4, 4), None, None, 2)
    assert c["k"].flatten().tolist() == [2., 3., 2., 3.] and c["position"].flatten().tolist() == [2, 3, 2, 3]
    assert c["length"].item() == 2 and c["seen"].item() == 4


# ------------------------------------------------------------------------------------------ refusals

def _args(**change):
    a = dict(q=torch.zeros(1, 4, 3, 16, dtype=torch.float16), k=torch.zeros(1, 2, 3, 16, dtype=torch.float16),
             v=torch.zeros(1, 2, 3, 16, dtype=torch.float16), kc=torch.zeros(1, 2, 8, 16, dtype=torch.float16),
             vc=torch.zeros(1, 2, 8, 16, dtype=torch.float16), length=torch.zeros(1, 2, dtype=torch.int32))
    a.update(change)
    return a


@pytest.mark.parametrize("change,match", [
    (dict(q=torch.zeros(4, 3, 16)), "shape"),
    (dict(k=torch.zeros(1, 2, 4, 16)), "equal batch, tokens"),
    (dict(kc=torch.zeros(1, 2, 8, 24)), "cache of their batch"),
    (dict(kc=torch.zeros(1, 2, 0, 16)), "nonempty"),
    (dict(q=torch.zeros(1, 3, 3, 16)), "divisible"),
    (dict(), "CUDA fp16 or bf16"),
])
def test_new_tokens_are_checked(change, match):
    a = _args(**change)
    with pytest.raises(ValueError, match=match):
        decode_attention(a["q"], a["k"], a["v"], a["kc"], a["vc"], a["length"])
    with pytest.raises(ValueError, match=match):
        replay_path(a["q"], a["k"], a["v"], a["kc"], a["length"], torch.zeros(1, 4, 3), None, torch.zeros(1, 2, 8))


def test_too_many_tokens_and_wide_heads_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="256 new tokens"):
        decode_attention(z(1, 1, 257, 8), z(1, 1, 257, 8), z(1, 1, 257, 8), z(1, 1, 4, 8), z(1, 1, 4, 8), None)
    with pytest.raises(ValueError, match="<= 256"):
        decode_attention(z(1, 1, 1, 264), z(1, 1, 1, 264), z(1, 1, 1, 264), z(1, 1, 4, 264), z(1, 1, 4, 264), None)


def test_insert_needs_a_gpu_cache_and_whole_arguments():
    z = torch.zeros(1, 1, 4, 8, dtype=torch.float16)
    i = torch.zeros(1, 1, 4)
    with pytest.raises(ValueError, match="CUDA"):
        insert_tokens(z, z, z, z, i, i.int(), i[..., 0].int(), i[..., 0].int(), 4)
    with pytest.raises(ValueError, match="nonempty"):
        insert_tokens(z, z, z[..., :0], z[..., :0], i, i.int(), i[..., 0].int(), i[..., 0].int(), 4)


@pytest.mark.parametrize("change,match", [
    (dict(batch=0), "batch"), (dict(budget=True), "budget"), (dict(head_dim=300), "head_dim"), (dict(dtype=torch.float32), "dtype"),
    (dict(recent=9), "recent"), (dict(recency_decay=-1.), "recency_decay"), (dict(recency_decay=math.nan), "recency_decay"),
])
def test_cache_arguments_are_checked(change, match):
    a = dict(batch=1, kv_heads=1, head_dim=8, budget=8, dtype=torch.float16, device="cpu")
    a.update(change)
    with pytest.raises(ValueError, match=match):
        DecodeCache(a.pop("batch"), a.pop("kv_heads"), a.pop("head_dim"), a.pop("budget"), **a)


def test_exports():
    for name in ("decode_attention", "replay_path", "insert_tokens", "DecodeCache"):
        assert name in flash_evict.__all__ and hasattr(flash_evict, name)


# The C entry points refuse before a launch: pointers are never followed.
P = ctypes.c_void_p(4096)
ST = (ctypes.c_int64 * 4)(1, 1, 1, 1)


def _attend_c(L, B=1, Hq=4, Hkv=2, T=3, C=8, D=16, dtype=1, scale=1., decay=0., ws=None, ws_bytes=None, imp=None, imp_st=8,
              length=P, st=ST, out=P, tree_st=0):
    if ws_bytes is None:
        ws_bytes = L.fe_decode_workspace_bytes(B, Hq, Hkv, T, C, D, imp is not None) - 1      # every call here is refused
    return L.fe_decode_attention(P, P, P, P, P, length, None, tree_st, out, P, imp, imp_st, None, 0, P, 8, P, B, Hq, Hkv, T, C, D,
                                 st, st, st, st, st, dtype, scale, decay, ws, ws_bytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(B=0), INVALID), (dict(Hq=3), INVALID), (dict(T=0), INVALID), (dict(T=257), INVALID), (dict(C=0), INVALID),
    (dict(D=0), INVALID), (dict(D=257), INVALID), (dict(dtype=2), INVALID), (dict(scale=math.inf), INVALID),
    (dict(decay=-1.), INVALID), (dict(decay=math.nan), INVALID), (dict(length=None), INVALID), (dict(out=None), INVALID),
    (dict(st=None), INVALID), (dict(st=(ctypes.c_int64 * 4)(1, 1, -1, 1)), INVALID), (dict(imp=P, imp_st=7), INVALID),
    (dict(tree_st=-1), INVALID), (dict(ws=None), WORKSPACE), (dict(ws=P), WORKSPACE),
    (dict(ws=ctypes.c_void_p(4104), ws_bytes=1 << 30), INVALID), (dict(out=ctypes.c_void_p(4100), ws=P, ws_bytes=1 << 30), INVALID),
    (dict(C=(1 << 30) + 1, imp_st=1 << 31), UNSUPPORTED), (dict(B=1 << 25), UNSUPPORTED), (dict(Hq=1 << 17, Hkv=1), UNSUPPORTED),
])
def test_c_decode_attention_refuses(change, code):
    L = _lib.lib()
    assert _attend_c(L, **change) == code
    assert L.fe_last_error().decode().startswith("fe_decode_attention")


def test_c_replay_path_refuses():
    L = _lib.lib()

    def call(T=3, A=2, path=P, lse=P, D=16, C=8, imp_st=8, B=1):
        return L.fe_replay_path(P, P, P, P, P, lse, path, P, imp_st, None, 0, P, 8, P, B, 4, 2, T, A, C, D, ST, ST, ST, ST, 1, 1., 0., None)

    for bad in (dict(A=0), dict(A=4), dict(path=None, A=2), dict(lse=None), dict(D=300), dict(imp_st=7), dict(B=0)):
        assert call(**bad) == INVALID, bad
        assert L.fe_last_error().decode().startswith("fe_replay_path")
    assert call(C=(1 << 30) + 1, imp_st=1 << 31) == UNSUPPORTED


def test_c_insert_tokens_refuses():
    L = _lib.lib()

    def call(B=1, Hkv=2, T=3, A=3, C=8, D=16, budget=8, recent=0, dtype=1, path=None, k=P, imp=P, imp_st=8, ws=None, ws_bytes=0, st=ST, pos_st=8):
        return L.fe_insert_tokens(k, k, P, P, imp, imp_st, P, pos_st, None, 0, P, P, None, path, B, Hkv, T, A, C, D, budget, recent,
                                  st, st, ST, ST, dtype, ws, ws_bytes, None)

    for bad in (dict(B=0), dict(Hkv=0), dict(T=-1), dict(A=2), dict(A=4, path=P), dict(C=0), dict(D=257), dict(budget=0), dict(budget=9),
                dict(recent=9), dict(recent=-1), dict(dtype=3), dict(k=None), dict(imp=None), dict(imp_st=7), dict(st=None)):
        assert call(**bad) == INVALID, bad
        assert L.fe_last_error().decode().startswith("fe_insert_tokens")
    assert call(C=(1 << 30) + 1, imp_st=1 << 31) == UNSUPPORTED
    assert call(B=1 << 16) == UNSUPPORTED
    # few rows need no workspace; a prompt's worth does
    assert L.fe_insert_workspace_bytes(1, 2, 3, 8, 8) == 0
    big = dict(T=300, A=300, C=1000, imp_st=1000, budget=900)
    need = L.fe_insert_workspace_bytes(1, 2, 300, 1000, 900)
    assert need >= 4 * 2 * 2 * 400
    # position_stride is 8 in every call: below 1000 slots
    assert call(**big) == INVALID
    assert call(pos_st=1000, **big) == WORKSPACE and call(pos_st=1000, ws=P, ws_bytes=need - 1, **big) == WORKSPACE


def test_workspace_sizes():
    L = _lib.lib()
    assert L.fe_decode_workspace_bytes(1, 3, 2, 1, 8, 16, 0) >= 0 and L.fe_decode_workspace_bytes(0, 4, 2, 1, 8, 16, 0) == 0
    assert L.fe_decode_workspace_bytes(1 << 40, 1 << 40, 1 << 40, 256, 1 << 40, 256, 1) == 0
    # partials of as many blocks as the card holds, whatever the cache's length; with weights, few rows' logits
    assert L.fe_decode_workspace_bytes(1, 32, 8, 1, 1 << 30, 128, 0) <= 16 << 20
    logits = 4 * 32 * 8 * 4 * (131072 // 32 + 1)
    size = [L.fe_decode_workspace_bytes(1, 32, 8, 1, 131072, 128, w) for w in (0, 1)]
    assert logits <= size[1] - size[0] <= logits + 256
    assert L.fe_decode_workspace_bytes(1, 32, 8, 32, 131072, 128, 1) == L.fe_decode_workspace_bytes(1, 32, 8, 32, 131072, 128, 0)
    assert L.fe_insert_workspace_bytes(1, 8, 0, 64, 64) == 0
