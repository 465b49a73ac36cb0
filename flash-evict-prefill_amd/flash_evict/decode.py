"""Decoding over a bounded KV cache on MI355X: attention of new tokens and drafted trees over the
cache, accumulation of the attention weight its rows receive, and eviction of the least of them.

`prefill` scores a prompt's tokens and `select_tokens` keeps the best of them; these operators go
on from there while a model generates. The reference has no counterpart: its decode cache only
grows (flash_evict/quality_adapter.py:116-136 in anishesg/flash-evict-prefill).

  decode_attention  new tokens over the cache and each other; importance of what they saw
  replay_path       the importance of a drafted tree's accepted path alone
  insert_tokens     new tokens enter the cache, the rows of least importance leave it, in place
  DecodeCache       one layer's cache with these three as `decode`, `draft`, `accept` and `evict`

Continuing a prompt chunk by chunk gives the importance `prefill` gives the whole: both weight
query t by exp(recency_decay * (t - newest)), and both may weight a key by its value's L1 norm.
The work runs in the library's kernels (fe_decode_attention, fe_replay_path, fe_insert_tokens) on
the current stream of the tensors' device; nothing synchronises, and lengths stay on the device,
so a step can be captured in a graph. Inference only, fp16 and bf16, head dims up to 256. The
kernels read 16 bytes at a time where the channel stride is 1, the head dim a multiple of 8 and
rows lie on 16-byte boundaries, and element by element otherwise.
"""
import functools
import math

import torch

from . import _lib
from .prefill import _DTYPES, _is_int

__all__ = ["DecodeCache", "decode_attention", "insert_tokens", "replay_path"]

MAX_TOKENS = 256    # new tokens of one call (a longer chunk is passed in parts)


def _check_new(q, k, v, k_cache, scale, recency_decay):
    """Shape, type and device rules shared by decode_attention and replay_path; the sizes, device,
    dtype, scale and decay."""
    qs, ks, cs = q.shape, k.shape, k_cache.shape
    if len(qs) != 4 or len(ks) != 4 or v.ndim != 4 or len(cs) != 4:
        raise ValueError("q must have shape [batch, heads, tokens, channels], k, v and the cache [batch, kv_heads, rows, channels]")
    b, hq, t, d = qs
    hk, c = ks[1], cs[2]
    if b < 1 or hq < 1 or t < 1 or d < 1 or hk < 1 or c < 1 or ks != (b, hk, t, d) or v.shape != ks or cs != (b, hk, c, d):
        raise ValueError("Expected nonempty q, k, v of equal batch, tokens and channels and a cache of their batch, KV heads and channels")
    if hq % hk or d > 256:
        raise ValueError("Query heads must be divisible by KV heads; head dimension must be <= 256")
    if t > MAX_TOKENS:
        raise ValueError("at most %d new tokens in one call" % MAX_TOKENS)
    device, dtype = q.device, q.dtype
    if not q.is_cuda or dtype not in _DTYPES:
        raise ValueError("CUDA fp16 or bf16 inputs required")
    if k.device != device or v.device != device or k_cache.device != device or k.dtype != dtype or v.dtype != dtype \
            or k_cache.dtype != dtype:
        raise ValueError("q, k, v and the cache must have the same device and dtype")
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_cache.requires_grad):
        raise ValueError("Inference only: no backward implementation")
    scale = d ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError("scale must be finite")
    recency_decay = float(recency_decay)
    if not (0. <= recency_decay < math.inf):
        raise ValueError("recency_decay must be finite and nonnegative")
    return b, hq, hk, t, c, d, device, dtype, scale, recency_decay


@functools.lru_cache(maxsize=4096)
def _decode_workspace(*sizes):
    return _lib.lib().fe_decode_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _insert_workspace(*sizes):
    return _lib.lib().fe_insert_workspace_bytes(*sizes)


def _check_heads(x, name, b, hk, device):
    """A [B, Hkv] int32 tensor the kernels index as b * Hkv + head."""
    if x.shape != (b, hk) or x.dtype != torch.int32 or x.device != device or not x.is_contiguous():
        raise ValueError("%s must be a contiguous int32 [batch, kv_heads] tensor on the cache's device" % name)


def _rows(x, name, shape, dtype, device, write):
    """Row stride of a [B, Hkv, C] slot tensor. Written ones must lie as evenly spaced rows of
    unit stride; a read one that does not is copied. Returns (tensor, stride)."""
    if x.shape != shape or x.dtype != dtype or x.device != device:
        raise ValueError("%s must be a %s [batch, kv_heads, slots] tensor of the cache's size, on its device"
                         % (name, str(dtype).replace("torch.", "")))
    sb, sh, sc = x.stride()
    b, hk, c = shape
    if hk == 1:
        sh = sb if b > 1 else c
    if (sc == 1 or c == 1) and sh >= c and (b == 1 or sb == hk * sh):
        return x, sh
    if write:
        raise ValueError("%s is written: it must have unit-stride rows, evenly spaced" % name)
    return x.contiguous(), c


def _check_tree(tree, b, t, device):
    if tree.dtype != torch.bool or tree.device != device or tree.shape not in ((t, t), (b, t, t)):
        raise ValueError("tree must be a bool [tokens, tokens] or [batch, tokens, tokens] mask on the inputs' device")
    tree = tree.contiguous()
    return tree, (t * t if tree.ndim == 3 else 0)


def _check_path(path, b, t, device):
    if path.ndim != 2 or path.shape[0] != b or not 1 <= path.shape[1] <= t or path.dtype != torch.int32 or path.device != device:
        raise ValueError("path must be an int32 [batch, nodes] tensor of 1 to `tokens` nodes on the inputs' device")
    return path.contiguous()


def decode_attention(q, k, v, k_cache, v_cache, length, *, tree=None, scale=None, importance=None, value_norm=None,
                     recency_decay=0., importance_out=None):
    """Attention of new tokens over a cache and each other.

    q [B, Hq, T, D] and k, v [B, Hkv, T, D] are T <= 256 new tokens, not in the cache yet; k_cache,
    v_cache [B, Hkv, C, D] hold length[b, j] rows (int32 [B, Hkv], read as clamped to [0, C]), every
    one visible to every query. `tree` (bool [T, T] or [B, T, T]) says which new tokens u query t
    sees, tree[t, u]; None is a causal chunk, u <= t. Whatever a hidden token holds, infinities and
    NaN too, reaches no query it is hidden from.

    Returns (out [B, Hq, T, D], lse [B, Hq, T] FP32 natural log-sum-exp, importance, new_importance).
    A query that sees nothing has zeros and -inf. The last two are None unless `importance` (FP32
    [B, Hkv, C]) is given: then all T tokens stay, w[t] = exp(recency_decay * (t - (T-1))), and
      importance[s] * exp(-recency_decay * T) + value_norm[s] * sum_(g,t) w[t] p[g,t,s]
    goes to `importance_out` (default: a copy of `importance`; `importance` itself updates it in
    place) for the slots below length, and new_importance [B, Hkv, T] is the new tokens' own, with
    their values' L1 norms. Without value_norm (FP32 [B, Hkv, C]) neither is weighted by a norm.
    For a drafted tree leave `importance` out, and call replay_path once the path is known.
    """
    b, hq, hk, t, c, d, device, dtype, scale, recency_decay = _check_new(q, k, v, k_cache, scale, recency_decay)
    if v_cache.shape != k_cache.shape or v_cache.device != device or v_cache.dtype != dtype:
        raise ValueError("k_cache and v_cache must have the same shape, device and dtype")
    _check_heads(length, "length", b, hk, device)
    tree_ptr, tree_stride = None, 0
    if tree is not None:
        tree, tree_stride = _check_tree(tree, b, t, device)
        tree_ptr = tree.data_ptr()
    new = imp_ptr = norm_ptr = out_ptr = new_ptr = None
    imp_st = norm_st = out_st = 0
    if importance is not None:
        slots = (b, hk, c)
        importance, imp_st = _rows(importance, "importance", slots, torch.float32, device, False)
        if value_norm is not None:
            value_norm, norm_st = _rows(value_norm, "value_norm", slots, torch.float32, device, False)
            norm_ptr = value_norm.data_ptr()
        if importance_out is None:
            importance_out = importance.clone(memory_format=torch.contiguous_format)
        importance_out, out_st = _rows(importance_out, "importance_out", slots, torch.float32, device, True)
        new = torch.empty((b, hk, t), dtype=torch.float32, device=device)
        imp_ptr, out_ptr, new_ptr = importance.data_ptr(), importance_out.data_ptr(), new.data_ptr()
    elif value_norm is not None or importance_out is not None:
        raise ValueError("value_norm and importance_out go with importance")
    out = torch.empty((b, hq, t, d), dtype=dtype, device=device)
    lse = torch.empty((b, hq, t), dtype=torch.float32, device=device)
    L = _lib.lib()
    ws_bytes = _decode_workspace(b, hq, hk, t, c, d, importance is not None)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    with _lib.on_device(device):
        rc = L.fe_decode_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                   length.data_ptr(), tree_ptr, tree_stride, out.data_ptr(), lse.data_ptr(), imp_ptr, imp_st,
                                   norm_ptr, norm_st, out_ptr, out_st, new_ptr, b, hq, hk, t, c, d, _lib.strides(q),
                                   _lib.strides(k), _lib.strides(v), _lib.strides(k_cache), _lib.strides(v_cache),
                                   _DTYPES[dtype], scale, recency_decay, ws.data_ptr(), ws_bytes,
                                   _lib.current_stream(device))
    _lib.check(rc, "fe_decode_attention")
    return out, lse, importance_out, new


def replay_path(q, k, v, k_cache, length, lse, path, importance, *, scale=None, value_norm=None, recency_decay=0.,
                importance_out=None):
    """Importance of a drafted tree's accepted path: (importance, new_importance [B, Hkv, A]).

    q, k, v, k_cache, length, scale and lse are those of the tree's decode_attention. path (int32
    [B, A], 1 <= A <= T) holds the accepted nodes from the root on; a row ends before its first
    entry outside [0, T) (-1 pads it), and may be empty. The path's i-th query sees the cache and
    the path up to itself; recency counts back from the path's last node. importance, value_norm
    and importance_out are as in decode_attention; new_importance is 0 past a path's end. None as
    the path stands for all T tokens in order.
    """
    b, hq, hk, t, c, d, device, dtype, scale, recency_decay = _check_new(q, k, v, k_cache, scale, recency_decay)
    _check_heads(length, "length", b, hk, device)
    if lse.shape != (b, hq, t) or lse.dtype != torch.float32 or lse.device != device:
        raise ValueError("lse must be the float32 [batch, heads, tokens] of decode_attention")
    lse = lse.contiguous()
    a = t
    if path is not None:
        path = _check_path(path, b, t, device)
        a = path.shape[1]
    slots = (b, hk, c)
    importance, imp_st = _rows(importance, "importance", slots, torch.float32, device, False)
    norm_st = 0
    if value_norm is not None:
        value_norm, norm_st = _rows(value_norm, "value_norm", slots, torch.float32, device, False)
    if importance_out is None:
        importance_out = importance.clone(memory_format=torch.contiguous_format)
    importance_out, out_st = _rows(importance_out, "importance_out", slots, torch.float32, device, True)
    new = torch.empty((b, hk, a), dtype=torch.float32, device=device)
    L = _lib.lib()
    with _lib.on_device(device):
        rc = L.fe_replay_path(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), length.data_ptr(), lse.data_ptr(),
                              None if path is None else path.data_ptr(), importance.data_ptr(), imp_st,
                              None if value_norm is None else value_norm.data_ptr(), norm_st, importance_out.data_ptr(), out_st,
                              new.data_ptr(), b, hq, hk, t, a, c, d, _lib.strides(q), _lib.strides(k), _lib.strides(v),
                              _lib.strides(k_cache), _DTYPES[dtype], scale, recency_decay, _lib.current_stream(device))
    _lib.check(rc, "fe_replay_path")
    return importance_out, new


def insert_tokens(k, v, k_cache, v_cache, importance, position, length, seen, budget, *, recent=0, new_importance=None,
                  value_norm=None, path=None):
    """New tokens enter the cache and the rows of least importance leave it, in place.

    Per (batch row, KV head) the candidates are the cache's length rows and the new rows behind
    them: all T of k, v [B, Hkv, T, D], or the nodes of `path` (as in replay_path; each may be
    named again). min(candidates, budget) stay: first the rows whose position is among the newest
    `recent`, then those of the largest importance (ties keep the lower slot, NaN ranks above every
    number). Kept rows below that count keep their slots; the others, in order, take the slots that
    were vacated, in order. So slots are in no particular order, and a step costs what it evicts.

    Updated in place: k_cache, v_cache [B, Hkv, C, D], importance (FP32) and position (int32)
    [B, Hkv, C], length and seen (int32 [B, Hkv]: rows in use, and tokens ever inserted, which new
    rows' positions count on from), value_norm (FP32 [B, Hkv, C]) where given. Slots from the new
    length on are left as they were. new_importance is FP32 [B, Hkv, T or A], None for zeros.
    k = v = None inserts nothing: an eviction down to `budget`. 1 <= budget <= C, recent <= budget.
    """
    cs = k_cache.shape
    if len(cs) != 4 or v_cache.shape != cs or min(cs) < 1 or cs[3] > 256:
        raise ValueError("The cache must be two nonempty [batch, kv_heads, slots, channels] tensors of at most 256 channels")
    b, hk, c, d = cs
    device, dtype = k_cache.device, k_cache.dtype
    if not k_cache.is_cuda or dtype not in _DTYPES or v_cache.device != device or v_cache.dtype != dtype:
        raise ValueError("CUDA fp16 or bf16 caches of one device and dtype required")
    if (k is None) != (v is None) or (k is None and (path is not None or new_importance is not None)):
        raise ValueError("k and v come together, path and new_importance with them")
    t = 0
    if k is not None:
        ks = k.shape
        if len(ks) != 4 or v.shape != ks or ks != (b, hk, ks[2], d):
            raise ValueError("k and v must be [batch, kv_heads, tokens, channels] tensors like the cache")
        if k.device != device or v.device != device or k.dtype != dtype or v.dtype != dtype:
            raise ValueError("k, v and the cache must have the same device and dtype")
        t = ks[2]
        # in place, and in no order: the new rows may not lie in the cache's memory
        mine = (k_cache.untyped_storage().data_ptr(), v_cache.untyped_storage().data_ptr())
        if t and (k.untyped_storage().data_ptr() in mine or v.untyped_storage().data_ptr() in mine):
            raise ValueError("k and v may not share the cache's memory")
    for x, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        st = x.stride()
        if 0 in st and any(y == 0 and z > 1 for y, z in zip(st, x.shape)):
            raise ValueError("%s is written: it may not be expanded" % name)
    if torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad or importance.requires_grad
                                    or (k is not None and (k.requires_grad or v.requires_grad))):
        raise ValueError("Inference only: no backward implementation")
    if not _is_int(budget) or not 1 <= budget <= c:
        raise ValueError("budget must be an integer in [1, cache slots]")
    if not _is_int(recent) or not 0 <= recent <= budget:
        raise ValueError("recent must be an integer in [0, budget]")
    _check_heads(length, "length", b, hk, device)
    _check_heads(seen, "seen", b, hk, device)
    slots = (b, hk, c)
    importance, imp_st = _rows(importance, "importance", slots, torch.float32, device, True)
    position, pos_st = _rows(position, "position", slots, torch.int32, device, True)
    norm_st, a = 0, t
    if value_norm is not None:
        value_norm, norm_st = _rows(value_norm, "value_norm", slots, torch.float32, device, True)
    if path is not None:
        path = _check_path(path, b, t, device)
        a = path.shape[1]
    if new_importance is not None:
        if new_importance.shape != (b, hk, a) or new_importance.dtype != torch.float32 or new_importance.device != device:
            raise ValueError("new_importance must be a float32 [batch, kv_heads, new rows] tensor on the cache's device")
        new_importance = new_importance.contiguous()
    if t == 0:
        k = v = k_cache                     # strides of a size-0 axis are not read
    L = _lib.lib()
    ws_bytes = _insert_workspace(b, hk, a, c, budget)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
    with _lib.on_device(device):
        rc = L.fe_insert_tokens(k.data_ptr() if t else None, v.data_ptr() if t else None, k_cache.data_ptr(), v_cache.data_ptr(),
                                importance.data_ptr(), imp_st, position.data_ptr(), pos_st,
                                None if value_norm is None else value_norm.data_ptr(), norm_st, length.data_ptr(),
                                seen.data_ptr(), None if new_importance is None else new_importance.data_ptr(),
                                None if path is None else path.data_ptr(), b, hk, t, a, c, d, budget, recent, _lib.strides(k),
                                _lib.strides(v), _lib.strides(k_cache), _lib.strides(v_cache), _DTYPES[dtype],
                                None if ws is None else ws.data_ptr(), ws_bytes, _lib.current_stream(device))
    _lib.check(rc, "fe_insert_tokens")


class DecodeCache:
    """One attention layer's KV cache of at most `budget` rows per (batch row, KV head).

    Rows hold K, V and, per slot, their accumulated importance, position and value norm (`k`, `v`,
    `importance`, `position`, `value_norm`; `length` and `seen` per head). `recent` newest tokens
    are never evicted. `recency_decay` and `value_weighted` are prefill's.

      load(k, v, importance)    start from a prompt: its K, V and prefill importance
      decode(q, k, v)           tokens that stay: their attention, then they enter the cache
      draft(q, k, v, tree)      drafted tokens: their attention alone
      accept(q, k, v, lse, path)    the drafted tokens that stay enter the cache
      evict(budget)             down to fewer rows
    """

    def __init__(self, batch, kv_heads, head_dim, budget, *, dtype, device, recent=0, recency_decay=0., value_weighted=True):
        for name, x in (("batch", batch), ("kv_heads", kv_heads), ("head_dim", head_dim), ("budget", budget)):
            if not _is_int(x) or x < 1:
                raise ValueError("%s must be a positive integer" % name)
        if head_dim > 256 or dtype not in _DTYPES:
            raise ValueError("head_dim must be <= 256 and dtype fp16 or bf16")
        if not _is_int(recent) or not 0 <= recent <= budget:
            raise ValueError("recent must be an integer in [0, budget]")
        recency_decay = float(recency_decay)
        if not math.isfinite(recency_decay) or recency_decay < 0:
            raise ValueError("recency_decay must be finite and nonnegative")
        slots = (batch, kv_heads, budget)
        self.budget, self.recent, self.recency_decay = budget, recent, recency_decay
        self.k = torch.zeros((*slots, head_dim), dtype=dtype, device=device)
        self.v = torch.zeros((*slots, head_dim), dtype=dtype, device=device)
        self.importance = torch.zeros(slots, dtype=torch.float32, device=device)
        self.position = torch.zeros(slots, dtype=torch.int32, device=device)
        self.value_norm = torch.zeros(slots, dtype=torch.float32, device=device) if value_weighted else None
        self.length = torch.zeros(slots[:2], dtype=torch.int32, device=device)
        self.seen = torch.zeros(slots[:2], dtype=torch.int32, device=device)

    def _insert(self, k, v, new_importance=None, path=None, budget=None):
        budget = self.budget if budget is None else budget
        insert_tokens(k, v, self.k, self.v, self.importance, self.position, self.length, self.seen, budget,
                      recent=min(self.recent, budget), new_importance=new_importance, value_norm=self.value_norm, path=path)

    def reset(self):
        """Empty the cache."""
        self.length.zero_()
        self.seen.zero_()

    def load(self, k, v, importance=None, position=None, seen=None):
        """Start from tokens k, v [B, Hkv, N, D] with their importance [B, Hkv, N] (None: zeros); of
        more than `budget` the most important stay. `position` [B, Hkv, N] and `seen` tell where the
        tokens of an already compacted cache (N <= budget) stood, and how many tokens there were."""
        n = k.shape[2]
        if position is not None and (n > self.budget or position.shape != k.shape[:3]):
            raise ValueError("position must be [batch, kv_heads, tokens], of at most `budget` tokens")
        self.reset()
        if importance is not None and importance.dtype != torch.float32:
            importance = importance.float()
        self._insert(k, v, importance)
        if position is not None:
            self.position[:, :, :n] = position
        if seen is not None:
            self.seen.fill_(seen)

    def decode(self, q, k, v, *, scale=None):
        """Attention output [B, Hq, T, D] of a causal chunk of new tokens, which then enter the cache;
        the rows they looked at least may leave it."""
        out, _, _, new = decode_attention(q, k, v, self.k, self.v, self.length, scale=scale, importance=self.importance,
                                          value_norm=self.value_norm, recency_decay=self.recency_decay,
                                          importance_out=self.importance)
        self._insert(k, v, new)
        return out

    def draft(self, q, k, v, tree, *, scale=None):
        """(out, lse) of drafted tokens; the cache stays as it is."""
        return decode_attention(q, k, v, self.k, self.v, self.length, tree=tree, scale=scale)[:2]

    def accept(self, q, k, v, lse, path, *, scale=None):
        """The drafted tokens on `path` (int32 [B, A]) stay: what they looked at counts, and they enter the cache."""
        _, new = replay_path(q, k, v, self.k, self.length, lse, path, self.importance, scale=scale, value_norm=self.value_norm,
                             recency_decay=self.recency_decay, importance_out=self.importance)
        self._insert(k, v, new, path)

    def evict(self, budget):
        """Evict down to `budget` rows a head (the cache's own budget stays)."""
        self._insert(None, None, budget=budget)
