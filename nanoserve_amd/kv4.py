"""The paged KV cache held in 4 bits: its tensors, the write, the read-back and
the attention over it.

A layer's K and V are one uint8 tensor each,

    [num_blocks, num_kv_heads, block_size, head_dim / 2 + 4]

(the record of a (block, head) is described in include/nanoserve_paged.h): 36
bytes per row of 64 values where the 16-bit cache takes 128, 68 instead of 256
at head size 128.  Every row carries its own scale and offset in the model's
dtype, so a token is quantised when it is written and never again.

    Int4PagedKVCache              PagedKVCache with these tensors
    reshape_and_cache_int4        the write (kv_cache.reshape_and_cache)
    rope_reshape_and_cache_int4   rotary embedding and write (rotary.rope_reshape_and_cache)
    gather_cache_int4             the stored values of given slots
    paged_attention_int4          attn_fn over the cache (attention.paged_attention_hip)

The 16-bit counterparts restate the reference (nanoserve/kv_cache.py:30-85,
attention.py:99-190); the reference has no such cache.
"""

from __future__ import annotations

import torch

from . import _lib
from .attention import AttentionMetadata

_CODES = {torch.float16: _lib.NS_DTYPE_F16, torch.bfloat16: _lib.NS_DTYPE_BF16}


def kv4_shape(cache: torch.Tensor) -> tuple[int, int, int, int]:
    """(num_blocks, num_kv_heads, block_size, head_dim) of a cache tensor."""
    if cache.dim() != 4 or cache.dtype != torch.uint8 or cache.shape[3] < 8:
        raise ValueError("a 4-bit cache is a uint8 [num_blocks, num_kv_heads, block_size, head_dim / 2 + 4] tensor, "
                         f"got {cache.dtype} {tuple(cache.shape)}")
    return cache.shape[0], cache.shape[1], cache.shape[2], 2 * (cache.shape[3] - 4)


def kv4_bytes_per_token(num_layers: int, num_kv_heads: int, head_dim: int) -> int:
    """K and V bytes one token occupies across all layers (kv_cache.kv_bytes_per_token)."""
    return 2 * num_layers * num_kv_heads * (head_dim // 2 + 4)


# These wrappers run once per layer and step and hold no launch back by more
# than a few microseconds: every tensor attribute is read once, and no context
# manager stands around a call.  None of the ops is differentiable; what they
# return has no history.


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, what: str) -> tuple[int, int, int, int]:
    shape = k_cache.shape
    if len(shape) != 4 or k_cache.dtype is not torch.uint8 or shape[3] < 8:
        kv4_shape(k_cache)
    if v_cache.shape != shape or v_cache.dtype is not torch.uint8:
        raise ValueError(f"{what}: K and V caches must have one shape, got {tuple(shape)} and "
                         f"{v_cache.dtype} {tuple(v_cache.shape)}")
    if not k_cache.is_cuda or v_cache.device != k_cache.device:
        raise ValueError(f"{what} needs GPU tensors on one device (the HIP path has no CPU fallback)")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError(f"{what}: caches must be contiguous")
    return shape[0], shape[1], shape[2], 2 * (shape[3] - 4)


def _indices(t: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype is not torch.int64 and t.dtype is not torch.int32:
        t = t.to(torch.int64)
    return t


def _vector(t: torch.Tensor, name: str, least: int, device: torch.device) -> torch.Tensor:
    t = _indices(t, name, device)
    if t.dim() != 1 or t.shape[0] < least:
        raise ValueError(f"{name} must hold at least {least} entries, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _slots(slot_mapping: torch.Tensor, tokens: int, device: torch.device) -> torch.Tensor:
    if slot_mapping.dim() != 1 or slot_mapping.shape[0] != tokens:
        raise ValueError(f"slot_mapping must hold {tokens} slots, got {tuple(slot_mapping.shape)}")
    return _vector(slot_mapping, "slot_mapping", tokens, device)


def _rows(x: torch.Tensor, shape: tuple, dtype: torch.dtype, device: torch.device, name: str):
    """(x with a unit stride in its last dimension, its strides)."""
    if x.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {tuple(x.shape)}")
    if x.dtype is not dtype:
        raise TypeError(f"{name} is {x.dtype}, expected {dtype}")
    if x.device != device:
        raise ValueError(f"{name} is on {x.device}, expected {device}")
    stride = x.stride()
    if stride[-1] != 1:
        x = x.contiguous()
        stride = x.stride()
    return x, stride


def _model_dtype(dtype: torch.dtype, what: str) -> int:
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"{what} supports float16 and bfloat16, got {dtype}")
    return code


def reshape_and_cache_int4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                           slot_mapping: torch.Tensor) -> None:
    """Quantise the rows of key and value ([T, Hkv, D], any token and head
    strides) into their slots.  Slots outside the cache (e.g. -1 padding) are
    skipped; the others must differ."""
    what = "reshape_and_cache_int4"
    num_blocks, heads, block_size, head_dim = _caches(k_cache, v_cache, what)
    dtype, device = key.dtype, k_cache.device
    code = _model_dtype(dtype, what)
    T = key.shape[0] if key.dim() else 0
    key, ks = _rows(key, (T, heads, head_dim), dtype, device, "key")
    value, vs = _rows(value, (T, heads, head_dim), dtype, device, "value")
    slots = _slots(slot_mapping, T, device)
    if T == 0:
        return
    _lib.launch(device, what, _lib.load().ns_reshape_and_cache_int4,
                key.data_ptr(), value.data_ptr(), ks[0], ks[1], vs[0], vs[1], k_cache.data_ptr(), v_cache.data_ptr(),
                slots.data_ptr(), slots.dtype is torch.int64, T, heads, head_dim, block_size, num_blocks, code)


def rope_reshape_and_cache_int4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                                cos: torch.Tensor, sin: torch.Tensor,
                                k_cache: torch.Tensor, v_cache: torch.Tensor,
                                slot_mapping: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary embedding of q [T, Hq, D] and k [T, Hkv, D], quantising write of
    the rotated k and of v; returns the rotated q as a contiguous tensor (`out`
    when given; it may be q itself when q is contiguous).

    cos, sin: [T, 1, D] or [T, D] in q's dtype.  The rotation is evaluated in
    float32 and rounded once (q) or not at all before the codes are taken (k);
    rope_reshape_and_cache rounds after every product and sum instead."""
    what = "rope_reshape_and_cache_int4"
    num_blocks, heads, block_size, head_dim = _caches(k_cache, v_cache, what)
    dtype, device = q.dtype, k_cache.device
    code = _model_dtype(dtype, what)
    if q.dim() != 3 or q.shape[1] == 0:
        raise ValueError(f"q must be [T, Hq, {head_dim}] with a head at least, got {tuple(q.shape)}")
    T, Hq, _ = q.shape
    q, qs = _rows(q, (T, Hq, head_dim), dtype, device, "q")
    k, ks = _rows(k, (T, heads, head_dim), dtype, device, "k")
    v, vs = _rows(v, (T, heads, head_dim), dtype, device, "v")
    tables = (T, head_dim), (T, 1, head_dim)
    cos, cs = _rows(cos, tables[cos.dim() == 3], dtype, device, "cos")
    sin, ss = _rows(sin, tables[sin.dim() == 3], dtype, device, "sin")
    if cs[0] != ss[0]:
        cos, sin = cos.contiguous(), sin.contiguous()
        cs = cos.stride()
    slots = _slots(slot_mapping, T, device)
    if out is None:
        out = torch.empty((T, Hq, head_dim), dtype=dtype, device=device)
    elif out.shape != (T, Hq, head_dim) or out.dtype != dtype or out.device != device or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous [{T}, {Hq}, {head_dim}] {dtype} tensor on {device}")
    elif out.data_ptr() == q.data_ptr() and not q.is_contiguous():
        raise ValueError("out may alias q only when q is contiguous")
    if T == 0:
        return out
    _lib.launch(device, what, _lib.load().ns_rope_reshape_and_cache_int4,
                out.data_ptr(), q.data_ptr(), qs[0], qs[1], k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                cos.data_ptr(), sin.data_ptr(), cs[0], k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(),
                slots.dtype is torch.int64, T, Hq, heads, head_dim, block_size, num_blocks, code)
    return out


def gather_cache_int4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                      dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The values stored in the given slots, (K, V) as [T, Hkv, D] tensors of
    `dtype`, the dtype the cache was written in; zero rows for slots outside
    the cache.  For moving a cached prefix, and for looking at a cache."""
    what = "gather_cache_int4"
    num_blocks, heads, block_size, head_dim = _caches(k_cache, v_cache, what)
    code = _model_dtype(dtype, what)
    device = k_cache.device
    T = slot_mapping.shape[0] if slot_mapping.dim() else 0
    slots = _slots(slot_mapping, T, device)
    k, v = torch.empty((2, T, heads, head_dim), dtype=dtype, device=device).unbind()
    if T:
        _lib.launch(device, what, _lib.load().ns_gather_cache_int4,
                    k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr(),
                    slots.dtype is torch.int64, T, heads, head_dim, block_size, num_blocks, code)
    return k, v


def paged_attention_int4(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         md: AttentionMetadata, scale: float) -> torch.Tensor:
    """Paged attention over a cache held in 4 bits: attn_fn's contract
    (attention.paged_attention_hip) with the caches of Int4PagedKVCache, in the
    dtype they were written in.  Returns [num_tokens, num_heads, head_dim], with
    zeros for rows without keys and rows behind the last sequence.

    The device's lengths, offsets and tables decide what is computed; the host's
    lists in `md`, where there are any, shape the launches and, outside of a
    graph capture, tell whether every row belongs to a sequence."""
    what = "paged_attention_int4"
    num_blocks, heads, block_size, head_dim = _caches(k_cache, v_cache, what)
    code = _model_dtype(query.dtype, what)
    device = k_cache.device
    shape = query.shape
    if len(shape) != 3 or shape[2] != head_dim:
        raise ValueError(f"query must be [T, Hq, {head_dim}], got {tuple(shape)}")
    if query.device != device:
        raise ValueError(f"query is on {query.device}, expected {device}")
    T, Hq, _ = shape
    n, longest = md.num_seqs, md.max_seq_len
    if md.num_tokens != T:
        raise ValueError(f"metadata has {md.num_tokens} tokens, query has {T}")
    if md.tree_mask is not None:
        raise ValueError(f"{what} takes no tree_mask: trees of drafted tokens need a 16-bit cache")
    if Hq % heads:
        raise ValueError(f"{Hq} query heads over {heads} KV heads")
    q = query if query.is_contiguous() else query.contiguous()
    if T == 0 or n == 0:
        return torch.zeros_like(q)
    bt = _indices(md.block_tables, "block_tables", device)
    if bt.dim() != 2 or bt.shape[0] < n:
        raise ValueError(f"block_tables must be [num_seqs, max_blocks], got {tuple(bt.shape)}")
    width = bt.shape[1]
    if width * block_size < longest:
        raise ValueError(f"block_tables has {width} columns but max_seq_len={longest} needs {-(-longest // block_size)}")
    bs = bt.stride()
    if bs[1] != 1 or bs[0] < width:
        bt = bt.contiguous()
        bs = bt.stride()
    sl = _vector(md.seq_lens, "seq_lens", n, device)
    decode_only = bool(md.is_decode_only)
    qsl_ptr, qsl64 = None, 0
    if decode_only:
        if T != n:
            raise ValueError("is_decode_only needs one query token per sequence")
        out = torch.empty_like(q)
    else:
        qsl = _vector(md.query_start_loc, "query_start_loc", n + 1, device)
        qsl_ptr, qsl64 = qsl.data_ptr(), qsl.dtype is torch.int64
        # Rows behind the last sequence are not written: zero unless the host
        # offsets show that there are none, which they cannot for the replays
        # of a capture.
        host = md.query_start_loc_cpu
        full = (host is not None and len(host) > n and host[0] == 0 and host[n] == T
                and not torch.cuda.is_current_stream_capturing())
        out = torch.empty_like(q) if full else torch.zeros_like(q)
    # The context lengths' sum and the number of decode rows, where the host
    # has them, shape the launches.  The partial results live in a tensor of
    # this call's: captured graphs hold their own, and calls on different
    # streams share nothing.
    lens, rows = md.seq_lens_cpu, md.query_lens_cpu
    context = 0 if lens is None else sum(lens if len(lens) == n else lens[:n])
    ones = n if decode_only else -1 if rows is None else rows[:n].count(1)
    lib = _lib.load()
    nbytes = lib.ns_paged_attention_int4_workspace_size(n, Hq, heads, head_dim, block_size, longest, T, decode_only,
                                                        context, ones)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    _lib.launch(device, what, lib.ns_paged_attention_int4,
                out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                bt.data_ptr(), bs[0], width, bt.dtype is torch.int64, sl.data_ptr(), sl.dtype is torch.int64,
                qsl_ptr, qsl64, n, T, longest, decode_only, context, ones, Hq, heads, head_dim, block_size, num_blocks,
                float(scale), code, None if ws is None else ws.data_ptr(), nbytes)
    return out


class Int4PagedKVCache:
    """PagedKVCache (kv_cache.py) with K and V held in 4 bits.  `dtype` is the
    model's, float16 or bfloat16: the dtype of the rows written and of every
    row's scale and offset."""

    bits = 4

    def __init__(self, num_blocks: int, block_size: int, num_layers: int, num_kv_heads: int, head_dim: int,
                 dtype: torch.dtype, device: str) -> None:
        _model_dtype(dtype, "Int4PagedKVCache")
        if head_dim <= 0 or head_dim % 8 or head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {head_dim}")
        if block_size <= 0 or block_size % 4:
            raise ValueError(f"block_size must be a multiple of 4, got {block_size}")
        self.num_blocks = num_blocks
        self.block_size = block_size
        self.num_layers = num_layers
        self.num_kv_heads = num_kv_heads
        self.head_dim = head_dim
        self.dtype = dtype
        self.device = device

        shape = (num_blocks, num_kv_heads, block_size, head_dim // 2 + 4)
        self.k_cache = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(num_layers)]
        self.v_cache = [torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(num_layers)]

    @property
    def num_bytes(self) -> int:
        return sum(t.numel() for t in self.k_cache + self.v_cache)

    @property
    def capacity_tokens(self) -> int:
        return self.num_blocks * self.block_size

    def write(self, layer: int, key: torch.Tensor, value: torch.Tensor, slot_mapping: torch.Tensor) -> None:
        """Quantise this step's K/V rows ([T, Hkv, D]) into their slots."""
        reshape_and_cache_int4(key, value, self.k_cache[layer], self.v_cache[layer], slot_mapping)

    def read(self, layer: int, slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """The stored (K, V) rows of the given slots, [T, Hkv, D] in the model's dtype."""
        return gather_cache_int4(self.k_cache[layer], self.v_cache[layer], slot_mapping, self.dtype)

    def zero_(self) -> None:
        for t in self.k_cache + self.v_cache:
            t.zero_()
