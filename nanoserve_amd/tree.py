"""A decode step that verifies drafted tokens: its addresses, attention for trees
of drafted tokens over the paged cache, and the commit of the accepted rows.

The reference computes one token per request and decode step
(nanoserve/model_runner.py:85-147).  Here a request's rows in a step are its last
token (row 0) and drafted ones, at most 64: a tree, whose rows name an earlier
row as their parent.  Row j's K and V take cache position c + j, c being the
tokens of the request with K and V before the step; its rotary position is c plus
its depth.

    step_inputs            lengths and new blocks -> offsets, positions, slots,
                           packed block tables and the rows' ancestors
    paged_attention_tree   attn_fn for such rows (paged_attention_hip calls it for
                           an md with a tree_mask)
    commit_drafts          the rows that the model's choices confirm, and their K
                           and V moved to the places of the tokens they became

Each is one launch on the current stream and reads the device's lengths, so a
captured graph serves other lengths, trees and choices on every replay.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from .attention import AttentionMetadata

MAX_TREE_ROWS = 64  # rows of a request that a 64-bit mask can name


@dataclass(frozen=True)
class StepInputs:
    """A step's addresses on the device, as AttentionMetadata takes them (int64;
    block_tables in the tables' dtype)."""

    query_start_loc: torch.Tensor         # [B + 1]
    seq_lens: torch.Tensor                # [B]
    positions: torch.Tensor               # [T]
    slot_mapping: torch.Tensor            # [T]
    block_tables: torch.Tensor            # [B, max_blocks]
    tree_mask: torch.Tensor | None        # [T], with parents


def _integers(tensors: dict, device: torch.device) -> tuple[dict, bool]:
    """The tensors (name -> tensor or None, and its length) contiguous and of one integer dtype; whether that is int64."""
    kinds = set()
    for name, (t, n) in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, expected {device}")
        if t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} must hold {n} entries, got {tuple(t.shape)}")
        if t.dtype is not torch.int64 and t.dtype is not torch.int32:
            raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
        kinds.add(t.dtype)
    wide = kinds != {torch.int32}
    out = {}
    for name, (t, _) in tensors.items():
        if t is not None and wide and t.dtype is torch.int32:
            t = t.to(torch.int64)
        out[name] = t if t is None or t.is_contiguous() else t.contiguous()
    return out, wide


def _pointer(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def step_inputs(tables: torch.Tensor, rows: torch.Tensor, computed: torch.Tensor, query_lens: torch.Tensor,
                num_tokens: int, block_size: int, max_blocks: int, new_blocks: torch.Tensor | None = None,
                new_start: torch.Tensor | None = None, held: torch.Tensor | None = None,
                parents: torch.Tensor | None = None) -> StepInputs:
    """The addresses of a step over B requests, on the device.

    tables [R, W] (int32 or int64, unit column stride) keeps the requests' block
    ids from step to step and is written: request i appends new_blocks[new_start[i]
    : new_start[i + 1]] to row rows[i] from column held[i] on (all three or none).
    computed [B] are the tokens with K and V, query_lens [B] the rows of this step,
    num_tokens their sum or more (rows behind the last request get slot -1),
    max_blocks the width of the packed tables.  parents [num_tokens]: every row's
    parent among its request's rows, -1 for a root; None: no trees.

    A row or block outside a table has slot and id -1.  The table rows must differ
    where blocks are appended; requests in a tree have at most 64 rows."""
    what = "step_inputs"
    if tables.dim() != 2 or tables.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tables must be [requests, blocks] of int32 or int64, got {tables.dtype} {tuple(tables.shape)}")
    if not tables.is_cuda:
        raise ValueError(f"{what} needs GPU tensors (the HIP path has no CPU fallback)")
    R, W = tables.shape
    if R and W and (tables.stride(1) != 1 and W > 1 or tables.stride(0) < W and R > 1):
        raise ValueError("tables must have contiguous rows that do not overlap")
    if num_tokens < 0 or block_size <= 0 or max_blocks < 0:
        raise ValueError(f"num_tokens {num_tokens}, block_size {block_size} and max_blocks {max_blocks} are no sizes")
    given = [x is not None for x in (new_blocks, new_start, held)]
    if any(given) and not all(given):
        raise ValueError("new_blocks, new_start and held belong together")
    device = tables.device
    B = rows.shape[0] if rows.dim() else 0
    N = 0 if new_blocks is None else new_blocks.numel()
    x, wide = _integers({"rows": (rows, B), "computed": (computed, B), "query_lens": (query_lens, B),
                         "new_blocks": (new_blocks, N), "new_start": (new_start, B + 1), "held": (held, B),
                         "parents": (parents, num_tokens)}, device)
    per_token = 2 if parents is None else 3
    # One allocation for every int64 output.
    flat = torch.empty(2 * B + 1 + per_token * num_tokens, dtype=torch.int64, device=device)
    qsl, lens, positions, slots, *mask = flat.split([B + 1, B] + [num_tokens] * per_token)
    packed = torch.empty((B, max_blocks), dtype=tables.dtype, device=device)
    out = StepInputs(qsl, lens, positions, slots, packed, mask[0] if mask else None)
    _lib.launch(device, what, _lib.load().ns_step_inputs,
                tables.data_ptr(), R, W, max(tables.stride(0), W), tables.dtype is torch.int64,
                _pointer(x["rows"]), _pointer(x["computed"]), _pointer(x["query_lens"]),
                _pointer(x["new_blocks"]), _pointer(x["new_start"]), _pointer(x["held"]), N,
                _pointer(x["parents"]), wide, B, num_tokens, block_size, max_blocks,
                qsl.data_ptr(), lens.data_ptr(), positions.data_ptr(), slots.data_ptr(), packed.data_ptr(),
                _pointer(out.tree_mask))
    return out


# Arrival counters of the key ranges, zero before and after every call, one
# buffer per (device, stream): calls on one stream follow each other.  A call
# that is recorded into a graph gets its own, cleared by the graph, so that graphs
# share none whichever streams they are replayed on.
_counters: dict[tuple[int, int], torch.Tensor] = {}


def _arrivals(device: torch.device) -> torch.Tensor:
    n = _lib.load().ns_paged_attention_tree_counters()
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(n, dtype=torch.int32, device=device)
    key = (device.index, torch._C._cuda_getCurrentRawStream(device.index))
    c = _counters.get(key)
    if c is None:
        c = _counters[key] = torch.zeros(n, dtype=torch.int32, device=device)
    return c


def paged_attention_tree(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         md: AttentionMetadata, scale: float) -> torch.Tensor:
    """Paged attention for trees of drafted tokens: attn_fn's contract
    (attention.paged_attention_hip) with md.tree_mask.  Row j of a sequence with
    context length L and q <= 64 rows sees keys 0 .. L - q - 1, and key L - q + i
    where bit i of its mask is set.  Returns [num_tokens, num_heads, head_dim],
    with zeros for rows without keys and rows behind the last sequence.

    float32, float16 and bfloat16, head sizes up to 256.  The device's lengths,
    offsets, masks and tables decide what is computed; of the host's only
    max_query_len, max_seq_len and query_start_loc_cpu are read, and shape the
    launch."""
    what = "paged_attention_tree"
    if query.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(
            f"expected query [T,Hq,D] and caches [NB,BS,Hkv,D], got "
            f"{tuple(query.shape)}, {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    T, Hq, D = query.shape
    num_blocks, block_size, heads, cache_dim = k_cache.shape
    device, dtype, n = query.device, query.dtype, md.num_seqs
    if cache_dim != D:
        raise ValueError(f"head_dim mismatch: query {D}, cache {cache_dim}")
    if not query.is_cuda or k_cache.device != device or v_cache.device != device:
        raise ValueError(f"{what} needs GPU tensors on one device (the HIP path has no CPU fallback)")
    if dtype not in _lib.DTYPE_CODES or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise TypeError(f"{what} takes float32, float16 or bfloat16 alike, got {dtype}, {k_cache.dtype}, {v_cache.dtype}")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous [num_blocks, block_size, num_kv_heads, head_dim]")
    if md.num_tokens != T:
        raise ValueError(f"metadata has {md.num_tokens} tokens, query has {T}")
    if heads == 0 or Hq % heads:
        raise ValueError(f"{Hq} query heads over {heads} KV heads")
    if md.max_query_len > MAX_TREE_ROWS:
        raise ValueError(f"a sequence of a tree has at most {MAX_TREE_ROWS} rows, got max_query_len {md.max_query_len}")
    if md.tree_mask is None:
        raise ValueError(f"{what} needs md.tree_mask")
    x, _ = _integers({"tree_mask": (md.tree_mask, T)}, device)
    mask = x["tree_mask"]
    if mask.dtype is not torch.int64:
        raise TypeError(f"tree_mask must be int64, got {mask.dtype}")
    q = query if query.is_contiguous() else query.contiguous()
    if T == 0 or n == 0:
        return torch.zeros_like(q)
    bt = _index(md.block_tables, "block_tables", device)
    if bt.dim() != 2 or bt.shape[0] < n:
        raise ValueError(f"block_tables must be [num_seqs, max_blocks], got {tuple(bt.shape)}")
    width = bt.shape[1]
    if width * block_size < md.max_seq_len:
        raise ValueError(f"block_tables has {width} columns but max_seq_len={md.max_seq_len} needs "
                         f"{-(-md.max_seq_len // block_size)}")
    if width == 0:
        return torch.zeros_like(q)
    if bt.stride(1) != 1 or bt.stride(0) < width:
        bt = bt.contiguous()
    sl = _index(md.seq_lens, "seq_lens", device)
    if sl.dim() != 1 or sl.shape[0] < n:
        raise ValueError(f"seq_lens must hold at least {n} entries, got {tuple(sl.shape)}")
    sl = sl.contiguous()
    qsl_ptr, qsl64 = None, 0
    if md.query_start_loc is None:
        if T != n:
            raise ValueError("without query_start_loc there is one row per sequence")
        out = torch.empty_like(q)
    else:
        qsl = _index(md.query_start_loc, "query_start_loc", device)
        if qsl.dim() != 1 or qsl.shape[0] < n + 1:
            raise ValueError(f"query_start_loc must hold at least {n + 1} entries, got {tuple(qsl.shape)}")
        qsl = qsl.contiguous()
        qsl_ptr, qsl64 = qsl.data_ptr(), qsl.dtype is torch.int64
        # Rows behind the last sequence are not written: zero unless the host's
        # offsets show that there are none, which they cannot for the replays of a
        # capture.
        host = md.query_start_loc_cpu
        full = (host is not None and len(host) > n and host[0] == 0 and host[n] == T
                and not torch.cuda.is_current_stream_capturing())
        out = torch.empty_like(q) if full else torch.zeros_like(q)
    lib = _lib.load()
    code = _lib.DTYPE_CODES[dtype]
    nbytes = lib.ns_paged_attention_tree_workspace_size(n, Hq, heads, D, block_size, md.max_query_len, T, code)
    # The partial results live in a tensor of this call's.
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    counters = _arrivals(device) if nbytes else None
    _lib.launch(device, what, lib.ns_paged_attention_tree,
                out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                bt.data_ptr(), bt.stride(0), width, bt.dtype is torch.int64, sl.data_ptr(), sl.dtype is torch.int64,
                qsl_ptr, qsl64, mask.data_ptr(), n, T, md.max_query_len, md.max_seq_len, Hq, heads, D, block_size,
                num_blocks, float(scale), code, _pointer(counters), _pointer(ws), nbytes)
    return out


def _index(t: torch.Tensor, name: str, device: torch.device) -> torch.Tensor:
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t if t.dtype is torch.int64 or t.dtype is torch.int32 else t.to(torch.int64)


def commit_drafts(chosen: torch.Tensor, input_ids: torch.Tensor, parents: torch.Tensor,
                  query_start_loc: torch.Tensor, slot_mapping: torch.Tensor, k_caches: list[torch.Tensor],
                  v_caches: list[torch.Tensor], max_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """What of a step's drafts holds: (counts [B], tokens [B, max_rows]), int64.

    chosen [T] is the token that the model takes after every row (argmax_rows or
    sample_rows of its logits), input_ids [T] what the row was fed, parents [T] as
    in step_inputs.  From row 0 of a request the walk goes on to the first child
    that was fed the current row's choice; its rows' choices are the request's next
    tokens (counts of them, then -1), and the rows' K and V move in every cache
    ([num_blocks, block_size, kv_heads, head_dim], one shape and dtype) from their
    slots to those of the request's first rows, where the tokens belong.  The slots
    of a request's rows must differ; slots outside the cache are left alone.
    max_rows (at most 64): the most rows of a request; later ones take no part."""
    what = "commit_drafts"
    device = chosen.device
    if not chosen.is_cuda:
        raise ValueError(f"{what} needs GPU tensors (the HIP path has no CPU fallback)")
    if not 0 <= max_rows <= MAX_TREE_ROWS:
        raise ValueError(f"max_rows must be between 0 and {MAX_TREE_ROWS}, got {max_rows}")
    T = chosen.shape[0] if chosen.dim() else 0
    x, wide = _integers({"chosen": (chosen, T), "input_ids": (input_ids, T), "parents": (parents, T)}, device)
    one, _ = _integers({"slot_mapping": (slot_mapping, T)}, device)
    slots = one["slot_mapping"]
    B = query_start_loc.shape[0] - 1 if query_start_loc.dim() else -1
    if B < 0:
        raise ValueError(f"query_start_loc must be [requests + 1], got {tuple(query_start_loc.shape)}")
    one, _ = _integers({"query_start_loc": (query_start_loc, B + 1)}, device)
    qsl = one["query_start_loc"]
    caches = [*k_caches, *v_caches]
    num_slots = row_bytes = 0
    if caches:
        first = caches[0]
        shape, dtype = first.shape, first.dtype
        if len(shape) != 4:
            raise ValueError(f"caches must be [num_blocks, block_size, kv_heads, head_dim], got {tuple(shape)}")
        for c in caches:
            if c.shape != shape or c.dtype is not dtype or c.device != device or not c.is_contiguous():
                raise ValueError(f"caches must be contiguous tensors of one shape and dtype on {device}, got "
                                 f"{c.dtype} {tuple(c.shape)} on {c.device} beside {dtype} {tuple(shape)}")
        num_slots, row_bytes = shape[0] * shape[1], shape[2] * shape[3] * first.element_size()
    out = torch.empty(B * (1 + max_rows), dtype=torch.int64, device=device)
    counts, tokens = out[:B], out[B:].view(B, max_rows)
    pointers = (ctypes.c_void_p * len(caches))(*[c.data_ptr() for c in caches]) if num_slots and row_bytes else None
    _lib.launch(device, what, _lib.load().ns_commit_drafts,
                counts.data_ptr(), tokens.data_ptr(), _pointer(x["chosen"]), _pointer(x["input_ids"]),
                _pointer(x["parents"]), wide, qsl.data_ptr(), qsl.dtype is torch.int64, slots.data_ptr(),
                slots.dtype is torch.int64, B, T, max_rows, pointers, 0 if pointers is None else len(caches),
                num_slots, row_bytes)
    return counts, tokens
