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
    BlockTables            the tables that step_inputs reads and extends

Each runs on the current stream and reads the device's lengths, so a captured graph
serves other lengths, trees and choices on every replay.  Each is one launch, but
paged_attention_tree takes one per 512 sequences, after a fill of the output where
rows may lie behind the last sequence (with query_start_loc in a capture: always) and,
in a capture, one of its arrival counters; commit_drafts takes one per 128 caches.
"""

from __future__ import annotations

import array
from dataclasses import dataclass
from functools import lru_cache
from operator import attrgetter

import torch

from . import _lib
from .attention import AttentionMetadata

_SIZE, _DEVICE, _CONTIGUOUS, _ADDRESS = (torch.Tensor.size, torch.Tensor.get_device, torch.Tensor.is_contiguous,
                                         torch.Tensor.data_ptr)
_DTYPE = attrgetter("dtype")

MAX_TREE_ROWS = 64  # rows of a request that a 64-bit mask can name


# These wrappers run in every step (paged_attention_tree in every layer) and hold a
# launch back by a few microseconds each: every tensor attribute is read once, and
# devices are compared by their index.  None of the ops is differentiable; what they
# return has no history.


@dataclass
class StepInputs:
    """A step's addresses on the device, as AttentionMetadata takes them (int64;
    block_tables in the tables' dtype)."""

    query_start_loc: torch.Tensor         # [B + 1]
    seq_lens: torch.Tensor                # [B]
    positions: torch.Tensor               # [T]
    slot_mapping: torch.Tensor            # [T]
    block_tables: torch.Tensor            # [B, max_blocks]
    tree_mask: torch.Tensor | None        # [T], with parents


def _vector(t: torch.Tensor, name: str, n: int, index: int) -> torch.Tensor:
    """t, contiguous, if it holds n int32 or int64 entries on GPU `index`."""
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if t.shape != (n,):
        raise ValueError(f"{name} must hold {n} entries, got {tuple(t.shape)}")
    if t.dtype is not torch.int64 and t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    return t if t.is_contiguous() else t.contiguous()


def _alike(tensors: list) -> tuple[list, bool]:
    """The tensors (or None) of one integer dtype, and whether that is int64."""
    kinds = {t.dtype for t in tensors if t is not None}
    if len(kinds) > 1:
        tensors = [t if t is None else t.to(torch.int64) for t in tensors]
    return tensors, torch.int64 in kinds


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
    if (new_blocks is None) != (new_start is None) or (new_blocks is None) != (held is None):
        raise ValueError("new_blocks, new_start and held belong together")
    index = tables.get_device()
    B = rows.shape[0] if rows.dim() else 0
    N = 0 if new_blocks is None else new_blocks.numel()
    vectors = [_vector(rows, "rows", B, index), _vector(computed, "computed", B, index),
               _vector(query_lens, "query_lens", B, index),
               None if new_blocks is None else _vector(new_blocks, "new_blocks", N, index),
               None if new_start is None else _vector(new_start, "new_start", B + 1, index),
               None if held is None else _vector(held, "held", B, index),
               None if parents is None else _vector(parents, "parents", num_tokens, index)]
    vectors, wide = _alike(vectors)
    device = tables.device
    # One allocation for every int64 output (no two overlap, and none has a history:
    # the split that keeps no record of the parts being views).
    T = num_tokens
    sizes = [B + 1, B, T, T] if parents is None else [B + 1, B, T, T, T]
    flat = torch.empty(sum(sizes), dtype=torch.int64, device=device)
    qsl, lens, positions, slots, *mask = torch.unsafe_split_with_sizes(flat, sizes)
    packed = torch.empty((B, max_blocks), dtype=tables.dtype, device=device)
    at = flat.data_ptr()
    pointers = [None if t is None else t.data_ptr() for t in vectors]
    _lib.launch(device, what, _lib.load().ns_step_inputs,
                tables.data_ptr(), R, W, max(tables.stride(0), W), tables.dtype is torch.int64,
                *pointers[:6], N, pointers[6], wide, B, T, block_size, max_blocks,
                at, at + 8 * (B + 1), at + 8 * (2 * B + 1), at + 8 * (2 * B + 1 + T), packed.data_ptr(),
                at + 8 * (2 * B + 1 + 2 * T) if mask else None)
    return StepInputs(qsl, lens, positions, slots, packed, mask[0] if mask else None)


class BlockTables:
    """The requests' block ids on the device, one row each, for step_inputs.

    `place` names a batch's rows and what the step has to append to them: a
    request's table grows in place (BlockSpaceManager.allocate), so a row that
    holds the same list needs only the blocks added since.  A request that has no
    row gets a free one, or that of a request outside the batch."""

    def __init__(self, width: int, device, rows: int = 64) -> None:
        self.width = width
        self.device = device
        self.tensor = torch.zeros(rows, width, dtype=torch.int64, device=device)
        # Per request: its row, the list written there (held, so that its identity is
        # its own) and how many of its entries.
        self._rows: dict[int, tuple[int, list[int], int]] = {}
        self._free = list(range(rows - 1, -1, -1))

    def forget(self, seq) -> None:
        held = self._rows.pop(seq.seq_id, None)
        if held is not None:
            self._free.append(held[0])

    def trimmed(self, seq) -> None:
        """`seq` has a shorter table of the same blocks (BlockSpaceManager.trim)."""
        held = self._rows.get(seq.seq_id)
        if held is not None:
            self._rows[seq.seq_id] = (held[0], seq.block_table, min(held[2], len(seq.block_table)))

    def place(self, seqs) -> tuple[list[int], list[int], list[int], list[int]]:
        """(rows, held, new_start, new_blocks) of the batch, as step_inputs takes them.  Counts on
        that call: `forget` the requests where it fails."""
        missing = sum(s.seq_id not in self._rows for s in seqs)
        if missing > len(self._free):
            here = {s.seq_id for s in seqs}
            for i in [i for i in self._rows if i not in here][:missing - len(self._free)]:
                self._free.append(self._rows.pop(i)[0])
        if missing > len(self._free):
            have = self.tensor.shape[0]
            more = max(have, missing)
            self.tensor = torch.cat((self.tensor, torch.zeros(more, self.width, dtype=torch.int64, device=self.device)))
            self._free += range(have + more - 1, have - 1, -1)
        rows, held, start, blocks = [], [], [0], []
        for s in seqs:
            table = s.block_table
            row, old, n = self._rows.get(s.seq_id) or (self._free.pop(), None, 0)
            if old is not table:
                n = 0
            rows.append(row)
            held.append(n)
            blocks += table[n:]
            start.append(len(blocks))
            self._rows[s.seq_id] = (row, table, len(table))
        return rows, held, start, blocks


# Arrival counters of the key ranges, zero before and after every call, one
# buffer per (device, stream): calls on one stream follow each other.  A call
# that is recorded into a graph gets its own, cleared by the graph, so that graphs
# share none whichever streams they are replayed on.
_counters: dict[tuple[int, int], torch.Tensor] = {}


def _arrivals(device: torch.device, capturing: bool) -> torch.Tensor:
    index = device.index
    if not capturing:
        c = _counters.get((index, torch._C._cuda_getCurrentRawStream(index)))
        if c is not None:
            return c
    with torch.cuda.device(index):  # as many as that device, not the current one, has workgroups
        n = _lib.load().ns_paged_attention_tree_counters()
    c = torch.zeros(n, dtype=torch.int32, device=device)
    if not capturing:
        _counters[index, torch._C._cuda_getCurrentRawStream(index)] = c
    return c


def _capturing(index: int) -> bool:
    """Whether the current stream of GPU `index`, which a call on its tensors takes, is recording a graph."""
    if index == torch._C._cuda_getDevice():
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(index):
        return torch._C._cuda_isCurrentStreamCapturing()


@lru_cache(maxsize=4096)
def _workspace_bytes(index: int, *sizes: int) -> int:
    """ns_paged_attention_tree_workspace_size, a function of sizes alone, which the layers of a step share."""
    with torch.cuda.device(index):
        return _lib.load().ns_paged_attention_tree_workspace_size(*sizes)


def paged_attention_tree(query: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                         md: AttentionMetadata, scale: float) -> torch.Tensor:
    """Paged attention for trees of drafted tokens: attn_fn's contract
    (attention.paged_attention_hip) with md.tree_mask.  Row j of a sequence with
    context length L and q <= 64 rows sees keys 0 .. L - q - 1, and key L - q + i
    where bit i of its mask is set.  Returns [num_tokens, num_heads, head_dim],
    with zeros for rows without keys, rows whose scores are all -inf (as in
    paged_attention_hip) and rows behind the last sequence.

    float32, float16 and bfloat16, head sizes up to 256.  The device's lengths,
    offsets, masks and tables decide what is computed; of the host's only
    max_query_len, max_seq_len and query_start_loc_cpu are read, and shape the
    launch."""
    what = "paged_attention_tree"
    shape, cache = query.shape, k_cache.shape
    if len(shape) != 3 or len(cache) != 4 or v_cache.shape != cache:
        raise ValueError(f"expected query [T,Hq,D] and caches [NB,BS,Hkv,D], got {tuple(shape)}, {tuple(cache)}, "
                         f"{tuple(v_cache.shape)}")
    T, Hq, D = shape
    num_blocks, block_size, heads, cache_dim = cache
    index, dtype, n, longest = query.get_device(), query.dtype, md.num_seqs, md.max_seq_len
    if cache_dim != D:
        raise ValueError(f"head_dim mismatch: query {D}, cache {cache_dim}")
    if index < 0 or k_cache.get_device() != index or v_cache.get_device() != index:
        raise ValueError(f"{what} needs GPU tensors on one device (the HIP path has no CPU fallback)")
    code = _lib.DTYPE_CODES.get(dtype)
    if code is None or k_cache.dtype is not dtype or v_cache.dtype is not dtype:
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
    mask = _vector(md.tree_mask, "tree_mask", T, index)
    if mask.dtype is not torch.int64:
        raise TypeError(f"tree_mask must be int64, got {mask.dtype}")
    q = query if query.is_contiguous() else query.contiguous()
    if T == 0 or n == 0:
        return torch.zeros_like(q)
    bt = _index(md.block_tables, "block_tables", index)
    if bt.dim() != 2 or bt.shape[0] < n:
        raise ValueError(f"block_tables must be [num_seqs, max_blocks], got {tuple(bt.shape)}")
    width = bt.shape[1]
    if width * block_size < longest:
        raise ValueError(f"block_tables has {width} columns but max_seq_len={longest} needs {-(-longest // block_size)}")
    if width == 0:
        return torch.zeros_like(q)
    stride = bt.stride()
    if stride[1] != 1 or stride[0] < width:
        bt = bt.contiguous()
        stride = bt.stride()
    sl = _prefix(md.seq_lens, "seq_lens", n, index)
    capturing = _capturing(index)
    qsl_ptr, qsl64 = None, 0
    if md.query_start_loc is None:
        if T != n:
            raise ValueError("without query_start_loc there is one row per sequence")
        full = True
    else:
        qsl = _prefix(md.query_start_loc, "query_start_loc", n + 1, index)
        qsl_ptr, qsl64 = qsl.data_ptr(), qsl.dtype is torch.int64
        # Rows behind the last sequence are not written: zero unless the host's
        # offsets show that there are none, which they cannot for the replays of a
        # capture.
        host = md.query_start_loc_cpu
        full = host is not None and len(host) > n and host[0] == 0 and host[n] == T and not capturing
    out = torch.empty_like(q) if full else torch.zeros_like(q)
    nbytes = _workspace_bytes(index, n, Hq, heads, D, block_size, md.max_query_len, T, code)
    ws = counters = None
    device = q.device
    if nbytes:
        # The partial results live in a tensor of this call's.
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        counters = _arrivals(device, capturing)
    _lib.launch(device, what, _lib.load().ns_paged_attention_tree,
                out.data_ptr(), q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                bt.data_ptr(), stride[0], width, bt.dtype is torch.int64, sl.data_ptr(), sl.dtype is torch.int64,
                qsl_ptr, qsl64, mask.data_ptr(), n, T, md.max_query_len, longest, Hq, heads, D, block_size,
                num_blocks, float(scale), code, _pointer(counters), _pointer(ws), nbytes)
    return out


def _index(t: torch.Tensor, name: str, index: int) -> torch.Tensor:
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    return t if t.dtype is torch.int64 or t.dtype is torch.int32 else t.to(torch.int64)


def _prefix(t: torch.Tensor, name: str, least: int, index: int) -> torch.Tensor:
    t = _index(t, name, index)
    if t.dim() != 1 or t.shape[0] < least:
        raise ValueError(f"{name} must hold at least {least} entries, got {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


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
    slots to those of the request's first rows, where the tokens belong.  No cache may
    be listed twice.  The slots of a request's rows must differ, and one that a row
    moves to must be no other request's; slots outside the cache are left alone.
    max_rows (at most 64): the most rows of a request; later ones take no part."""
    what = "commit_drafts"
    index = chosen.get_device()
    if index < 0:
        raise ValueError(f"{what} needs GPU tensors (the HIP path has no CPU fallback)")
    if not 0 <= max_rows <= MAX_TREE_ROWS:
        raise ValueError(f"max_rows must be between 0 and {MAX_TREE_ROWS}, got {max_rows}")
    T = chosen.shape[0] if chosen.dim() else 0
    B = query_start_loc.shape[0] - 1 if query_start_loc.dim() else -1
    if B < 0:
        raise ValueError(f"query_start_loc must be [requests + 1], got {tuple(query_start_loc.shape)}")
    rows, wide = _alike([_vector(chosen, "chosen", T, index), _vector(input_ids, "input_ids", T, index),
                         _vector(parents, "parents", T, index)])
    slots = _vector(slot_mapping, "slot_mapping", T, index)
    qsl = _vector(query_start_loc, "query_start_loc", B + 1, index)
    caches = [*k_caches, *v_caches]
    num_slots = row_bytes = 0
    if caches:
        first = caches[0]
        shape, dtype = first.shape, first.dtype
        if len(shape) != 4:
            raise ValueError(f"caches must be [num_blocks, block_size, kv_heads, head_dim], got {tuple(shape)}")
        # Some tens of tensors in every call: checked without a Python loop.
        if ([*map(_SIZE, caches)].count(shape) != len(caches) or {*map(_DTYPE, caches)} != {dtype}
                or {*map(_DEVICE, caches)} != {index} or not all(map(_CONTIGUOUS, caches))):
            raise ValueError(f"caches must be contiguous tensors of one shape and dtype on cuda:{index}, got "
                             f"{sorted({(str(c.dtype), tuple(c.shape), str(c.device)) for c in caches})}")
        num_slots, row_bytes = shape[0] * shape[1], shape[2] * shape[3] * first.element_size()
    device = chosen.device
    counts = torch.empty(B, dtype=torch.int64, device=device)
    tokens = torch.empty((B, max_rows), dtype=torch.int64, device=device)
    held = len(caches) if num_slots and row_bytes else 0
    pointers = array.array("Q", map(_ADDRESS, caches)) if held else None
    try:
        _lib.launch(device, what, _lib.load().ns_commit_drafts,
                    counts.data_ptr(), tokens.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), rows[2].data_ptr(), wide,
                    qsl.data_ptr(), qsl.dtype is torch.int64, slots.data_ptr(), slots.dtype is torch.int64, B, T, max_rows,
                    pointers.buffer_info()[0] if held else None, held, num_slots, row_bytes)
    except RuntimeError:
        # The library refuses caches that overlap.
        if held and len({*pointers}) != held:
            raise ValueError("a cache is listed twice") from None
        raise
    return counts, tokens
