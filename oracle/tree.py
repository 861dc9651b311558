"""A decode step over trees of drafted tokens, restated plainly on the CPU: its
addresses, its attention in float64 and the walk that ends it.

Citations: the addresses of a row are the reference's (nanoserve/model_runner.py:85-147,
block_manager.py:93-157), attention is the textbook formula over the keys that a row
sees.  The reference has neither trees nor drafts.
"""

from __future__ import annotations

import torch


def ancestors(parents: list[int]) -> list[int]:
    """The mask of every row of one request: its way to the root and itself."""
    masks: list[int] = []
    for j, p in enumerate(parents):
        if j >= 64:
            masks.append(0)
            continue
        masks.append((masks[p] if 0 <= p < j else 0) | (1 << j))
    return masks


def signed(mask: int) -> int:
    """64 bits as the int64 that holds them."""
    return mask - (1 << 64) if mask >= 1 << 63 else mask


def step_inputs_ref(tables: list[list[int]], rows, computed, query_lens, num_tokens, block_size, max_blocks,
                    new=None, held=None, parents=None):
    """(query_start_loc, seq_lens, positions, slots, packed tables, masks or None); tables grows in place.
    new[i], held[i]: request i's new blocks and the column of the first."""
    R, W = len(tables), len(tables[0]) if tables else 0
    for i, r in enumerate(rows):
        for k, b in enumerate(new[i] if new else ()):
            if 0 <= r < R and 0 <= held[i] and held[i] + k < W:
                tables[r][held[i] + k] = b
    qsl, lens, pos, slots, packed, masks = [0], [], [], [], [], []
    for i, r in enumerate(rows):
        c, q = max(0, computed[i]), max(0, query_lens[i])
        block = lambda col: tables[r][col] if 0 <= r < R and col < W else -1  # noqa: E731, B023
        par = None if parents is None else parents[qsl[-1]:qsl[-1] + q]
        seen = ancestors(par) if par is not None else None
        for j in range(q):
            b = block((c + j) // block_size)
            slots.append(-1 if b < 0 else b * block_size + (c + j) % block_size)
            in_tree = seen is not None and j < 64
            pos.append(c + (bin(seen[j]).count("1") - 1 if in_tree else j))
            if seen is not None:
                masks.append(signed(seen[j]))
        lens.append(c + q)
        qsl.append(qsl[-1] + q)
        used = -(-(c + q) // block_size)
        packed.append([block(k) if k < used else 0 for k in range(max_blocks)])
    rest = num_tokens - len(slots)
    return (qsl, lens, pos + [0] * rest, slots + [-1] * rest, packed, None if parents is None else masks + [0] * rest)


def tree_attention_ref(query, k_cache, v_cache, starts, lens, tables, masks, scale):
    """([T, Hq, D] float64 outputs, the same over |V|: what errors of the weights are relative to).

    starts, lens, masks: Python ints; tables: lists of block ids."""
    T, hq, d = query.shape
    hkv, bs = k_cache.shape[2], k_cache.shape[1]
    group = hq // hkv
    out, mag = torch.zeros(2, T, hq, d, dtype=torch.float64).unbind()
    for i, L in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        if b <= a:
            continue
        blocks = tables[i][:-(-L // bs)]
        k, v = (c[blocks].double().reshape(-1, hkv, d)[:L] for c in (k_cache, v_cache))
        base = L - (b - a)
        for t in range(a, b):
            keys = [j for j in range(L) if j < base or (j - base < 64 and (masks[t] >> (j - base)) & 1)]
            if not keys:
                continue
            kk, vv = k[keys], v[keys]
            for h in range(hkv):
                q = query[t, h * group:(h + 1) * group].double()
                p = (q @ kk[:, h].T * scale).softmax(-1)
                out[t, h * group:(h + 1) * group] = p @ vv[:, h]
                mag[t, h * group:(h + 1) * group] = p @ vv[:, h].abs()
    return out, mag


def commit_ref(chosen, ids, parents, starts, slots, max_rows, flat_caches, num_slots):
    """(counts, tokens): the walk of every request, and its rows moved in flat_caches ([slots, ...] tensors)."""
    counts, tokens = [], []
    for a, b in zip(starts, starts[1:]):
        q = min(max(b - a, 0), max_rows)
        path = [0] if q else []
        while path:
            at = path[-1]
            nxt = [j for j in range(at + 1, q) if parents[a + j] == at and ids[a + j] == chosen[a + at]]
            if not nxt:
                break
            path.append(nxt[0])
        counts.append(len(path))
        tokens.append([chosen[a + j] for j in path] + [-1] * (max_rows - len(path)))
        moves = [(slots[a + j], slots[a + d]) for d, j in enumerate(path)]
        moves = [(f, t) for f, t in moves if f != t and 0 <= f < num_slots and 0 <= t < num_slots]
        for c in flat_caches:
            got = [c[f].clone() for f, _ in moves]
            for (_, t), x in zip(moves, got):
                c[t] = x
    return counts, tokens
