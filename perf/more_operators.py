"""Timed cases of a decode step that verifies drafted tokens: the step's addresses,
attention for trees of drafted tokens over the paged cache, and the end of the
step, which keeps the accepted tokens.

Three kinds of case:

  inputs   a step's query offsets, lengths, positions, slots, packed block tables
           and (with drafted trees) every row's ancestors, from the requests'
           lengths, new blocks and a table of their blocks that stays on the GPU.
  attend   paged attention of a tree of rows per sequence: all keys before the
           rows, and of the rows themselves those on the way to the tree's root.
  commit   the walk along the tokens that the model chose, and K and V of the
           accepted rows moved to the places of the tokens they have become.

A sequence's rows are its last token (row 0) and the drafted ones, at most 64; a
row's parent is an earlier row of the sequence, or -1.  Bit i of a row's mask says
that it sees row i.  Row j's K and V lie at cache position (context before the
step) + j, whatever its depth.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# (query heads, KV heads, head size): the 0.5B model's, the larger-GQA
# benchmark's, and group sizes 1, 8 and 16 that the attention tests run.
HEADS = ((14, 2, 64), (28, 4, 128), (16, 2, 128), (8, 8, 64), (32, 2, 64))


def listed():
    return [
        # One interactive request with a bushy draft.
        _step("inputs", "inputs_one", batch=1, rows=24, median=700, width=256),
        # A decode batch at serving load, a short draft each.
        _step("inputs", "inputs_step", batch=32, rows=8, median=1024, sigma=0.8, width=512),
        # A prompt step at a large token budget: no drafts, many new blocks.
        _step("inputs", "inputs_prompts", batch=11, rows=1009, median=512, sigma=1.0, width=512, tree=False),
        # Every request of a large deployment: tables of 32K contexts.
        _step("inputs", "inputs_fleet", batch=1024, rows=16, median=4096, sigma=1.0, width=2048, index="int32"),
        # The interactive request's attention.
        _attend("tree_one", batch=1, rows=24, median=750),
        # The headline benchmark's 32 contexts around 1K, eight rows each.
        _attend("tree_serving", batch=32, rows=8, median=1024, sigma=0.8),
        # Drafts of different lengths, some requests without one, larger heads.
        _attend("tree_ragged", batch=17, rows=21, ragged=True, median=900, sigma=0.6, heads=(28, 4, 128),
                dtype="bf16", block=32, index="int32"),
        # Long contexts of the larger model: the stream of the cache.
        _attend("tree_long", batch=64, rows=12, median=4096, sigma=1.0, heads=(28, 4, 128), dtype="bf16"),
        # Few requests with the widest drafts.
        _attend("tree_wide", batch=8, rows=64, median=4000, sigma=0.4, heads=(28, 4, 128), dtype="bf16"),
        # The interactive request's accepted rows, the 0.5B model's 24 layers.
        _commit("commit_one", batch=1, rows=24, shape=20),
        # The serving batch's.
        _commit("commit_step", batch=32, rows=8),
        # Many requests with wide drafts, a larger model.
        _commit("commit_wide", batch=128, rows=32, layers=28, heads=(28, 4, 128), dtype="bf16"),
    ]


def _step(kind, name, batch, rows, median, sigma=0.0, width=0, tree=True, ragged=False, index="int64", block=16,
          shape=1, **more):
    c = {"kind": kind, "batch": batch, "rows": rows, "ragged": ragged, "median": median, "sigma": sigma,
         "width": width, "tree": tree, "index": index, "block": block, "shape": shape, **more}
    return c if name is None else {"name": name, **c}


def _attend(name, heads=(14, 2, 64), dtype="fp16", **more):
    return _step("attend", name, hq=heads[0], hkv=heads[1], dim=heads[2], dtype=dtype, **more)


def _commit(name, layers=24, heads=(14, 2, 64), dtype="fp16", **more):
    return _step("commit", name, layers=layers, hkv=heads[1], dim=heads[2], dtype=dtype, median=100, sigma=0.5, **more)


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["inputs", "inputs", "attend", "attend", "attend", "attend", "commit", "commit"])
    more = {"shape": rng.randrange(1 << 20), "block": rng.choice([16, 16, 32]), "index": rng.choice(["int32", "int64"]),
            "ragged": rng.random() < 0.5}
    heads = rng.choice(HEADS)
    if kind == "inputs":
        tree = rng.random() < 0.6
        batch = _log_int(rng, 1, 1024 if tree else 64)
        rows = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, 8192 // batch)
        while batch * rows > 16384:
            rows = max(1, rows // 2)
        width = _log_int(rng, 64, 2048)
        fits = width * more["block"] - rows
        return _step("inputs", None, batch=batch, rows=rows, median=_log_int(rng, 1, min(8192, max(1, fits // 4))),
                     sigma=rng.choice([0.0, 0.5, 1.0]), width=width, tree=tree, **more)
    more["dtype"] = rng.choice(["fp16", "bf16"])
    if kind == "commit":
        batch, layers = _log_int(rng, 1, 128), rng.randint(1, 28)
        return _commit(None, batch=batch, rows=_log_int(rng, 2, 48), layers=layers, heads=heads, **more)
    batch, rows = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
    # at most the padded cache and scores of the largest listed cases
    longest = min(64 * 32768 * 4 * 128 // (batch * heads[1] * heads[2]), 64 * 28 * 12 * 32768 // (batch * heads[0] * rows))
    return _attend(None, heads=heads, batch=batch, rows=rows, median=_log_int(rng, 1, max(2, min(6000, longest // 8))),
                   sigma=rng.choice([0.0, 0.5, 1.0]), **more)


# ---- the step's requests: what the case alone decides -----------------------


def _lengths(case):
    """(tokens computed before the step, rows) of every request."""
    rng = np.random.default_rng(case["shape"])
    n, m = case["batch"], case["median"]
    most = 8 * m if not case["width"] else min(8 * m, case["width"] * case["block"] - case["rows"])
    base = np.clip(rng.lognormal(np.log(m), case["sigma"], n).astype(int), 0, max(0, most))
    rows = rng.integers(1, case["rows"], size=n, endpoint=True) if case["ragged"] else np.full(n, case["rows"])
    return base.tolist(), rows.tolist()


def _parents(case, rows):
    """Every row's parent: trees that are deeper than they are wide."""
    rng = np.random.default_rng(case["shape"] + 1)
    return [[-1] + [int(rng.integers(max(0, j - 4), j)) for j in range(1, n)] for n in rows]


def _path(case, parents):
    """The rows that a walk from row 0 takes: on with 4 in 5, to any child."""
    rng = np.random.default_rng(case["shape"] + 2)
    paths = []
    for par in parents:
        path = [0]
        while rng.random() < 0.8:
            children = [j for j, p in enumerate(par) if p == path[-1]]
            if not children:
                break
            path.append(children[int(rng.integers(len(children)))])
        paths.append(path)
    return paths


def _masks(parents):
    out = []
    for par in parents:
        seen = []
        for j, p in enumerate(par):
            seen.append((seen[p] if p >= 0 else 0) | (1 << j))
        out += seen
    return out


# ---- inputs -----------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"inputs": _prepare_inputs, "attend": _prepare_attend, "commit": _prepare_commit}[case["kind"]](case, seed, g)


def _ints(values, dtype=torch.int64):
    v = np.asarray(values, dtype=np.uint64 if dtype is None else np.int64)
    return torch.from_numpy(v.view(np.int64)).to(DEV, dtype or torch.int64)


def _flat(lists):
    return [v for x in lists for v in x]


def _prepare_inputs(case, seed, g):
    base, rows = _lengths(case)
    n, bs, width = case["batch"], case["block"], case["width"]
    it = torch.int32 if case["index"] == "int32" else torch.int64
    # A request's blocks up to its computed tokens are in the table, the others come with the step.
    held = [-(-b // bs) for b in base]
    new = [max(0, -(-(b + q) // bs) - h) for b, q, h in zip(base, rows, held)]
    pool = n + 3
    tables = torch.randint(0, 1 << 20, (pool, width), generator=g, device=DEV).to(it)
    place = torch.randperm(pool, generator=g, device=DEV)[:n]
    s = {"case": case, "tables": tables, "rows": place, "computed": _ints(base), "query_lens": _ints(rows),
         "held": _ints(held), "new_start": _ints([0, *np.cumsum(new).tolist()]),
         "new_blocks": torch.randint(0, 1 << 20, (sum(new),), generator=g, device=DEV),
         "num_tokens": sum(rows), "max_blocks": max(1, max(-(-(b + q) // bs) for b, q in zip(base, rows)))}
    s["parents"] = _ints(_flat(_parents(case, rows))) if case["tree"] else None
    return s


def _prepare_attend(case, seed, g):
    base, rows = _lengths(case)
    hq, hkv, d, bs = case["hq"], case["hkv"], case["dim"], case["block"]
    dt = DTYPES[case["dtype"]]
    lens = [b + q for b, q in zip(base, rows)]
    need = [-(-n // bs) for n in lens]
    pool = math.ceil(1.25 * sum(need))
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))
    it = torch.int32 if case["index"] == "int32" else torch.int64
    tables = torch.zeros(len(lens), max(need), dtype=it)
    cur = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[cur:cur + n].to(it)
        cur += n
    kc, vc = (torch.empty(pool, bs, hkv, d, dtype=dt, device=DEV).normal_(generator=g) for _ in range(2))
    query = torch.randn(sum(rows), hq, d, generator=g, device=DEV).to(dt)
    starts = [0, *np.cumsum(rows).tolist()]
    return {"case": case, "query": query, "kc": kc, "vc": vc, "tables": tables.to(DEV), "lens": _ints(lens, it),
            "starts": _ints(starts, it), "mask": _ints(_masks(_parents(case, rows)), None),
            "lens_cpu": lens, "rows_cpu": rows, "starts_cpu": starts, "scale": d ** -0.5,
            "slots": torch.zeros(sum(rows), dtype=torch.int64, device=DEV)}


def _prepare_commit(case, seed, g):
    base, rows = _lengths(case)
    n, hkv, d, bs = case["batch"], case["hkv"], case["dim"], case["block"]
    parents = _parents(case, rows)
    T = sum(rows)
    # Only the blocks that the step's rows lie in: the others are not touched.
    first = [b % bs for b in base]
    need = [-(-(f + q) // bs) for f, q in zip(first, rows)]
    blocks = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).tolist()
    slots, cur = [], 0
    for f, q, k in zip(first, rows, need):
        slots += [blocks[cur + (f + j) // bs] * bs + (f + j) % bs for j in range(q)]
        cur += k
    # Token ids at random; the model chooses a child's along the walk, and what nobody drafted at its end.
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, 150000, size=T)
    chosen = rng.integers(150000, 151936, size=T)
    at = 0
    for q, path in zip(rows, _path(case, parents)):
        for a, b in zip(path, path[1:]):
            chosen[at + a] = ids[at + b]
        at += q
    it = torch.int32 if case["index"] == "int32" else torch.int64
    cache = torch.empty(2, case["layers"], sum(need) + 2, bs, hkv, d, dtype=DTYPES[case["dtype"]],
                        device=DEV).normal_(generator=g)
    starts = [0, *np.cumsum(rows).tolist()]
    return {"case": case, "cache": cache, "k": list(cache[0].unbind()), "v": list(cache[1].unbind()),
            "slots": _ints(slots), "ids": _ints(ids), "chosen": _ints(chosen), "parents": _ints(_flat(parents)),
            "starts": _ints(starts, it), "rows_cpu": rows, "max_rows": max(rows)}


# ---- one pass ---------------------------------------------------------------


def run(state):
    return {"inputs": _run_inputs, "attend": _run_attend, "commit": _run_commit}[state["case"]["kind"]](state)


def _padded(starts, rows):
    """(row j of request i in the batch [B, rows], whether there is one)."""
    j = torch.arange(rows, device=DEV)
    return starts[:-1, None] + j, j < (starts[1:] - starts[:-1])[:, None]


def _ancestors(parents):
    """[B, N] parents -> [B, N, N] truth values: row j's way to the root, itself included."""
    n = parents.shape[1]
    i = torch.arange(n, device=DEV)
    step = (parents[:, :, None] == i).float() + torch.eye(n, device=DEV)
    return torch.linalg.matrix_power(step, 64) > 0


def _run_inputs(s):
    case, tables = s["case"], s["tables"]
    bs, T = case["block"], s["num_tokens"]
    if own:
        from nanoserve_amd import step_inputs

        x = step_inputs(tables, s["rows"], s["computed"], s["query_lens"], T, bs, s["max_blocks"],
                        new_blocks=s["new_blocks"], new_start=s["new_start"], held=s["held"], parents=s["parents"])
        out = (x.query_start_loc, x.seq_lens, x.positions, x.slot_mapping, x.block_tables, tables)
        return out if s["parents"] is None else (*out, x.tree_mask)
    q = s["query_lens"]
    starts = torch.nn.functional.pad(q.cumsum(0), (1, 0))
    lens = s["computed"] + q
    k = torch.arange(s["new_blocks"].shape[0], device=DEV)
    i = torch.searchsorted(s["new_start"], k, right=True) - 1
    tables[s["rows"][i], s["held"][i] + k - s["new_start"][i]] = s["new_blocks"].to(tables.dtype)
    t = torch.arange(T, device=DEV)
    i = torch.searchsorted(starts, t, right=True) - 1
    at = s["computed"][i] + t - starts[i]
    slots = tables[s["rows"][i], at // bs].long() * bs + at % bs
    col = torch.arange(s["max_blocks"], device=DEV)
    packed = torch.where(col < ((lens + bs - 1) // bs)[:, None], tables[s["rows"]][:, :s["max_blocks"]], 0)
    if s["parents"] is None:
        return starts, lens, at, slots, packed, tables
    rows, there = _padded(starts, case["rows"])
    way = _ancestors(torch.where(there, s["parents"][rows.clamp(max=T - 1)], -1))
    mask = (way.long() << torch.arange(case["rows"], device=DEV)).sum(-1)[there]
    return starts, lens, s["computed"][i] + way.sum(-1)[there] - 1, slots, packed, tables, mask


def _run_attend(s):
    if own:
        from nanoserve_amd import AttentionMetadata, paged_attention_tree

        md = AttentionMetadata(
            slot_mapping=s["slots"], query_start_loc=s["starts"], seq_lens=s["lens"], block_tables=s["tables"],
            max_query_len=max(s["rows_cpu"]), max_seq_len=max(s["lens_cpu"]), num_seqs=len(s["lens_cpu"]),
            num_tokens=s["query"].shape[0], is_decode_only=max(s["rows_cpu"]) == 1, query_lens_cpu=s["rows_cpu"],
            seq_lens_cpu=s["lens_cpu"], query_start_loc_cpu=s["starts_cpu"], tree_mask=s["mask"])
        return paged_attention_tree(s["query"], s["kc"], s["vc"], md, s["scale"])
    q, dt = s["query"], s["query"].dtype
    T, hq, d = q.shape
    hkv, n, most = s["case"]["hkv"], len(s["lens_cpu"]), max(s["rows_cpu"])
    keys = s["tables"].shape[1] * s["case"]["block"]
    # Rows padded to the widest draft, keys to the longest table.
    starts, lens = s["starts"].long(), s["lens"].long()
    row, there = _padded(starts, most)
    row = row.clamp(max=T - 1)
    qp = q[row].float().view(n, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)

    def gathered(cache):
        return cache[s["tables"].long()].float().view(n, keys, hkv, d).transpose(1, 2)

    x = torch.matmul(qp, gathered(s["kc"]).transpose(-1, -2).contiguous()) * s["scale"]
    x = x.view(n, hkv, most, hq // hkv, keys)
    of = torch.arange(keys, device=DEV) - (lens - (starts[1:] - starts[:-1]))[:, None]  # the key's row of the tree
    bit = (s["mask"][row][:, :, None] >> of.clamp(0, 63)[:, None]) & 1
    seen = (of < 0)[:, None] | ((of < 64)[:, None] & (bit == 1) & (of < (starts[1:] - starts[:-1])[:, None])[:, None])
    x.masked_fill_(~seen[:, None, :, None], -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, keys), gathered(s["vc"]).contiguous()).view(n, hkv, most, hq // hkv, d) / total
    return o.permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)[there].to(dt)


def _run_commit(s):
    if own:
        from nanoserve_amd import commit_drafts

        counts, tokens = commit_drafts(s["chosen"], s["ids"], s["parents"], s["starts"], s["slots"], s["k"], s["v"],
                                       s["max_rows"])
        return counts, tokens, s["cache"]
    n, starts = s["max_rows"], s["starts"].long()
    row, there = _padded(starts, n)
    row = row.clamp(max=s["ids"].shape[0] - 1)
    ids, chosen = s["ids"][row], s["chosen"][row]
    par = torch.where(there, s["parents"][row], -1)
    # A row is taken up where its token is its parent's choice, and no earlier row has both.
    same = (par[:, :, None] == par[:, None]) & (ids[:, :, None] == ids[:, None])
    first = ~(same & torch.ones(n, n, dtype=torch.bool, device=DEV).tril(-1)).any(-1)
    taken = (par >= 0) & (ids == chosen.gather(1, par.clamp(min=0))) & first
    taken[:, 0] = True
    way = _ancestors(par)
    kept = way[:, :, 0] & there & (taken[:, None] | ~way).all(-1)
    counts = kept.sum(-1)
    rank = kept.cumsum(-1) - 1
    tokens = torch.full(row.shape, -1, dtype=torch.int64, device=DEV)
    i, j = kept.nonzero(as_tuple=True)
    tokens[i, rank[i, j]] = chosen[i, j]
    to, of = s["slots"][starts[i] + rank[i, j]], s["slots"][starts[i] + j]
    flat = s["cache"].flatten(0, 1).flatten(1, 2)
    flat[:, to] = flat[:, of]
    return counts, tokens, s["cache"]


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    base, rows = _lengths(case)
    T, n = sum(rows), len(rows)
    isz = 4 if case["index"] == "int32" else 8
    if case["kind"] == "inputs":
        bs = case["block"]
        blocks = sum(-(-(b + q) // bs) for b, q in zip(base, rows))
        new = sum(max(0, -(-(b + q) // bs) - -(-b // bs)) for b, q in zip(base, rows))
        width = max(1, max(-(-(b + q) // bs) for b, q in zip(base, rows)))
        return {"bytes": 8 * 6 * n + 16 * T + (16 * T if case["tree"] else 0) + isz * (blocks + n * width)
                + (8 + isz) * new, "flops": 0}
    if case["kind"] == "commit":
        moved = sum(j != d for p in _path(case, _parents(case, rows)) for d, j in enumerate(p))
        return {"bytes": 2 * moved * 2 * case["layers"] * case["hkv"] * case["dim"] * 2 + 8 * 4 * T + 8 * n, "flops": 0}
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    own_keys = sum(bin(m).count("1") for m in _masks(_parents(case, rows)))
    pairs = sum(q * b for b, q in zip(base, rows)) + own_keys
    return {"bytes": 2 * sum(b + q for b, q in zip(base, rows)) * hkv * d * 2 + 4 * T * hq * d + 8 * T,
            "flops": 4 * hq * d * pairs}


# ---- the definition in 64 bits ------------------------------------------------


def exact(case, seed):
    if case["kind"] == "inputs":
        return None
    s = prepare(case, seed)
    return _exact_attend(s) if case["kind"] == "attend" else _exact_commit(s)


def _exact_attend(s):
    case = s["case"]
    hkv, d = case["hkv"], case["dim"]
    group = case["hq"] // hkv
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=DEV)
    parents = _parents(case, s["rows_cpu"])
    for i, (n, q) in enumerate(zip(s["lens_cpu"], s["rows_cpu"])):
        blocks = s["tables"][i, :-(-n // case["block"])].long()
        k, v = (c[blocks].double().view(-1, hkv, d)[:n].transpose(0, 1).contiguous() for c in (s["kc"], s["vc"]))
        own_part = torch.zeros(q, q, dtype=torch.bool)
        for j, p in enumerate(parents[i]):
            if p >= 0:
                own_part[j] = own_part[p]
            own_part[j, j] = True
        seen = torch.cat((torch.ones(q, n - q, dtype=torch.bool), own_part), 1).to(DEV)
        a = s["starts_cpu"][i]
        qi = s["query"][a:a + q].double().view(q, hkv, group, d)
        for h in range(hkv):
            x = (qi[:, h].reshape(-1, d) @ k[h].T.contiguous() * s["scale"]).view(q, group, n)
            p = x.masked_fill_(~seen[:, None], -torch.inf).softmax(-1)
            out[a:a + q].view(q, hkv, group, d)[:, h] = (p.view(-1, n) @ v[h]).view(q, group, d)
    return out


def _exact_commit(s):
    cache = s["cache"].double().flatten(0, 1).flatten(1, 2)
    ids, chosen, par, slots = (s[k].tolist() for k in ("ids", "chosen", "parents", "slots"))
    a, to, of = 0, [], []
    for q in s["rows_cpu"]:
        at, d = 0, 0
        while at is not None:
            to.append(slots[a + d])
            of.append(slots[a + at])
            d += 1
            at = next((j for j in range(at + 1, q) if par[a + j] == at and ids[a + j] == chosen[a + at]), None)
        a += q
    cache[:, to] = cache[:, of]
    return None, None, cache.view(s["cache"].shape)
