"""Timed cases of the 4-bit KV cache and the sampler: what a decode or prompt step
of the engine runs between its projections, and what ends it.

Three kinds of case:

  write    the step's rotary embedding (or none) and the cache write of K and V
           in 4 bits, and the rows written, read back from the cache.
  attend   paged attention over a cache in 4 bits: decode rows, whole prompts,
           prompt chunks behind a context, or a mix of them.
  sample   one token per row of logits by temperature, top-k, top-p and min-p
           from given uniform numbers.

The cache of a layer is one uint8 tensor for K and one for V,
[num_blocks, kv_heads, block_size, head_dim / 2 + 4].  The bytes of a (block,
head) are its 4-bit codes, then one 32-bit word per token with the row's scale
in the high half and its offset in the low half, both in the model's dtype; a
value is scale * code + offset.  K's codes lie token after token, dims 2i and
2i + 1 in the low and high nibble of byte i.  V's lie in groups of four tokens:
the byte of dims 2i and 2i + 1 of token t is byte 4 i + (0, 2, 1, 3)[t % 4] of
group t / 4.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
VOCAB = 151936

# (query heads, KV heads, head size): the 0.5B model's, the larger-GQA
# benchmark's, and group sizes 1, 8 and 16 that the attention tests run.
HEADS = ((14, 2, 64), (28, 4, 128), (16, 2, 128), (8, 8, 64), (32, 2, 64))


def listed():
    return [
        # A decode step's write: one token of 32 sequences, the 0.5B heads.
        {"name": "write_step", "kind": "write", "tokens": 32, "rope": True, "hq": 14, "hkv": 2, "dim": 64,
         "block": 16, "dtype": "fp16"},
        # A prompt step's write at the engine's default token budget, larger heads.
        {"name": "write_prompt", "kind": "write", "tokens": 2048, "rope": True, "hq": 28, "hkv": 4, "dim": 128,
         "block": 16, "dtype": "bf16"},
        # Rows without a rotary embedding: a prefix brought in from elsewhere, odd length.
        {"name": "write_rows", "kind": "write", "tokens": 517, "rope": False, "hq": 8, "hkv": 8, "dim": 64,
         "block": 32, "dtype": "fp16"},
        # One interactive request: a single decode row.
        _attend("attend_one", "uniform", 1, 700, 800, lengths=1),
        # Decode at serving load: the headline benchmark's 32 contexts around 1K.
        _attend("attend_serving", "lognormal", 32, 16, 8192, median=1024, sigma=0.8, lengths=2),
        # Long-context decode of a larger GQA model: the stream of the cache.
        _attend("attend_long", "lognormal", 64, 128, 32768, median=4096, sigma=1.0, lengths=3,
                heads=(28, 4, 128), dtype="bf16"),
        # A continuous-batching step: 28 decode rows and four 512-token chunks.
        _attend("attend_mixed", "lognormal", 28, 16, 8192, median=1024, sigma=0.8, lengths=4,
                chunks=4, chunk=512, chunk_context=2048),
        # Two whole ragged prompts of the larger model within an 8K-token budget.
        _attend("attend_prompts", "uniform", 0, 1, 1, lengths=6, chunks=2, chunk=3700, chunk_context=0,
                heads=(28, 4, 128), dtype="bf16"),
        # The token of one interactive request.
        {"name": "sample_one", "kind": "sample", "rows": 1, "vocab": VOCAB, "dtype": "fp16", "filters": True},
        # A decode batch with every request's own settings.
        {"name": "sample_batch", "kind": "sample", "rows": 32, "vocab": VOCAB, "dtype": "bf16", "filters": True},
        # Many samples at once in float32, nothing filtered on some rows.
        {"name": "sample_wide", "kind": "sample", "rows": 256, "vocab": VOCAB, "dtype": "fp32", "filters": True},
    ]


def _attend(name, law, batch, lo, hi, median=0, sigma=0.0, lengths=0, chunks=0, chunk=0, chunk_context=0,
            heads=(14, 2, 64), dtype="fp16", block=16, index="int64"):
    c = {"kind": "attend", "law": law, "batch": batch, "lo": lo, "hi": hi, "median": median, "sigma": sigma,
         "lengths": lengths, "chunks": chunks, "chunk": chunk, "chunk_context": chunk_context,
         "hq": heads[0], "hkv": heads[1], "dim": heads[2], "dtype": dtype, "block": block, "index": index}
    return c if name is None else {"name": name, **c}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "decode", "decode", "decode", "mixed", "prefill", "sample", "sample"])
    heads = rng.choice(HEADS)
    dtype = rng.choice(["fp16", "bf16"])
    block = rng.choice([16, 16, 32])
    if kind == "write":
        # at most the rows of the largest listed write
        most = 2048 * (28 + 8) * 128 // ((heads[0] + 2 * heads[1]) * heads[2])
        return {"kind": "write", "tokens": _log_int(rng, 1, most), "rope": rng.random() < 0.7,
                "hq": heads[0], "hkv": heads[1], "dim": heads[2], "block": block, "dtype": dtype}
    if kind == "sample":
        return {"kind": "sample", "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 1000, VOCAB),
                "dtype": rng.choice(["fp16", "bf16", "fp32"]), "filters": rng.random() < 0.8}
    more = {"heads": heads, "dtype": dtype, "block": block, "index": rng.choice(["int32", "int64"]),
            "lengths": rng.randrange(1 << 20)}
    if kind == "decode":
        batch = _log_int(rng, 1, 64)
        # at most the cache of the largest listed decode step
        most = int(64 * 4 * 128 * 6000 / (heads[1] * heads[2] * batch))
        median = _log_int(rng, 48, max(64, min(6000, most)))
        return _attend(None, "lognormal", batch, 1, 8 * median, median=median, sigma=rng.choice([0.0, 0.5, 1.0]), **more)
    if kind == "mixed":
        return _attend(None, "lognormal", rng.randint(1, 40), 16, 4096, median=_log_int(rng, 64, 1024), sigma=0.7,
                       chunks=rng.randint(1, 4), chunk=_log_int(rng, 2, 512), chunk_context=_log_int(rng, 1, 2048),
                       **more)
    return _attend(None, "uniform", 0, 1, 1, chunks=rng.randint(1, 3), chunk=_log_int(rng, 16, 1200),
                   chunk_context=rng.choice([0, 0, _log_int(rng, 1, 4000)]), **more)


def _lengths(case):
    """(seq_lens, query_lens): decode rows, then prompt chunks."""
    rng = np.random.default_rng(case["lengths"])
    n = case["batch"]
    if case["law"] == "uniform":
        dec = rng.integers(case["lo"], case["hi"], size=n, endpoint=True)
    else:
        dec = np.clip(rng.lognormal(np.log(case["median"]), case["sigma"], n).astype(int), case["lo"], case["hi"])
    sl, ql = [int(v) for v in dec], [1] * n
    for _ in range(case["chunks"]):
        # ragged: at most an eighth shorter than the chunk
        q = case["chunk"] - int(rng.integers(0, case["chunk"] // 8, endpoint=True))
        ctx = int(rng.integers(0, case["chunk_context"], endpoint=True))
        sl.append(ctx + q)
        ql.append(q)
    return sl, ql


# ---- the cache's format, in plain torch ------------------------------------


def _quantise(x, dtype):
    """(codes, scale, offset) of the rows of float32 x; scale and offset as the dtype's values."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, offset = ((hi - lo) / 15).to(dtype), lo.to(dtype)
    s = scale.float()
    codes = torch.where(s > 0, ((x - offset.float()) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
    return codes.to(torch.uint8), scale, offset


def _params(scale, offset):
    """The 4 bytes of each row: offset, then scale."""
    return torch.cat((offset, scale), -1).view(torch.uint8)


def _records(x, dtype, is_v):
    """float32 [NB, H, BS, D] -> the cache tensor [NB, H, BS, D / 2 + 4]."""
    nb, h, bs, d = x.shape
    codes, scale, offset = _quantise(x, dtype)
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    if is_v:
        packed = packed.view(nb, h, bs // 4, 4, d // 2)[:, :, :, [0, 2, 1, 3]].transpose(-1, -2)
    both = torch.cat((packed.reshape(nb, h, -1), _params(scale, offset).reshape(nb, h, -1)), -1)
    return both.view(nb, h, bs, d // 2 + 4).contiguous()


def _values(cache, dtype, is_v):
    """The cache tensor's records [N, H, BS, D / 2 + 4] -> float32 values [N, H, BS, D]."""
    nb, h, bs, w = cache.shape
    d = 2 * (w - 4)
    flat = cache.reshape(nb, h, -1)
    packed, par = flat[..., :bs * (d // 2)], flat[..., bs * (d // 2):].contiguous().view(dtype).view(nb, h, bs, 2)
    if is_v:
        packed = packed.view(nb, h, bs // 4, d // 2, 4).transpose(-1, -2)[:, :, :, [0, 2, 1, 3]]
    packed = packed.reshape(nb, h, bs, d // 2)
    codes = torch.stack((packed & 15, packed >> 4), -1).view(nb, h, bs, d).float()
    return codes * par[..., 1:].float() + par[..., :1].float()


def _places(slots, heads, bs, d, is_v):
    """Byte places of the codes [T, H, D / 2] and of the parameters [T, H, 4] of the slots' rows."""
    rec = bs * (d // 2 + 4)
    blk, t = slots // bs, slots % bs
    base = (blk[:, None] * heads + torch.arange(heads, device=slots.device)) * rec
    i = torch.arange(d // 2, device=slots.device)
    if is_v:
        pos = torch.tensor([0, 2, 1, 3], device=slots.device)[t % 4]
        codes = ((t // 4)[:, None] * (d // 2) + i) * 4 + pos[:, None]
    else:
        codes = t[:, None] * (d // 2) + i
    par = bs * (d // 2) + t[:, None] * 4 + torch.arange(4, device=slots.device)
    return base[:, :, None] + codes[:, None], base[:, :, None] + par[:, None]


# ---- inputs -----------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return {"write": _prepare_write, "attend": _prepare_attend, "sample": _prepare_sample}[case["kind"]](case, seed, g)


def _prepare_write(case, seed, g):
    T, hq, hkv, d, bs = case["tokens"], case["hq"], case["hkv"], case["dim"], case["block"]
    dt = DTYPES[case["dtype"]]
    # The rows are views of one fused q|k|v projection's output.
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g, device=DEV).to(dt)
    q = qkv[:, :hq * d].view(T, hq, d)
    k = qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d)
    v = qkv[:, (hq + hkv) * d:].view(T, hkv, d)
    # Sequences of up to 64 tokens at scattered blocks, as a step's slots are.
    nb = 2 * (T // bs + T // 64 + 2)
    blocks = torch.randperm(nb, generator=g, device=DEV)
    t = torch.arange(T, device=DEV)
    slots = blocks[t // bs] * bs + t % bs
    pos = torch.randint(0, 4096, (T,), generator=g, device=DEV)
    inv = 1e6 ** (-torch.arange(0, d, 2, device=DEV, dtype=torch.float64) / d)
    ang = pos[:, None].double() * inv
    table = torch.cat((ang, ang), -1)
    cos, sin = table.cos().to(dt)[:, None], table.sin().to(dt)[:, None]
    shape = (nb, hkv, bs, d // 2 + 4)
    kc, vc = (torch.zeros(shape, dtype=torch.uint8, device=DEV) for _ in range(2))
    return {"case": case, "q": q, "k": k, "v": v, "cos": cos, "sin": sin, "slots": slots, "kc": kc, "vc": vc}


def _prepare_attend(case, seed, g):
    hq, hkv, d, bs = case["hq"], case["hkv"], case["dim"], case["block"]
    dt = DTYPES[case["dtype"]]
    sl, ql = _lengths(case)
    need = [max(1, -(-n // bs)) for n in sl]
    pool = math.ceil(1.25 * sum(need))
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))
    it = torch.int32 if case["index"] == "int32" else torch.int64
    tables = torch.zeros(len(sl), max(need), dtype=it)
    cur = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[cur:cur + n].to(it)
        cur += n
    # Rows around N(0, 1) with a head's own spread and shift, as K after its bias has.
    wide = 0.5 + torch.rand(hkv, 1, d, generator=g, device=DEV)
    shift = 0.5 * torch.randn(hkv, 1, d, generator=g, device=DEV)
    kc, vc = (_records(torch.randn(pool, hkv, bs, d, generator=g, device=DEV) * wide + shift, dt, is_v)
              for is_v in (False, True))
    query = torch.randn(sum(ql), hq, d, generator=g, device=DEV).to(dt)
    starts = [0, *np.cumsum(ql).tolist()]
    dev = lambda v: torch.tensor(v, dtype=it, device=DEV)  # noqa: E731
    return {"case": case, "query": query, "kc": kc, "vc": vc, "tables": tables.to(DEV), "lens": dev(sl),
            "starts": dev(starts), "sl": sl, "ql": ql, "starts_cpu": starts, "scale": d ** -0.5,
            "slots": torch.zeros(sum(ql), dtype=torch.int64, device=DEV)}


def _prepare_sample(case, seed, g):
    m, n = case["rows"], case["vocab"]
    z = 2.5 * torch.randn(m, n, generator=g, device=DEV)
    # A few tokens that the model favours, as real rows have.
    fav = torch.randint(0, n, (m, 24), generator=g, device=DEV)
    z.scatter_add_(1, fav, 12 * torch.rand(m, 24, generator=g, device=DEV))
    pick = lambda v, t: torch.tensor(v, dtype=t, device=DEV)[torch.randint(0, len(v), (m,), generator=g, device=DEV)]  # noqa: E731
    on = case["filters"]
    return {"case": case, "logits": z.to(DTYPES[case["dtype"]]),
            "uniform": torch.rand(m, generator=g, device=DEV),
            "temperature": pick([0.6, 0.8, 1.0, 1.3], torch.float32),
            "top_k": pick([0, 20, 50, 400] if on else [0], torch.int64),
            "top_p": pick([0.8, 0.9, 0.95, 1.0] if on else [1.0], torch.float32),
            "min_p": pick([0.0, 0.0, 0.02, 0.1] if on else [0.0], torch.float32)}


# ---- one pass ---------------------------------------------------------------


def run(state):
    return {"write": _run_write, "attend": _run_attend, "sample": _run_sample}[state["case"]["kind"]](state)


def _rotate(x, cos, sin):
    h = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., h:], x[..., :h]), -1) * sin


def _run_write(s):
    if own:
        from nanoserve_amd import gather_cache_int4, reshape_and_cache_int4, rope_reshape_and_cache_int4

        if s["case"]["rope"]:
            q = rope_reshape_and_cache_int4(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["kc"], s["vc"], s["slots"])
            return (q, *gather_cache_int4(s["kc"], s["vc"], s["slots"], s["q"].dtype))
        reshape_and_cache_int4(s["k"], s["v"], s["kc"], s["vc"], s["slots"])
        return gather_cache_int4(s["kc"], s["vc"], s["slots"], s["q"].dtype)
    dt, hkv, d, bs, slots = s["q"].dtype, s["case"]["hkv"], s["case"]["dim"], s["case"]["block"], s["slots"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if s["case"]["rope"]:
        cos, sin = s["cos"].float(), s["sin"].float()
        q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)

    def store_and_read(x, cache, is_v):
        codes, scale, offset = _quantise(x, dt)
        at, par = _places(slots, hkv, bs, d, is_v)
        flat = cache.view(-1)
        flat[at] = codes[..., 0::2] | (codes[..., 1::2] << 4)
        flat[par] = _params(scale, offset)
        both, p = flat[at], flat[par].view(dt)
        got = torch.stack((both & 15, both >> 4), -1).view(x.shape).float()
        return (got * p[..., 1:].float() + p[..., :1].float()).to(dt)

    kv = store_and_read(k, s["kc"], False), store_and_read(v, s["vc"], True)
    return (q.to(dt), *kv) if s["case"]["rope"] else kv


def _run_attend(s):
    if own:
        from nanoserve_amd import AttentionMetadata, paged_attention_int4

        md = AttentionMetadata(
            slot_mapping=s["slots"], query_start_loc=s["starts"], seq_lens=s["lens"], block_tables=s["tables"],
            max_query_len=max(s["ql"]), max_seq_len=max(s["sl"]), num_seqs=len(s["sl"]),
            num_tokens=s["query"].shape[0], is_decode_only=max(s["ql"]) == 1, query_lens_cpu=s["ql"],
            seq_lens_cpu=s["sl"], query_start_loc_cpu=s["starts_cpu"])
        return paged_attention_int4(s["query"], s["kc"], s["vc"], md, s["scale"])
    q, dt = s["query"], s["query"].dtype
    T, hq, d = q.shape
    hkv, n, most = s["case"]["hkv"], len(s["sl"]), max(s["ql"])
    keys = s["tables"].shape[1] * s["case"]["block"]
    # Rows padded to the longest query, keys to the longest table.
    starts, lens = s["starts"].long(), s["lens"].long()
    ql = starts[1:] - starts[:-1]
    j = torch.arange(most, device=DEV)
    row = (starts[:-1, None] + j).clamp(max=T - 1)
    qp = q[row].float().view(n, most, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, d)

    def gathered(cache, is_v):
        x = _values(cache[s["tables"].long().reshape(-1)], dt, is_v)
        return x.view(n, -1, hkv, x.shape[2], d).transpose(1, 2).reshape(n, hkv, keys, d)

    x = torch.matmul(qp, gathered(s["kc"], False).transpose(-1, -2).contiguous()) * s["scale"]
    x = x.view(n, hkv, most, hq // hkv, keys)
    last = (lens - ql)[:, None] + j
    seen = torch.arange(keys, device=DEV) <= last[..., None]
    x.masked_fill_(~seen[:, None, :, None], -torch.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, hkv, -1, keys), gathered(s["vc"], True)).view(n, hkv, most, hq // hkv, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(n, most, hq, d)
    return o[j < ql[:, None]].to(dt)


def _run_sample(s):
    if own:
        from nanoserve_amd import sample_rows

        return sample_rows(s["logits"], s["uniform"], s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                           min_p=s["min_p"])
    n = s["logits"].shape[1]
    # Sums in 64 bits: a token's place in the running sum decides whether it is kept or taken.
    z, at = s["logits"].float().sort(dim=-1, descending=True, stable=True)
    w = torch.exp((z.double() - z[:, :1].double()) / s["temperature"].double()[:, None])
    upto = w.cumsum(-1)
    k = torch.where((s["top_k"] > 0) & (s["top_k"] < n), s["top_k"], n)[:, None]
    rank = torch.arange(n, device=DEV)
    total = upto.gather(1, k - 1)
    keep = (rank < k) & (w >= s["min_p"].double()[:, None])
    p = s["top_p"].double()[:, None]
    keep &= (upto - w < p * total) | (p >= 1)
    keep[:, 0] = True
    kept = keep.sum(-1, keepdim=True)
    target = s["uniform"].double()[:, None] * upto.gather(1, kept - 1)
    taken = (upto <= target).sum(-1, keepdim=True).minimum(kept - 1)
    return at.gather(1, taken)[:, 0]


# ---- what a pass cannot do without -------------------------------------------


def work(case):
    if case["kind"] == "write":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        kv = 2 * t * hkv * (2 * d + (d // 2 + 4)) + 8 * t  # rows in, records out
        rope = 2 * t * (2 * hq * d + 2 * d) if case["rope"] else 0
        read = 2 * t * hkv * (d // 2 + 4 + 2 * d) + 8 * t
        return {"bytes": kv + rope + read, "flops": t * (3 * (hq + hkv) * d + 6 * hkv * d)}
    if case["kind"] == "sample":
        isz = 4 if case["dtype"] == "fp32" else 2
        return {"bytes": case["rows"] * (case["vocab"] * isz + 32), "flops": 0}
    sl, ql = _lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    pairs = sum(q * (n - q) + q * (q + 1) // 2 for n, q in zip(sl, ql))
    return {"bytes": 2 * sum(sl) * hkv * (d // 2 + 4) + 4 * sum(ql) * hq * d, "flops": 4 * hq * d * pairs}


# ---- the definition in 64 bits ------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "sample": _exact_sample}[case["kind"]](s)


def _exact_write(s):
    dt = s["q"].dtype

    def turned(x):
        x = x.double()
        if not s["case"]["rope"]:
            return x
        c, sn, h = s["cos"].double(), s["sin"].double(), x.shape[-1] // 2
        a, b = x[..., :h], x[..., h:]
        return torch.cat((a * c[..., :h] - b * sn[..., :h], b * c[..., h:] + a * sn[..., h:]), -1)

    def held(x):
        b = x.min(-1, keepdim=True).values
        step = ((x.max(-1, keepdim=True).values - b) / 15).to(dt).double()
        b = b.to(dt).double()
        return step * ((x - b) / step).nan_to_num().round().clamp(0, 15) + b

    kv = held(turned(s["k"])), held(s["v"].double())
    return (turned(s["q"]), *kv) if s["case"]["rope"] else kv


def _exact_attend(s):
    case = s["case"]
    hkv, bs, d, dt = case["hkv"], case["block"], case["dim"], s["query"].dtype
    group = case["hq"] // hkv
    out = torch.empty(s["query"].shape, dtype=torch.float64, device=DEV)
    split = bs * d // 2
    for i, (n, q) in enumerate(zip(s["sl"], s["ql"])):
        blocks = s["tables"][i, :-(-n // bs)].long()
        k, v = (c[blocks].view(len(blocks), hkv, -1) for c in (s["kc"], s["vc"]))
        nib = lambda b: torch.stack((b % 16, b // 16), -1).flatten(-2).double()  # noqa: E731
        kcode = nib(k[..., :split].reshape(-1, hkv, bs, d // 2))
        vb = v[..., :split].reshape(-1, hkv, bs // 4, d // 2, 4)
        vcode = nib(torch.stack((vb[..., 0], vb[..., 2], vb[..., 1], vb[..., 3]), 3).reshape(-1, hkv, bs, d // 2))
        rows = []
        for code, rec in ((kcode, k), (vcode, v)):
            par = rec[..., split:].contiguous().view(dt).double().view(-1, hkv, bs, 2)
            x = par[..., 1:] * code + par[..., :1]
            rows.append(x.transpose(0, 1).reshape(hkv, -1, d)[:, :n])
        a = s["starts_cpu"][i]
        qi = s["query"][a:a + q].double().view(q, hkv, group, d)
        late = torch.arange(n, device=DEV) > (n - q + torch.arange(q, device=DEV))[:, None]
        for h in range(hkv):
            x = (qi[:, h].reshape(-1, d) @ rows[0][h].T.contiguous() * s["scale"]).view(q, group, n)
            p = x.masked_fill_(late[:, None], -torch.inf).softmax(-1)
            out[a:a + q].view(q, hkv, group, d)[:, h] = (p.view(-1, n) @ rows[1][h]).view(q, group, d)
    return out


def _exact_sample(s):
    z = s["logits"].double().cpu().numpy()
    t, p, mp, u = (s[n].double().cpu().numpy() for n in ("temperature", "top_p", "min_p", "uniform"))
    k = s["top_k"].cpu().numpy()
    out = []
    for i in range(z.shape[0]):
        order = np.argsort(-z[i], kind="stable")
        w = np.exp((z[i][order] - z[i][order[0]]) / t[i])
        n = int(k[i]) if 0 < k[i] < len(w) else len(w)
        c = np.cumsum(w)
        if p[i] < 1:
            n_p = int(np.searchsorted(c, p[i] * c[n - 1], side="left")) + 1  # ranks with the sum before them below it
        else:
            n_p = n
        n = max(1, min(n, n_p, int((w >= mp[i]).sum())))
        r = min(n - 1, int(np.searchsorted(c, u[i] * c[n - 1], side="right")))
        out.append(int(order[r]))
    return torch.tensor(out, dtype=torch.int64)
