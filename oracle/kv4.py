"""The 4-bit paged cache restated on the CPU: rows to codes, codes to records
and back, and attention over the stored values in float64.

The reference has no such cache; the record layout and the rounding rules are
those that include/nanoserve_paged.h declares.  Written from that description,
byte by byte where the product works in words.
"""

from __future__ import annotations

import numpy as np
import torch

V_POS = (0, 2, 1, 3)  # place of token t % 4 in its group of four


def quantise_rows(x: torch.Tensor, dtype: torch.dtype):
    """float32 rows [..., D] -> (codes uint8 [..., D], scale, offset [..., 1] in dtype)."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, offset = ((hi - lo) * torch.tensor(1 / 15)).to(dtype), lo.to(dtype)
    fine = torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(scale) & torch.isfinite(offset)
    scale = torch.where(fine, scale, torch.zeros_like(scale))
    offset = torch.where(fine, offset, torch.full_like(offset, float("nan")))
    s, b = scale.float(), offset.float()
    codes = torch.zeros_like(x)
    some = (s > 0).expand_as(x)
    codes[some] = ((x - b) / s)[some].round().clamp(0, 15)  # round: half to even, as rint
    return codes.to(torch.uint8), scale, offset


def stored_values(codes, scale, offset) -> torch.Tensor:
    """float64 values of stored rows."""
    return scale.double() * codes.double() + offset.double()


def _bits(x: torch.Tensor) -> np.ndarray:
    return x.view(torch.int16).numpy().view(np.uint16)


def put_rows(cache: torch.Tensor, slots, codes, scale, offset, is_v: bool) -> None:
    """Write rows [T, H, D] into a CPU cache tensor at slots (outside ones skipped)."""
    nb, heads, bs, w = cache.shape
    half = w - 4
    flat = cache.view(nb, heads, bs * w).numpy()
    c, s, b = codes.numpy(), _bits(scale)[..., 0], _bits(offset)[..., 0]
    for t, slot in enumerate(slots):
        slot = int(slot)
        if not 0 <= slot < nb * bs:
            continue
        blk, tk = divmod(slot, bs)
        for h in range(heads):
            packed = c[t, h, 0::2] | (c[t, h, 1::2] << 4)
            rec = flat[blk, h]
            if is_v:
                at = (tk // 4) * 4 * half + V_POS[tk % 4]
                rec[at:at + 4 * half:4] = packed
            else:
                rec[tk * half:(tk + 1) * half] = packed
            par = bs * half + 4 * tk
            rec[par:par + 4] = np.frombuffer(np.array([b[t, h], s[t, h]], dtype="<u2").tobytes(), dtype=np.uint8)


def get_rows(cache: torch.Tensor, slots, dtype: torch.dtype, is_v: bool):
    """(codes, scale, offset) of the rows in the given slots of a CPU cache tensor."""
    nb, heads, bs, w = cache.shape
    half = w - 4
    flat = cache.view(nb, heads, bs * w).numpy()
    T = len(slots)
    codes = np.zeros((T, heads, 2 * half), np.uint8)
    par = np.zeros((T, heads, 2), np.uint16)
    for t, slot in enumerate(slots):
        blk, tk = divmod(int(slot), bs)
        for h in range(heads):
            rec = flat[blk, h]
            if is_v:
                at = (tk // 4) * 4 * half + V_POS[tk % 4]
                b = rec[at:at + 4 * half:4]
            else:
                b = rec[tk * half:(tk + 1) * half]
            codes[t, h, 0::2], codes[t, h, 1::2] = b & 15, b >> 4
            par[t, h] = np.frombuffer(rec[bs * half + 4 * tk:bs * half + 4 * tk + 4].tobytes(), dtype="<u2")
    p = torch.from_numpy(par.view(np.int16)).view(dtype)
    return torch.from_numpy(codes), p[..., 1:], p[..., :1]


def attention_ref(query, kv, seq_lens, query_lens, scale: float):
    """Attention over stored rows in float64.

    kv[i] = ((codes, scale, offset) of K, of V), each over seq_lens[i] tokens.
    Returns (out [T, Hq, D], scaled [T, Hq, D], whole [T, Hq, D]): the result,
    sum p s |c - 8| and sum p |v| of each element (what roundings of p s act on
    where codes count from the middle, and roundings of p).
    """
    T, hq, d = query.shape
    out, scaled, whole = (torch.zeros(T, hq, d, dtype=torch.float64) for _ in range(3))
    row = 0
    for (k, v), n, ql in zip(kv, seq_lens, query_lens):
        if n and ql:
            hkv = k[0].shape[1]
            group = hq // hkv
            seen = torch.arange(n) <= (n - ql + torch.arange(ql))[:, None]  # [ql, n]
            some = seen.any(-1)
            for g in range(hkv):
                kk = stored_values(*(x[:n, g] for x in k))
                vc, vs, vb = (x[:n, g].double() for x in v)
                q = query[row:row + ql, g * group:(g + 1) * group].double().reshape(-1, d)
                s = ((q @ kk.T) * scale).view(ql, group, n).masked_fill(~seen[:, None], -torch.inf)
                p = torch.softmax(s[some], -1).reshape(-1, n)
                # A row that holds a NaN reaches the query rows that see it and no others.
                holds = torch.isnan(vb)[:, 0]
                reached = (seen[some] & holds).any(-1)[:, None, None]
                at = torch.arange(row, row + ql)[some]
                for dst, x in ((out, vs * vc + vb), (scaled, vs * (vc - 8).abs()), (whole, (vs * vc + vb).abs())):
                    o = (p @ torch.where(holds[:, None], 0.0, x)).view(-1, group, d)
                    dst[at, g * group:(g + 1) * group] = torch.where(reached, torch.nan, o)
        row += ql
    return out, scaled, whole
