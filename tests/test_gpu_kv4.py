"""The 4-bit KV cache on an MI355X: the write, the rotary write and the
read-back against the CPU oracle bit for bit where no product is contracted,
and attention against the oracle's float64.

Attention's tolerance, per element, from the roundings that the kernels make:
  the output's own, eps(dtype) / 2 of the result;
  every product p * scale rounded once to float16, 2^-11 relative (half a unit
  of 2^-10).  With w the product and r its rounded value, the kernel forms
  sum r c - 8 sum r + sum (w (8) + p b) = sum p v + sum (r - w) (c - 8), so the
  roundings come to at most 2^-11 of sum p s |c - 8|;
  scores in float32: a dot product of up to 256 terms and the exponential are
  within 2^-13 of sum p |v| together for the scores drawn here (|score| < 64:
  64 * 2^-22 from the argument's rounding, as much again from the sum's order,
  2^-22 from the exponential, and factors of two to spare).
"""

from __future__ import annotations

import dataclasses
import itertools

import numpy as np
import pytest
import torch

from nanoserve_amd import (Int4PagedKVCache, gather_cache_int4, paged_attention_int4, reshape_and_cache_int4,
                           rope_reshape_and_cache_int4)
from nanoserve_amd import _lib
from nanoserve_amd.capture import graph_capture
from oracle import kv4
from tests._helpers import make_md, md_to
from tests.test_oracle_kv4 import WIDE_GROUPS

pytestmark = pytest.mark.gpu

DEV = "cuda"
DTYPES = [torch.float16, torch.bfloat16]


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _gap_cache(nb, heads, bs, d, dtype, seed=5):
    """A CPU cache tensor whose codes are random and whose every row holds NaN."""
    c = torch.randint(0, 256, (nb, heads, bs, d // 2 + 4), generator=_g(seed), dtype=torch.int32).to(torch.uint8)
    nan = torch.full((nb, heads, 2 * bs), float("nan"), dtype=dtype)
    c.view(nb, heads, -1)[:, :, bs * d // 2:] = nan.view(torch.uint8)
    return c


# ---- write -------------------------------------------------------------------


def _write_case(T, heads, bs, d, dtype, spread=1.0, seed=0):
    nb = -(-T // bs) + 3
    x = [(torch.randn(T, heads, d, generator=_g(seed + i)) * spread + i).to(dtype) for i in range(2)]
    slots = torch.randperm(nb * bs, generator=_g(seed + 2))[:T]
    caches = [_gap_cache(nb, heads, bs, d, dtype, seed + 3 + i) for i in range(2)]
    return x, slots, caches


def _expect(x, slots, caches, dtype):
    want = [c.clone() for c in caches]
    for i in range(2):
        kv4.put_rows(want[i], slots.tolist(), *kv4.quantise_rows(x[i].float(), dtype), is_v=i == 1)
    return want


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,heads,bs,d", [(1, 1, 4, 8), (1, 2, 16, 64), (7, 3, 8, 24), (33, 2, 16, 64), (50, 4, 32, 128),
                                          (19, 2, 12, 80), (16, 1, 16, 256), (300, 2, 16, 64)])
def test_write_is_the_oracles_bytes(T, heads, bs, d, dtype):
    (k, v), slots, caches = _write_case(T, heads, bs, d, dtype)
    got = [c.to(DEV) for c in caches]
    reshape_and_cache_int4(k.to(DEV), v.to(DEV), *got, slots.to(DEV))
    for a, b in zip(got, _expect((k, v), slots, caches, dtype)):
        assert torch.equal(a.cpu(), b)  # rows that are not written keep their bytes


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_of_wide_constant_and_non_finite_rows(dtype):
    T, heads, bs, d = 12, 2, 16, 64
    (k, v), slots, caches = _write_case(T, heads, bs, d, dtype)
    top = torch.finfo(dtype).max
    k[0], k[1, 0], k[1, 1] = 3.0, 0.0, -0.0                 # constant rows
    k[2, 0, 5], k[2, 1, 63], k[3, 0, 0] = float("nan"), float("inf"), -float("inf")
    k[4, 0, 0], k[4, 0, 1] = top, -top                      # the dtype's whole range
    k[5, 0] *= torch.finfo(dtype).smallest_normal           # a scale that rounds to a subnormal or zero
    v[6, 1, 7], v[7] = top, torch.finfo(dtype).tiny
    got = [c.to(DEV) for c in caches]
    reshape_and_cache_int4(k.to(DEV), v.to(DEV), *got, slots.to(DEV))
    want = _expect((k, v), slots, caches, dtype)
    for i, (a, b) in enumerate(zip(got, want)):
        ca, cb = (kv4.get_rows(c, slots, dtype, i == 1) for c in (a.cpu(), b))
        for x, y in zip(ca, cb):
            x, y = x.float(), y.float()
            assert torch.equal(torch.isnan(x), torch.isnan(y)) and torch.equal(x.nan_to_num(), y.nan_to_num())
    # A row with a NaN reads back as NaN, its neighbours as they were written.
    kk, _ = gather_cache_int4(*got, slots.to(DEV), dtype)
    assert torch.isnan(kk[2].float()).all() and torch.isnan(kk[3, 0].float()).all()
    assert torch.isfinite(kk[3, 1].float()).all() and torch.equal(kk[0].cpu(), k[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_write_of_strided_rows_and_skipped_slots(dtype, index):
    T, heads, bs, d = 21, 2, 16, 64
    _, slots, caches = _write_case(T, heads, bs, d, dtype)
    slots = slots.to(index)
    slots[3], slots[9] = -1, caches[0].shape[0] * bs
    fused = torch.randn(T, 4 * heads * d + 3, generator=_g(8)).to(dtype)  # an odd row length: rows off 8 bytes
    k = fused[:, 1:1 + heads * d].view(T, heads, d)
    v = fused[:, 2 * heads * d:4 * heads * d].view(T, heads, 2 * d)[:, :, ::2]  # no unit stride
    want = _expect((k, v), slots, caches, dtype)
    got = [c.to(DEV) for c in caches]
    dev = fused.to(DEV)
    reshape_and_cache_int4(dev[:, 1:1 + heads * d].view(T, heads, d),
                           dev[:, 2 * heads * d:4 * heads * d].view(T, heads, 2 * d)[:, :, ::2], *got, slots.to(DEV))
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,bs,d", [(1, 16, 64), (40, 8, 128), (13, 4, 24)])
def test_gather_reads_the_values_and_zero_outside(T, bs, d, dtype):
    heads = 2
    (k, v), slots, caches = _write_case(T, heads, bs, d, dtype)
    want = _expect((k, v), slots, caches, dtype)
    asked = torch.cat((slots.flip(0), slots[:1], torch.tensor([-1, want[0].shape[0] * bs])))  # a slot asked for twice
    got = gather_cache_int4(want[0].to(DEV), want[1].to(DEV), asked.to(DEV), dtype)
    for i in range(2):
        val = kv4.stored_values(*kv4.get_rows(want[i], asked[:-2], dtype, i == 1))
        # scale * code is exact in float32 (at most 15 bits), the sum rounds there and once more.
        assert ((got[i][:-2].double().cpu() - val).abs() <= val.abs() * (torch.finfo(dtype).eps / 2 + 2 ** -22)
                + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps).all()
        assert (got[i][-2:] == 0).all()


def _rope_case(T, hq, hkv, d, dtype, seed=0):
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=_g(seed)).to(dtype)
    ang = torch.rand(T, 1, d // 2, generator=_g(seed + 1)) * 6.3
    ang = torch.cat((ang, ang), -1)
    return qkv, ang.cos().to(dtype), ang.sin().to(dtype)


def _split(qkv, hq, hkv, d):
    T = qkv.shape[0]
    return (qkv[:, :hq * d].view(T, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(T, hkv, d),
            qkv[:, (hq + hkv) * d:].view(T, hkv, d))


def _turn(x, cos, sin):
    x, c, s, h = x.double(), cos.double(), sin.double(), x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * c[..., :h] - b * s[..., :h], b * c[..., h:] + a * s[..., h:]), -1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,hq,hkv,d,bs", [(1, 14, 2, 64, 16), (37, 28, 4, 128, 16), (5, 4, 4, 80, 8), (9, 3, 1, 8, 4),
                                            (2100, 14, 2, 64, 16), (701, 27, 3, 128, 16), (3500, 6, 2, 40, 8)])
def test_rope_write_matches_float64(T, hq, hkv, d, bs, dtype):
    qkv, cos, sin = _rope_case(T, hq, hkv, d, dtype)
    nb = -(-T // bs) + 2
    slots = torch.randperm(nb * bs, generator=_g(4))[:T]
    caches = [_gap_cache(nb, hkv, bs, d, dtype, 6 + i) for i in range(2)]
    got = [c.to(DEV) for c in caches]
    q, k, v = _split(qkv, hq, hkv, d)
    out = rope_reshape_and_cache_int4(*_split(qkv.to(DEV), hq, hkv, d), cos.to(DEV), sin.to(DEV), *got, slots.to(DEV))
    eps = torch.finfo(dtype).eps
    want = _turn(q, cos, sin)
    size = q.double().abs() + q.double().roll(d // 2, -1).abs()  # |x1| + |x2|: two float32 roundings of each product
    # Half a step of a subnormal result is smallest_normal * eps / 2 whatever its size: the step below the smallest
    # normal number is the one just above it, smallest_normal * eps.
    tiny = torch.finfo(dtype).smallest_normal * eps
    assert ((out.double().cpu() - want).abs() <= want.abs() * eps / 2 + size * 2 ** -22 + tiny / 2).all()
    # K: within half a step of the rotated row, plus what the roundings of scale and offset move.
    codes, s, b = kv4.get_rows(got[0].cpu(), slots, dtype, False)
    kr = _turn(k, cos, sin)
    err = (kv4.stored_values(codes, s, b) - kr).abs()
    assert (err <= s.double() * (0.5 + 15 * eps / 2 + 1e-4) + kr.abs().amax(-1, keepdim=True) * eps + 16 * tiny).all()
    lo, hi = kr.amin(-1, keepdim=True), kr.amax(-1, keepdim=True)
    assert ((b.double() - lo).abs() <= lo.abs() * (eps / 2 + 2 ** -20) + 2 ** -20).all()
    assert ((s.double() - (hi - lo) / 15).abs() <= (hi - lo) / 15 * (eps / 2 + 2 ** -20) + 2 ** -20).all()
    # The same in float32, each product and sum rounded: the oracle's bytes.
    x, c, n = k.float(), cos.float(), sin.float()
    h = d // 2
    k32 = torch.cat((x[..., :h] * c[..., :h] - x[..., h:] * n[..., :h], x[..., h:] * c[..., h:] + x[..., :h] * n[..., h:]),
                    -1)
    kv4.put_rows(caches[0], slots.tolist(), *kv4.quantise_rows(k32, dtype), is_v=False)
    assert torch.equal(got[0].cpu(), caches[0])
    # V is not rotated.
    kv4.put_rows(caches[1], slots.tolist(), *kv4.quantise_rows(v.float(), dtype), is_v=True)
    assert torch.equal(got[1].cpu(), caches[1])
    # In place: the same.
    q = q.contiguous().to(DEV)
    rope_reshape_and_cache_int4(q, k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), *got, slots.to(DEV), out=q)
    assert torch.equal(q, out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rope_write_in_place_without_rotation_and_unaligned(dtype):
    T, hq, hkv, d, bs = 11, 4, 2, 64, 16
    qkv, _, _ = _rope_case(T, hq, hkv, d, dtype)
    q, k, v = (x.contiguous().to(DEV) for x in _split(qkv, hq, hkv, d))
    one, zero = torch.ones(T, d, dtype=dtype, device=DEV), torch.zeros(T, 1, d, dtype=dtype, device=DEV)
    slots = torch.arange(T, device=DEV, dtype=torch.int32) + 3
    a, b, c = (Int4PagedKVCache(2, bs, 1, hkv, d, dtype, DEV) for _ in range(3))
    reshape_and_cache_int4(k, v, a.k_cache[0], a.v_cache[0], slots)
    before = q.clone()
    out = rope_reshape_and_cache_int4(q, k, v, one, zero, b.k_cache[0], b.v_cache[0], slots, out=q)
    assert out.data_ptr() == q.data_ptr() and torch.equal(q, before)  # cos 1, sin 0
    assert torch.equal(a.k_cache[0], b.k_cache[0]) and torch.equal(a.v_cache[0], b.v_cache[0])
    # Rows that start off an 8-byte boundary.
    odd = torch.empty(T * hq * d + 1, dtype=dtype, device=DEV)[1:].view(T, hq, d)
    odd.copy_(before)
    cos, sin = (x.to(DEV) for x in _rope_case(T, hq, hkv, d, dtype, seed=3)[1:])
    x = rope_reshape_and_cache_int4(odd, k, v, cos, sin, b.k_cache[0], b.v_cache[0], slots)
    y = rope_reshape_and_cache_int4(before, k, v, cos, sin, c.k_cache[0], c.v_cache[0], slots)
    assert torch.equal(x, y) and torch.equal(b.k_cache[0], c.k_cache[0])


def test_write_refuses_what_it_cannot_take():
    c = Int4PagedKVCache(2, 16, 1, 2, 64, torch.float16, DEV)
    kc, vc = c.k_cache[0], c.v_cache[0]
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16, device=DEV), torch.arange(3, device=DEV)
    with pytest.raises(TypeError):
        reshape_and_cache_int4(x.float(), x.float(), kc, vc, slots)
    with pytest.raises(TypeError):
        reshape_and_cache_int4(x, x.bfloat16(), kc, vc, slots)
    with pytest.raises(ValueError):
        reshape_and_cache_int4(x[:, :1], x[:, :1], kc, vc, slots)
    with pytest.raises(ValueError):
        reshape_and_cache_int4(x, x, kc, vc, slots[:2])
    with pytest.raises(ValueError):
        reshape_and_cache_int4(x, x, kc, vc.transpose(0, 1), slots)
    with pytest.raises(ValueError):
        reshape_and_cache_int4(x, x, kc, vc, slots.cpu())
    with pytest.raises(ValueError):
        rope_reshape_and_cache_int4(x, x, x, x[:, 0], x[:, 0, :32], kc, vc, slots)
    with pytest.raises(ValueError):
        gather_cache_int4(kc, vc, slots[None], torch.float16)
    with pytest.raises(TypeError):
        gather_cache_int4(kc, vc, slots, torch.float32)
    # No tokens: nothing happens.
    reshape_and_cache_int4(x[:0], x[:0], kc, vc, slots[:0])
    assert rope_reshape_and_cache_int4(x[:0], x[:0], x[:0], x[:0, 0], x[:0, 0], kc, vc, slots[:0]).shape == (0, 2, 64)
    assert gather_cache_int4(kc, vc, slots[:0], torch.float16)[0].shape == (0, 2, 64)


# ---- attention ----------------------------------------------------------------


@dataclasses.dataclass
class Case:
    q: torch.Tensor
    kc: torch.Tensor
    vc: torch.Tensor
    md: object
    kv: list
    seqs: list
    query_lens: list
    scale: float


def _case(seqs, query_lens, hq, hkv, d, bs, dtype, seed=0, index=torch.int32, spread=1.0, host=True, extra=2):
    need = [-(-n // bs) for n in seqs]
    nb = sum(need) + extra
    perm = torch.randperm(nb, generator=_g(seed)).tolist()
    kc, vc = (_gap_cache(nb, hkv, bs, d, dtype, seed + i) for i in range(2))
    tables, kv, cur = [], [], 0
    for i, n in enumerate(seqs):
        t = perm[cur:cur + need[i]]
        cur += need[i]
        tables.append(t)
        slots = [t[p // bs] * bs + p % bs for p in range(n)]
        pair = []
        for j, c in enumerate((kc, vc)):
            x = torch.randn(n, hkv, d, generator=_g(seed + 10 * i + j)) * spread + 0.3 * j
            rows = kv4.quantise_rows(x, dtype) if n else tuple(
                torch.zeros(0, hkv, w, dtype=t) for w, t in ((d, torch.uint8), (1, dtype), (1, dtype)))
            kv4.put_rows(c, slots, *rows, is_v=j == 1)
            pair.append(rows)
        kv.append(tuple(pair))
    md = make_md(seqs, query_lens, tables, bs, index_dtype=index, with_cpu_lists=host)
    q = torch.randn(sum(query_lens), hq, d, generator=_g(seed + 99)).to(dtype)
    return Case(q, kc, vc, md, kv, list(seqs), list(query_lens), d ** -0.5)


def _run(c: Case, scale=None):
    return paged_attention_int4(c.q.to(DEV), c.kc.to(DEV), c.vc.to(DEV), md_to(c.md, DEV),
                                c.scale if scale is None else scale)


def _check(got, c: Case, scale=None, what=""):
    out, scaled, whole = kv4.attention_ref(c.q, c.kv, c.seqs, c.query_lens, c.scale if scale is None else scale)
    got = got.double().cpu()
    tol = out.abs() * torch.finfo(c.q.dtype).eps / 2 + scaled * 2 ** -11 + whole * 2 ** -13 + 1e-7
    assert torch.equal(torch.isnan(got), torch.isnan(out)), what
    over = ((got - out).abs() - tol).nan_to_num(nan=-1.0)
    assert (over <= 0).all(), f"{what}: {(over > 0).sum()} of {over.numel()} over, worst {over.max():.3e}"


HEADS = [(14, 2, 64), (28, 4, 128), (4, 4, 64), (8, 1, 128), (16, 1, 64), (6, 2, 128)]
ODD_HEADS = [(4, 2, 8), (6, 3, 24), (4, 1, 80), (2, 2, 256), (40, 2, 64), (34, 2, 128)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS + ODD_HEADS)
def test_decode_over_lengths(hq, hkv, d, dtype):
    seqs = [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 127, 200]
    c = _case(seqs, [1] * len(seqs), hq, hkv, d, 16, dtype)
    _check(_run(c), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [4, 8, 12, 16, 24, 32, 48, 64])
def test_block_sizes(bs, d, dtype):
    c = _case([5, 70, 131, 48], [1, 1, 1, 1], 6, 2, d, bs, dtype, index=torch.int64)
    _check(_run(c), c)
    c = _case([5, 70, 131, 48], [5, 1, 40, 3], 6, 2, d, bs, dtype, seed=1)
    _check(_run(c), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", HEADS + ODD_HEADS)
def test_prompts_chunks_and_decode_rows_together(hq, hkv, d, dtype):
    # whole prompts, chunks behind a context, single rows, an empty query, one longer than its context
    seqs, query_lens = [33, 100, 1, 77, 20, 64, 3], [33, 37, 1, 1, 0, 64, 5]
    c = _case(seqs, query_lens, hq, hkv, d, 16, dtype)
    _check(_run(c), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128)])
def test_one_long_context(hq, hkv, d, dtype):
    c = _case([5000], [1], hq, hkv, d, 16, dtype)
    _check(_run(c), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("host", [True, False])
def test_a_short_chunk_behind_a_long_context(hq, hkv, d, dtype, host):
    c = _case([3000, 900, 1], [4, 300, 1], hq, hkv, d, 16, dtype, host=host)
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("host", [True, False])
def test_many_sequences(d, host):
    """More sequences than a wave has lanes, contexts of one and of several ranges, empty ones among them."""
    rng = np.random.default_rng(3)
    n = 150
    seqs = [int(x) for x in rng.integers(0, 60, n)]
    for i, long in ((5, 1500), (63, 1200), (64, 1100), (149, 1300)):
        seqs[i] = long
    c = _case(seqs, [1] * n, 4, 2, d, 16, torch.float16, host=host)
    _check(_run(c), c)
    ql = [1] * n
    for i in range(0, n, 7):
        ql[i] = min(40, seqs[i])
    c = _case(seqs, ql, 4, 2, d, 16, torch.bfloat16, host=host, seed=1)
    _check(_run(c), c)


@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("n", [4200, 700])
def test_thousands_of_sequences(n, host):
    rng = np.random.default_rng(n)
    seqs = [int(x) for x in rng.integers(0, 5, n)]
    seqs[0] = seqs[n // 2] = seqs[-1] = 40
    c = _case(seqs, [1] * n, 2, 1, 64, 16, torch.float16, host=host, extra=0)
    _check(_run(c), c)
    ql = [1 + int(x) for x in rng.integers(0, 2, n)]
    ql[5], ql[-1] = 0, 40
    c = _case(seqs, ql, 2, 1, 64, 16, torch.bfloat16, host=host, extra=0, seed=1)
    _check(_run(c), c)
    ql = [1] * n
    ql[n // 2], ql[-2] = 30, 3
    c = _case(seqs, ql, 2, 1, 64, 16, torch.float16, host=host, extra=0, seed=2)
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128])
def test_one_row_of_a_longer_query_layout(d):
    """One-row sequences given by offsets, with no decode-only flag, and none of them."""
    c = _case([700, 40, 1], [1, 1, 1], 6, 2, d, 16, torch.float16)
    want = _run(c)
    c.md.is_decode_only = False
    assert torch.equal(_run(c), want)
    _check(want, c)
    c = _case([700, 40], [2, 40], 6, 2, d, 16, torch.float16)
    _check(_run(c), c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,n", [(14, 2, 64, 60), (14, 2, 64, 30), (28, 4, 128, 16), (28, 4, 128, 8), (40, 2, 64, 24)])
def test_enough_rows_to_fill_the_device(hq, hkv, d, n, dtype):
    """Thousands of query rows, whole prompts and chunks, with decode rows among them."""
    rng = np.random.default_rng(d)
    ql = [int(x) for x in rng.integers(70, 130, n)]
    seqs = [q + int(rng.integers(0, 60)) * int(i % 3 == 0) for i, q in enumerate(ql)]
    for i, long in ((1, 400), (2, 33), (n - 1, 1)):
        seqs[i], ql[i] = long, 1
    c = _case(seqs, ql, hq, hkv, d, 16, dtype)
    _check(_run(c), c)


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (28, 4, 128), (4, 2, 24)])
@pytest.mark.parametrize("told", [[1, 1, 1], [2, 2, 2], [34, 1, 40]])
def test_lengths_that_the_host_did_not_expect(hq, hkv, d, told):
    """The device's lengths decide what is computed: here the host's lists are of another step."""
    c = _case([700, 33, 90], [1, 33, 41], hq, hkv, d, 16, torch.float16)
    c.md.query_lens_cpu = told
    c.md.seq_lens_cpu = [1, 1, 1]
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
def test_empty_contexts_are_zero(d):
    c = _case([0, 3, 0], [1, 1, 1], 4, 2, d, 16, torch.float16)
    got = _run(c)
    assert (got[0] == 0).all() and (got[2] == 0).all()
    _check(got, c)
    c = _case([0, 3, 0], [2, 6, 3], 4, 2, d, 16, torch.float16, seed=3)
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(d, scale):
    c = _case([40, 90], [1, 50], 4, 2, d, 16, torch.bfloat16, spread=0.4)
    _check(_run(c, scale), c, scale)
    c = _case([40, 90], [1, 1], 4, 2, d, 16, torch.float16, spread=0.4)
    _check(_run(c, scale), c, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 24])
def test_nan_rows_reach_the_queries_that_see_them_and_no_others(d, dtype):
    bs = 16
    c = _case([90, 70], [90, 1], 4, 2, d, bs, dtype)
    for which, pos, head in ((0, 40, 0), (1, 61, 1)):
        cache = (c.kc, c.vc)[which]
        slot = int(c.md.block_tables[0, pos // bs]) * bs + pos % bs
        codes, s, b = (x[pos:pos + 1].clone() for x in c.kv[0][which])
        b[:, head] = float("nan")
        c.kv[0][which][2][pos, head] = float("nan")
        kv4.put_rows(cache, [slot], codes, s, b, is_v=which == 1)
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
def test_a_bad_block_id_is_nan_for_the_rows_that_need_it(d):
    bs = 16
    c = _case([100, 100, 30], [100, 1, 1], 4, 2, d, bs, torch.float16)
    c.md.block_tables[0, 3] = c.kc.shape[0]      # keys 48..63
    c.md.block_tables[1, 6] = -1                 # keys 96..99
    c.md.block_tables[2, 2:] = 1 << 30           # behind the context: never read
    got = _run(c).float().cpu()
    assert torch.isfinite(got[:48]).all() and torch.isnan(got[48:101]).all() and torch.isfinite(got[101]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_scales_that_differ_by_orders_of_magnitude(dtype):
    """Rows of V from 1e-3 to 1e3: the float16 operand p * scale keeps its bits."""
    d, bs, hkv = 64, 16, 2
    for seqs, ql in (([200], [1]), ([200], [60])):
        c = _case(seqs, ql, 4, hkv, d, bs, dtype)
        size = torch.logspace(-3, 3, 200)[torch.randperm(200, generator=_g(1))][:, None, None]
        rows = kv4.quantise_rows(torch.randn(200, hkv, d, generator=_g(2)) * size, dtype)
        slots = [int(c.md.block_tables[0, p // bs]) * bs + p % bs for p in range(200)]
        kv4.put_rows(c.vc, slots, *rows, is_v=True)
        c.kv[0] = (c.kv[0][0], rows)
        _check(_run(c), c)


@pytest.mark.parametrize("size", [1e-30, 1e-4, 30.0])
def test_query_sizes(size):
    """The query is scaled by a power of two into float16's range and back."""
    dtype = torch.bfloat16
    for d, ql in itertools.product((64, 128), (1, 20)):
        c = _case([120], [ql], 4, 2, d, 16, dtype, spread=0.05)
        c.q = (c.q.float() * size).to(dtype)
        _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("dtype,size", [(torch.float16, 6e4), (torch.bfloat16, 6e4), (torch.bfloat16, 3e7),
                                        (torch.bfloat16, 1e25)])
def test_query_rows_of_very_different_sizes(d, dtype, size):
    """A row up to 10^25 times its neighbours leaves them their precision."""
    for seqs, ql in (([120], [40]), ([90, 50], [1, 1]), ([400], [200])):
        c = _case(seqs, ql, 4, 2, d, 16, dtype, spread=0.05)
        c.q[0, 1] *= size
        c.q[-1, 2] = torch.sign(c.q[-1, 2]) * size
        _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_query_rows_spoil_no_others(d, dtype):
    for seqs, ql in (([120], [40]), ([90, 50], [1, 1])):
        c = _case(seqs, ql, 4, 2, d, 16, dtype)
        want = _run(c)
        c.q[0, 1, 3], c.q[-1, 2, 7] = float("nan"), float("inf")
        got = _run(c)
        assert torch.isnan(got[0, 1]).all() and torch.isnan(got[-1, 2]).all()
        got[0, 1], got[-1, 2] = want[0, 1], want[-1, 2]
        assert torch.equal(got, want)


def test_rows_of_no_sequence_are_zero():
    c = _case([40, 20], [30, 1], 4, 2, 64, 16, torch.float16, host=False)
    q = torch.cat((c.q, torch.ones(5, 4, 64, dtype=torch.float16)))
    md = dataclasses.replace(md_to(c.md, DEV), num_tokens=36)
    got = paged_attention_int4(q.to(DEV), c.kc.to(DEV), c.vc.to(DEV), md, c.scale)
    assert (got[31:] == 0).all()
    _check(got[:31], c)


def test_offsets_past_32_bits():
    """A cache of more than 4 GiB: the last blocks' rows are the first blocks'."""
    hkv, d, bs = 2, 128, 16
    record = hkv * bs * (d // 2 + 4)
    nb = (1 << 32) // record + 40
    c = _case([100, 300], [1, 64], 4, hkv, d, bs, torch.float16)
    small = c.kc.shape[0]
    big = []
    for cache in (c.kc, c.vc):
        x = torch.zeros((nb, *cache.shape[1:]), dtype=torch.uint8, device=DEV)
        x[nb - small:] = cache.to(DEV)
        big.append(x)
    md = md_to(c.md, DEV)
    md.block_tables = md.block_tables + (nb - small)
    _check(paged_attention_int4(c.q.to(DEV), *big, md, c.scale), c)
    slots = torch.arange(nb * bs - 8, nb * bs, device=DEV)
    x = torch.randn(8, hkv, d, generator=_g(1)).half()
    reshape_and_cache_int4(x.to(DEV), x.to(DEV), *big, slots)
    got = gather_cache_int4(*big, slots, torch.float16)[0].double().cpu()
    assert ((got - x.double()).abs() <= (x.amax(-1) - x.amin(-1))[..., None].double() / 15 * 0.51 + 2 ** -10).all()


def test_attention_refuses_what_it_cannot_take():
    c = _case([20, 20], [1, 1], 4, 2, 64, 16, torch.float16)
    q, kc, vc, md = c.q.to(DEV), c.kc.to(DEV), c.vc.to(DEV), md_to(c.md, DEV)
    with pytest.raises(TypeError):
        paged_attention_int4(q.float(), kc, vc, md, 1.0)
    with pytest.raises(ValueError):
        paged_attention_int4(q[:1], kc, vc, md, 1.0)
    with pytest.raises(ValueError):
        paged_attention_int4(q[:, :3], kc, vc, md, 1.0)
    with pytest.raises(ValueError):
        paged_attention_int4(q[..., :32], kc, vc, md, 1.0)
    with pytest.raises(ValueError):
        paged_attention_int4(q.cpu(), kc, vc, md, 1.0)
    with pytest.raises(ValueError):
        paged_attention_int4(q, kc, vc, dataclasses.replace(md, max_seq_len=33), 1.0)
    with pytest.raises(RuntimeError):
        paged_attention_int4(q, kc, vc, md, float("nan"))
    none = dataclasses.replace(md, num_tokens=0)
    assert paged_attention_int4(q[:0], kc, vc, none, 1.0).shape == (0, 4, 64)


def _graph_case(c: Case):
    return c.q.to(DEV), c.kc.to(DEV), c.vc.to(DEV), md_to(c.md, DEV)


@pytest.mark.parametrize("seqs,query_lens", [([700, 33, 1500, 1], [1, 1, 1, 1]), ([700, 33, 90], [1, 33, 40])])
def test_graph_replays_with_eager_calls_between(seqs, query_lens):
    a = _case(seqs, query_lens, 14, 2, 64, 16, torch.float16)
    q, kc, vc, md = _graph_case(a)
    b = _case([64, 2000], [1, 1], 8, 2, 128, 16, torch.bfloat16, seed=4)
    other = _graph_case(b)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged_attention_int4(q, kc, vc, md, a.scale)
    stream.synchronize()
    g, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with graph_capture(g, stream):
        out = paged_attention_int4(q, kc, vc, md, a.scale)
    with graph_capture(g2, stream):
        out2 = paged_attention_int4(*other, b.scale)
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=_g(step)).half())
        md.seq_lens[0] = 700 - 100 * step  # a replay follows the device's lengths
        want = paged_attention_int4(q, kc, vc, dataclasses.replace(md, seq_lens_cpu=None), a.scale)
        want2 = paged_attention_int4(*other, b.scale)
        torch.cuda.synchronize()
        # Two graphs at once, on streams of their own.
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(s1):
            g.replay()
        with torch.cuda.stream(s2):
            g2.replay()
        torch.cuda.synchronize()
        # Both are held to float64's tolerance of each other; the splits may differ.
        assert torch.allclose(out.float(), want.float(), atol=2e-3, rtol=2e-3)
        assert torch.equal(out2, want2)


@pytest.mark.parametrize("d", [64, 128])
def test_a_replay_with_longer_contexts_and_other_chunks(d):
    """A graph captured at one step's lengths and replayed at another's."""
    first = _case([20, 9, 30], [1, 1, 30], 6, 2, d, 16, torch.float16)
    later = _case([1500, 60, 17], [1, 30, 1], 6, 2, d, 16, torch.float16, seed=5)
    width = max(c.md.block_tables.shape[1] for c in (first, later))
    blocks = max(c.kc.shape[0] for c in (first, later))

    def padded(c):
        grow = lambda x: torch.cat((x, torch.zeros(blocks - x.shape[0], *x.shape[1:], dtype=x.dtype)))  # noqa: E731
        tables = torch.zeros(3, width, dtype=c.md.block_tables.dtype)
        tables[:, :c.md.block_tables.shape[1]] = c.md.block_tables
        return c.q.to(DEV), grow(c.kc).to(DEV), grow(c.vc).to(DEV), tables.to(DEV)

    q, kc, vc, tables = padded(first)
    md = dataclasses.replace(md_to(first.md, DEV), block_tables=tables, max_seq_len=1500)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged_attention_int4(q, kc, vc, md, first.scale)
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with graph_capture(g, stream):
        out = paged_attention_int4(q, kc, vc, md, first.scale)
    for c in (later, first, later, later):
        for dst, src in zip((q, kc, vc, tables), padded(c)):
            dst.copy_(src)
        md.seq_lens.copy_(c.md.seq_lens)
        md.query_start_loc.copy_(c.md.query_start_loc)
        g.replay()
        _check(out, c)


def test_streams_and_repeated_calls_agree():
    c = _case([900, 40, 2200], [1, 1, 1], 28, 4, 128, 16, torch.bfloat16)
    q, kc, vc, md = _graph_case(c)
    want = paged_attention_int4(q, kc, vc, md, c.scale)
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs.append(paged_attention_int4(q, kc, vc, md, c.scale))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    _check(want, c)


@pytest.mark.parametrize("dtype", DTYPES)
def test_write_then_attend_and_write_again(dtype):
    """A sequence grown token by token, as decoding grows it: rotary write, attention, next token."""
    hq, hkv, d, bs, n = 14, 2, 64, 16, 37
    cache = Int4PagedKVCache(6, bs, 1, hkv, d, dtype, DEV)
    kc, vc = cache.k_cache[0], cache.v_cache[0]
    table = [4, 1, 5]
    qkv, cos, sin = _rope_case(n, hq, hkv, d, dtype)
    stored = []
    for t in range(n):
        q, k, v = (x.to(DEV) for x in _split(qkv[t:t + 1], hq, hkv, d))
        slot = torch.tensor([table[t // bs] * bs + t % bs], device=DEV)
        q = rope_reshape_and_cache_int4(q, k, v, cos[t:t + 1].to(DEV), sin[t:t + 1].to(DEV), kc, vc, slot)
        md = make_md([t + 1], [1], [table], bs, device=DEV)
        out = paged_attention_int4(q, kc, vc, md, d ** -0.5)
        stored.append((q.cpu(), out.cpu()))
    slots = [table[t // bs] * bs + t % bs for t in range(n)]
    rows = tuple(kv4.get_rows(c.cpu(), slots, dtype, i == 1) for i, c in enumerate((kc, vc)))
    # All rows at once, as one prompt over the same cache.
    q = torch.cat([s[0] for s in stored])
    md = make_md([n], [n], [table], bs)
    c = Case(q, kc.cpu(), vc.cpu(), md, [rows], [n], [n], d ** -0.5)
    _check(torch.cat([s[1] for s in stored]), c, what="grown")
    _check(_run(c), c, what="whole")
    k, v = cache.read(0, torch.tensor(slots, device=DEV))
    assert np.allclose(k.double().cpu().numpy(), kv4.stored_values(*rows[0]).numpy(), atol=2e-2, rtol=1e-2)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,seqs", WIDE_GROUPS)
def test_decode_of_wide_groups_over_split_keys(hq, hkv, d, seqs, dtype):
    """More than 16 query heads per KV head, one row a sequence, no query offsets, keys in
    ranges: eager calls and replays, with the host's lengths and without."""
    c = _case(seqs, [1] * len(seqs), hq, hkv, d, 16, dtype)
    q, kc, vc, md = _graph_case(c)
    md = dataclasses.replace(md, query_start_loc=None, query_start_loc_cpu=None)
    _check(paged_attention_int4(q, kc, vc, md, c.scale), c, what="host lengths")
    md = dataclasses.replace(md, query_lens_cpu=None, seq_lens_cpu=None)
    want = paged_attention_int4(q, kc, vc, md, c.scale)
    _check(want, c, what="device lengths")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with graph_capture(g, stream):
        out = paged_attention_int4(q, kc, vc, md, c.scale)
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def _workspace(c: Case):
    """The workspace of the call, as its wrapper asks for it."""
    md, (_, hq, d), (_, hkv, bs, _) = c.md, c.q.shape, c.kc.shape
    ones = md.num_seqs if md.is_decode_only else md.query_lens_cpu.count(1)
    return _lib.load().ns_paged_attention_int4_workspace_size(md.num_seqs, hq, hkv, d, bs, md.max_seq_len, md.num_tokens,
                                                              md.is_decode_only, sum(md.seq_lens_cpu), ones)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hq,hkv,d,n", [(14, 2, 64, 40), (28, 4, 128, 40), (4, 2, 64, 300), (20, 1, 128, 70)])
@pytest.mark.parametrize("host", [True, False])
def test_one_long_context_among_short_ones(hq, hkv, d, n, host, dtype):
    """Only the long contexts have ranges, and cells for them; one is the last of all."""
    rng = np.random.default_rng(n)
    seqs = [int(x) for x in rng.integers(0, 30, n)]
    seqs[n // 3], seqs[-1] = 5000, 1700
    c = _case(seqs, [1] * n, hq, hkv, d, 16, dtype, host=host)
    _check(_run(c), c)
    ql = [1] * n
    ql[n // 3], ql[n // 2], ql[-1] = 3, min(5, seqs[n // 2]), 2
    c = _case(seqs, ql, hq, hkv, d, 16, dtype, host=host, seed=1)
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("short", [0, 70])
def test_decode_ranges_that_outgrow_the_workspace(d, short):
    """Lists of another step promise few keys: ranges get longer until their results fit."""
    h, long = 64, 3000
    seqs = [20] * short + [long] * 5
    c = _case(seqs, [1] * len(seqs), h, h, d, 16, torch.float16)
    c.md.seq_lens_cpu = [1] * len(seqs)
    cells = 5 * -(-long // 384)
    assert 0 < _workspace(c) < cells * h * (d + 2) * 4
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128])
def test_column_ranges_that_outgrow_the_workspace(d):
    hq, hkv = 64, 4
    seqs = [2000] * 10 + [50] * 10 + [30] * 84
    ql = [5] * 20 + [1] * 4 + [0] * 80
    c = _case(seqs, ql, hq, hkv, d, 16, torch.bfloat16)
    c.md.query_lens_cpu = [1] * 100 + [2] * 4
    cells = 10 * 5 * -(-2000 // 256)
    decode = 2048 // hkv
    assert 0 < _workspace(c) < (cells + decode) * hq * (d + 2) * 4
    _check(_run(c), c)


@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("ql", [1, 40])
def test_values_of_v_far_beyond_float16(d, ql):
    """bfloat16 rows of V with a scale above 2^104: 2^24 times it is no float32.  The header's
    bound holds here, 1.7e32 * 40 < 2^113."""
    n, hkv = 40, 2
    c = _case([n], [ql], 4, hkv, d, 16, torch.bfloat16)
    x = torch.rand(n, hkv, d, generator=_g(3)) * 3.4e32 - 1.7e32
    x[..., 0], x[..., 1] = -1.7e32, 1.7e32
    rows = kv4.quantise_rows(x, torch.bfloat16)
    assert (rows[1].float() > 2.0 ** 104).all()
    slots = [int(c.md.block_tables[0, p // 16]) * 16 + p % 16 for p in range(n)]
    kv4.put_rows(c.vc, slots, *rows, is_v=True)
    c.kv[0] = (c.kv[0][0], rows)
    _check(_run(c), c)


def test_rope_write_without_query_heads_is_refused():
    """Its K and V would be left unwritten."""
    c = Int4PagedKVCache(2, 16, 1, 2, 64, torch.float16, DEV)
    x = torch.ones(3, 2, 64, dtype=torch.float16, device=DEV)
    with pytest.raises(ValueError):
        rope_reshape_and_cache_int4(x[:, :0], x, x, x[:, 0], x[:, 0], c.k_cache[0], c.v_cache[0],
                                    torch.arange(3, device=DEV))


@pytest.mark.parametrize("d", [64, 128, 24])
def test_a_replay_of_a_shorter_batch_leaves_zeros_behind_its_last_row(d):
    """The host's offsets at capture cover every row; those of a later replay need not."""
    full = _case([40, 20], [30, 3], 4, 2, d, 16, torch.float16)
    q, kc, vc, md = _graph_case(full)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged_attention_int4(q, kc, vc, md, full.scale)
    stream.synchronize()
    g = torch.cuda.CUDAGraph()
    with graph_capture(g, stream):
        out = paged_attention_int4(q, kc, vc, md, full.scale)
    for ql in ([30, 3], [20, 1], [30, 3], [0, 2], [1, 20]):
        part = dataclasses.replace(full, q=full.q[:sum(ql)], query_lens=ql)
        md.query_start_loc.copy_(torch.tensor([0, ql[0], sum(ql)], dtype=md.query_start_loc.dtype))
        g.replay()
        _check(out[:sum(ql)], part, what=str(ql))
        assert (out[sum(ql):] == 0).all(), ql
