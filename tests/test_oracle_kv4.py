"""The 4-bit cache's oracle, pinned on the CPU, and what the product refuses
without touching a GPU."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import nanoserve_amd
from nanoserve_amd import Int4PagedKVCache, _lib
from nanoserve_amd.attention import AttentionMetadata
from nanoserve_amd.kv4 import kv4_bytes_per_token, kv4_shape
from oracle import kv4

DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("spread,shift", [(1.0, 0.0), (3.0, 20.0), (1e-3, -1.0)])
def test_stored_rows_are_within_half_a_step(dtype, spread, shift):
    x = (torch.randn(50, 2, 64, generator=torch.Generator().manual_seed(0)) * spread + shift).to(dtype).float()
    codes, s, b = kv4.quantise_rows(x, dtype)
    assert codes.max() <= 15 and codes.dtype == torch.uint8
    err = (kv4.stored_values(codes, s, b) - x.double()).abs()
    # Half a step; a scale rounded down leaves the top code short by 15 of its
    # roundings, and a float32 quotient at a tie may fall on either side.
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal  # below it a scale rounds by an absolute step
    assert (err <= s.double() * (0.5 + 15 * half + 1e-5) + 15 * tiny * half).all()
    # The minimum is a value of the dtype, so it is stored exactly.
    assert torch.equal(b.float(), x.amin(-1, keepdim=True))


def test_constant_single_and_non_finite_rows():
    x = torch.full((5, 1, 8), 2.5)
    x[1, 0, 3] = float("nan")
    x[2, 0, 0] = float("inf")
    x[3, 0, 7] = -float("inf")
    x[4] = 0.0
    codes, s, b = kv4.quantise_rows(x, torch.float16)
    assert (codes == 0).all() and (s == 0).all()
    assert torch.equal(torch.isnan(b[:, 0, 0]), torch.tensor([False, True, True, True, False]))
    assert b[0, 0, 0] == 2.5 and b[4, 0, 0] == 0


@pytest.mark.parametrize("is_v", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_records_round_trip_and_rows_do_not_touch_each_other(dtype, is_v):
    g = torch.Generator().manual_seed(1)
    nb, heads, bs, d = 3, 2, 8, 24
    cache = torch.zeros(nb, heads, bs, d // 2 + 4, dtype=torch.uint8)
    slots = torch.randperm(nb * bs, generator=g).tolist()
    rows = kv4.quantise_rows(torch.randn(nb * bs, heads, d, generator=g), dtype)
    for i in range(0, nb * bs, 5):  # in several writes
        kv4.put_rows(cache, slots[i:i + 5], *(x[i:i + 5] for x in rows), is_v)
    for a, b in zip(kv4.get_rows(cache, slots, dtype, is_v), rows):
        assert torch.equal(a, b)
    before = cache.clone()
    kv4.put_rows(cache, [-1, nb * bs], *(x[:2] for x in rows), is_v)
    assert torch.equal(cache, before)


def test_every_byte_of_a_record_belongs_to_one_row():
    nb, heads, bs, d = 1, 1, 4, 16
    for is_v in (False, True):
        owner = np.zeros(bs * (d // 2 + 4), int)
        for t in range(bs):
            cache = torch.zeros(nb, heads, bs, d // 2 + 4, dtype=torch.uint8)
            par = torch.full((1, 1, 1), -1, dtype=torch.int16).view(torch.float16)
            kv4.put_rows(cache, [t], torch.full((1, 1, d), 15, dtype=torch.uint8), par, par, is_v)
            owner += (cache.view(-1).numpy() != 0)
        assert (owner == 1).all()


def test_attention_closed_forms():
    g = torch.Generator().manual_seed(2)
    d, n = 16, 5
    rows = kv4.quantise_rows(torch.randn(n, 1, d, generator=g), torch.float16)
    q = torch.randn(n, 2, d, generator=g)
    out, _, _ = kv4.attention_ref(q, [(rows, rows)], [n], [n], 0.3)
    values = kv4.stored_values(*rows)[:, 0]
    assert torch.allclose(out[0, 0], values[0], atol=1e-12)  # one key
    zero, _, _ = kv4.attention_ref(torch.zeros_like(q), [(rows, rows)], [n], [n], 0.3)
    assert torch.allclose(zero[4, 1], values.mean(0), atol=1e-12)  # equal weights
    # A scalar softmax of the last row.
    w = [math.exp(0.3 * sum(float(a) * float(b) for a, b in zip(q[4, 1], k))) for k in values]
    want = sum(a * k for a, k in zip(w, values)) / sum(w)
    assert torch.allclose(out[4, 1], want, atol=1e-12)
    # More query rows than keys: the first rows see none.
    short, _, _ = kv4.attention_ref(q, [(rows, rows)], [3], [n], 0.3)
    assert (short[:2] == 0).all() and torch.allclose(short[2, 0], values[0], atol=1e-12)


def test_the_cache_object_and_its_bytes():
    c = Int4PagedKVCache(4, 16, 3, 2, 64, torch.bfloat16, "cpu")
    assert len(c.k_cache) == 3 and c.k_cache[0].shape == (4, 2, 16, 36) and c.capacity_tokens == 64
    assert kv4_shape(c.v_cache[1]) == (4, 2, 16, 64)
    assert c.num_bytes == 64 * kv4_bytes_per_token(3, 2, 64)
    for bad in (dict(head_dim=60), dict(head_dim=264), dict(block_size=6)):
        with pytest.raises(ValueError):
            Int4PagedKVCache(**{**dict(num_blocks=1, block_size=16, num_layers=1, num_kv_heads=1, head_dim=64,
                                       dtype=torch.float16, device="cpu"), **bad})
    with pytest.raises(TypeError):
        Int4PagedKVCache(1, 16, 1, 1, 64, torch.float32, "cpu")


def test_the_product_has_no_cpu_path():
    c = Int4PagedKVCache(2, 16, 1, 2, 64, torch.float16, "cpu")
    x, slots = torch.zeros(3, 2, 64, dtype=torch.float16), torch.arange(3)
    md = AttentionMetadata(slots, None, torch.ones(3, dtype=torch.int64), torch.zeros(3, 1, dtype=torch.int64), 1, 1, 3,
                           3, True)
    with pytest.raises(ValueError, match="GPU"):
        c.write(0, x, x, slots)
    with pytest.raises(ValueError, match="GPU"):
        c.read(0, slots)
    with pytest.raises(ValueError, match="GPU"):
        nanoserve_amd.rope_reshape_and_cache_int4(x, x, x, x[:, :1], x[:, :1], c.k_cache[0], c.v_cache[0], slots)
    with pytest.raises(ValueError, match="GPU"):
        nanoserve_amd.paged_attention_int4(x, c.k_cache[0], c.v_cache[0], md, 1.0)
    with pytest.raises(ValueError, match="uint8"):
        nanoserve_amd.paged_attention_int4(x, x[None], x[None], md, 1.0)


OK, INV, UNS = _lib.NS_OK, _lib.NS_ERR_INVALID_ARG, _lib.NS_ERR_UNSUPPORTED


def _write_args(**over):
    a = dict(key=16, value=16, kst=128, ksh=64, vst=128, vsh=64, kc=16, vc=16, slots=16, s64=1,
             T=4, Hkv=2, D=64, bs=16, nb=8, dtype=_lib.NS_DTYPE_F16, stream=None)
    a.update(over)
    return list(a.values())


WRITE_BAD = [(dict(key=None), INV), (dict(vc=None), INV), (dict(slots=None), INV), (dict(T=-1), INV),
             (dict(Hkv=0), INV), (dict(D=0), INV), (dict(nb=0), INV), (dict(D=60), UNS), (dict(D=264), UNS),
             (dict(bs=6), UNS), (dict(dtype=_lib.NS_DTYPE_F32), UNS), (dict(kc=24), INV), (dict(key=17), INV),
             (dict(slots=20), INV)]


@pytest.mark.parametrize("over,code", WRITE_BAD)
def test_write_rejects_bad_arguments(over, code):
    assert _lib.load().ns_reshape_and_cache_int4(*_write_args(**over)) == code


@pytest.mark.parametrize("over,code", WRITE_BAD + [
    (dict(qo=None), INV), (dict(q=None), INV), (dict(cos=None), INV), (dict(sin=None), INV), (dict(Hq=0), INV),
    (dict(cos=17), INV)])
def test_rope_write_rejects_bad_arguments(over, code):
    a = dict(qo=16, q=16, qst=896, qsh=64, key=16, kst=128, ksh=64, value=16, vst=128, vsh=64, cos=16, sin=16, cst=64,
             kc=16, vc=16, slots=16, s64=1, T=4, Hq=14, Hkv=2, D=64, bs=16, nb=8, dtype=_lib.NS_DTYPE_F16, stream=None)
    a.update(over)
    assert _lib.load().ns_rope_reshape_and_cache_int4(*a.values()) == code


@pytest.mark.parametrize("over,code", [
    (dict(ko=None), INV), (dict(vo=24), INV), (dict(slots=None), INV), (dict(T=-1), INV), (dict(Hkv=0), INV),
    (dict(D=60), UNS), (dict(bs=6), UNS), (dict(dtype=7), UNS), (dict(vc=8), INV)])
def test_gather_rejects_bad_arguments(over, code):
    a = dict(ko=16, vo=16, kc=16, vc=16, slots=16, s64=1, T=4, Hkv=2, D=64, bs=16, nb=8, dtype=_lib.NS_DTYPE_F16,
             stream=None)
    a.update(over)
    assert _lib.load().ns_gather_cache_int4(*a.values()) == code


def _attend_args(**over):
    a = dict(out=16, query=16, kc=16, vc=16, bt=16, bt_stride=4, bt_width=4, bt64=0, sl=16, sl64=0, qsl=16, qsl64=0,
             S=2, T=2, maxs=64, decode_only=1, context=0, ones=-1, Hq=14, Hkv=2, D=64, bs=16, nb=32, scale=0.125,
             dtype=_lib.NS_DTYPE_F16, ws=None, ws_bytes=0, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(out=None), INV), (dict(query=None), INV), (dict(kc=None), INV), (dict(bt=None), INV), (dict(sl=None), INV),
    (dict(decode_only=0, qsl=None), INV), (dict(T=3), INV), (dict(Hq=15), INV), (dict(Hkv=0), INV), (dict(nb=0), INV),
    (dict(S=-1), INV), (dict(maxs=-1), INV), (dict(bt_stride=3), INV), (dict(bt_width=0), INV), (dict(out=24), INV),
    (dict(vc=20), INV), (dict(sl=18), INV), (dict(bt=20, bt64=1), INV), (dict(scale=float("nan")), INV),
    (dict(scale=float("inf")), INV), (dict(context=-1), INV), (dict(ones=3), INV), (dict(ones=-2), INV),
    (dict(D=60), UNS), (dict(D=264), UNS), (dict(bs=18), UNS), (dict(dtype=_lib.NS_DTYPE_F32), UNS),
    (dict(T=1 << 28, S=1 << 28), UNS), (dict(maxs=(1 << 30) + 1), UNS),
    (dict(maxs=4096, bt_width=256, bt_stride=256), _lib.NS_ERR_WORKSPACE),
    (dict(maxs=4096, bt_width=256, bt_stride=256, ws=256, ws_bytes=1000), _lib.NS_ERR_WORKSPACE),
    (dict(maxs=4096, bt_width=256, bt_stride=256, ws=128, ws_bytes=1 << 30), _lib.NS_ERR_WORKSPACE),
])
def test_attention_rejects_bad_arguments(over, code):
    assert _lib.load().ns_paged_attention_int4(*_attend_args(**over)) == code


def test_workspace_is_needed_only_where_keys_are_split():
    size = _lib.load().ns_paged_attention_int4_workspace_size
    assert size(32, 14, 2, 64, 16, 1024, 32, 1, 0, -1) == 0
    assert size(32, 14, 2, 64, 16, 8192, 32, 1, 0, -1) > 0
    assert size(32, 14, 2, 24, 16, 8192, 32, 1, 0, -1) == 0       # the plain kernel
    assert size(2, 28, 4, 128, 16, 4000, 8000, 0, 0, -1) == size(2, 28, 4, 128, 16, 4000, 2, 1, 0, -1)
    assert size(2, 28, 4, 128, 16, 4000, 8000, 0, 0, 0) == 0      # whole prompts fill the device
    assert size(1, 28, 4, 128, 16, 16000, 16, 0, 0, 0) > 0        # a short chunk behind a long context
    assert size(2, 13, 2, 64, 16, 4000, 2, 1, 0, -1) == 0 and size(0, 14, 2, 64, 16, 4000, 2, 1, 0, -1) == 0


WIDE_GROUPS = [(hq, 1, d, seqs) for hq in (20, 32) for d in (64, 128)
               for seqs in ((1000, 900), (1000, 40, 2000, 1), (3000, 900, 1, 0, 1500, 2000, 960, 1100))]


@pytest.mark.parametrize("hq,hkv,d,seqs", WIDE_GROUPS)
def test_decode_rows_of_wide_groups_split_their_keys(hq, hkv, d, seqs):
    """More than 16 query heads per KV head: these decode-only calls, which have no
    query offsets, join ranges of keys (test_gpu_kv4 runs them)."""
    for context in (0, sum(seqs)):
        size = _lib.load().ns_paged_attention_int4_workspace_size(len(seqs), hq, hkv, d, 16, max(seqs), len(seqs), 1,
                                                                  context, len(seqs))
        assert size > 0


@pytest.mark.parametrize("hq,hkv,d", [(28, 4, 128), (14, 2, 64), (64, 4, 128), (8, 8, 128), (64, 64, 64)])
def test_partial_results_follow_the_ranges_not_the_longest_context(hq, hkv, d):
    """A split context has at most twice its share of the about 1024 / hkv ranges that a
    device's worth of keys is cut into, and longer queries at most 16384 / hq (row, range)s:
    many short contexts beside a long one cost 8 bytes each."""
    size = _lib.load().ns_paged_attention_int4_workspace_size
    cell = hq * (d + 2) * 4
    decode, chunk = 2048 // hkv * cell, 16384 // hq * cell
    for short, count, long in ((400, 511, 131072), (1000, 63, 131072), (500, 255, 131072), (30, 20000, 32768)):
        n = count + 1
        total = short * count + long
        for context in (total, 0, 1):
            got = size(n, hq, hkv, d, 16, long, n, 1, context, n)
            assert got <= decode + 8 * n + 256
        # The same rows beside a chunk behind the long context, of which the host knows all, the rows or nothing.
        for ql in (3, 16):
            for context, ones in ((total, count), (0, count), (0, -1)):
                got = size(n, hq, hkv, d, 16, long, count + ql, 0, context, ones)
                assert got <= decode + chunk + 16 * n + 512
    # No more than every row in every range, either.
    assert size(2, hq, hkv, d, 16, 1500, 2, 1, 0, 2) <= 2 * 4 * cell + 16 + 256


def test_no_tokens_is_a_no_op():
    lib = _lib.load()
    assert lib.ns_reshape_and_cache_int4(*_write_args(T=0, key=None)) == OK
    assert lib.ns_paged_attention_int4(*_attend_args(S=0, T=0, out=None)) == OK
    assert lib.ns_gather_cache_int4(None, None, None, None, None, 1, 0, 2, 64, 16, 8, _lib.NS_DTYPE_F16, None) == OK
