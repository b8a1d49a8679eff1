"""Calls of the 8-bit caches and shared prefixes that their documentation allows: scales in other orders, caches filled far below
their capacity, sources without rows, positions at the ends of 32 bits, empty lists.  Bounds: kvq_util."""
import math

import pytest
import torch

from kvq_util import CODES, DTYPES, SCALE, check_attention, quantise64, random_cache
from topk_attn_amd import _lib as L, ops
from util import announce

pytestmark = pytest.mark.gpu

TYPES = [(d, f) for d in DTYPES for f in CODES]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _interleaved(gen, shape, fmt):
    """Keys and values side by side: codes [B,N,H,2,128] and scales [B,N,H,2], the cache a view of either half."""
    held = [random_cache(gen, shape, fmt) for _ in range(2)]
    codes = torch.stack([c.view(torch.uint8) for c, _ in held], -2).cuda().view(CODES[fmt])
    scale = torch.stack([s for _, s in held], -1).cuda()
    cache = ops.QuantCache(codes[..., 0, :], codes[..., 1, :], scale[..., 0], scale[..., 1])
    return cache, *(c.float().double() * s.double()[..., None] for c, s in held)


def _check(out, lse, q, k, v, dtype, G):
    for h in range(k.shape[1]):
        at = slice(h * G, (h + 1) * G)
        check_attention(out[at], lse[at], q[at], k[:, h], v[:, h], out.dtype, dtype == "f16")


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_interleaved_caches(dtype, fmt):
    """Scales of one head 2 H floats apart: every reader, and the write into such a cache."""
    B, N, H, G = 2, 700, 3, 4
    gen = torch.Generator().manual_seed(2)
    cache, k, v = _interleaved(gen, (B, N, H, 128), fmt)
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    length = [N, 333]
    announce("kvq interleaved %s %s" % (dtype, fmt))
    for splits in (0, 1):
        out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, G, num_splits=splits, kv_len=_i32(length), return_lse=True)
        for b in range(B):
            _check(out[b], lse[b], q[b], k[b, :length[b]], v[b, :length[b]], dtype, G)
    ids = torch.randint(0, 333, (B, H, 100), generator=gen, dtype=torch.int32)
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, G, kv_idx=ids.cuda(), return_lse=True)
    for b in range(B):
        for h in range(H):
            rows, at = ids[b, h].long(), slice(h * G, (h + 1) * G)
            check_attention(out[b, at], lse[b, at], q[b, at], k[b, rows, h], v[b, rows, h], out.dtype, dtype == "f16")
    plain = ops.QuantCache(*(x.contiguous() for x in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale)))
    assert torch.equal(ops.kvq_scores(q.cuda(), cache, SCALE, G), ops.kvq_scores(q.cuda(), plain, SCALE, G))
    assert all(torch.equal(a, b) for a, b in zip(ops.kvq_read(cache, N, dtype=DTYPES[dtype]), ops.kvq_read(plain, N, dtype=DTYPES[dtype])))
    new = [torch.randn((B, 5, H, 128), generator=gen).to(DTYPES[dtype]) for _ in range(2)]
    for c in (cache, plain):
        ops.kvq_write(c, new[0].cuda(), new[1].cuda(), start=_i32([100, 0]))
    for name in ("k_codes", "v_codes", "k_scale", "v_scale"):
        a, b = getattr(cache, name), getattr(plain, name)
        assert torch.equal(a.contiguous().view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("row_tiles", [1, 2, 4, 8, 16])
@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_interleaved_prefix(row_tiles, dtype, fmt):
    B, H, G, P, S = 19, 2, 8, 300, 20
    gen = torch.Generator().manual_seed(3)
    pre, kp, vp = _interleaved(gen, (1, P, H, 128), fmt)
    suf, ks, vs = _interleaved(gen, (B, S, H, 128), fmt)
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    announce("kvq interleaved prefix: blocks of %d, %s %s" % (16 * row_tiles, dtype, fmt))
    assert L.lib().tka_kvq_test_row_tiles(row_tiles) == 0
    try:
        out, lse = ops.prefix_decode(q.cuda(), pre, suf, SCALE, G, suffix_len=_i32([b % (S + 1) for b in range(B)]), return_lse=True)
    finally:
        assert L.lib().tka_kvq_test_row_tiles(0) == 0
    for b in range(B):
        n = b % (S + 1)
        _check(out[b], lse[b], q[b], torch.cat([kp[0], ks[b, :n]]), torch.cat([vp[0], vs[b, :n]]), dtype, G)


@pytest.mark.parametrize("fmt", list(CODES))
@pytest.mark.parametrize("N,splits", [(20000, 0), (20000, 40), (3000, 1024)])
def test_lengths_far_below_the_capacity(fmt, N, splits):
    """Splits are cut for the capacity; sequences of every length from none to some, ending inside the first split, at and just
    behind the edges of others; the rows behind them hold NaN."""
    B, H, G = 8, 2, 2
    gen = torch.Generator().manual_seed(N)
    held = 1600
    cache = ops.QuantCache.empty(B, N, H, CODES[fmt])
    for x in (cache.k_scale, cache.v_scale):
        x.fill_(math.nan)
    new = [torch.randn((B, held, H, 128), generator=gen).bfloat16() for _ in range(2)]
    length = [0, 1, 31, 128, 129, 512, 1279, 1600]
    ops.kvq_write(cache, new[0].cuda(), new[1].cuda(), count=_i32(length))
    k, v = (c * s.double()[..., None] for c, s in (quantise64(x, fmt) for x in new))
    q = torch.randn((B, H * G, 128), generator=gen).bfloat16()
    announce("kvq below capacity %s N%d splits %d" % (fmt, N, splits))
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, G, num_splits=splits, kv_len=_i32(length), return_lse=True)
    for b in range(B):
        _check(out[b], lse[b], q[b], k[b, :length[b]], v[b, :length[b]], "bf16", G)
    scores = ops.kvq_scores(q.cuda(), cache, SCALE, G, kv_len=_i32(length))
    for b in range(B):
        assert torch.isfinite(scores[b, :, :length[b]]).all() and (scores[b, :, length[b]:] == -math.inf).all()


@pytest.mark.parametrize("fmt", ["16bit"] + list(CODES))
def test_sources_without_rows(fmt):
    """Tensors of no rows stand for no prefix or no suffix; a call with neither is refused, as is a cache without rows."""
    B, H, G = 3, 2, 4
    gen = torch.Generator().manual_seed(7)
    if fmt == "16bit":
        whole = tuple(torch.randn((B, 50, H, 128), generator=gen).bfloat16().cuda() for _ in range(2))
        cut = lambda s, n: tuple(x[:, :n] for x in s)   # noqa: E731
        one = lambda s: tuple(x[0] for x in s)          # noqa: E731
    else:
        held = [random_cache(gen, (B, 50, H, 128), fmt) for _ in range(2)]
        whole = ops.QuantCache(held[0][0].cuda(), held[1][0].cuda(), held[0][1].cuda(), held[1][1].cuda())
        cut = lambda s, n: ops.QuantCache(s.k_codes[:, :n], s.v_codes[:, :n], s.k_scale[:, :n], s.v_scale[:, :n])   # noqa: E731
        one = lambda s: ops.QuantCache(s.k_codes[0], s.v_codes[0], s.k_scale[0], s.v_scale[0])                      # noqa: E731
    q = torch.randn((B, H * G, 128), generator=gen).bfloat16().cuda()
    announce("prefix without rows %s" % fmt)
    assert torch.equal(ops.prefix_decode(q, one(cut(whole, 0)), whole, SCALE, G), ops.prefix_decode(q, None, whole, SCALE, G))
    assert torch.equal(ops.prefix_decode(q, one(whole), cut(whole, 0), SCALE, G), ops.prefix_decode(q, one(whole), None, SCALE, G))
    with pytest.raises(L.TkaError):
        ops.prefix_decode(q, one(cut(whole, 0)), cut(whole, 0), SCALE, G)
    if fmt != "16bit":
        with pytest.raises(L.TkaError):
            ops.kvq_flash_decode(q, cut(whole, 0), SCALE, G)
        with pytest.raises(L.TkaError):
            ops.kvq_scores(q, cut(whole, 0), SCALE, G)
        with pytest.raises(ValueError):
            ops.kvq_flash_decode(q, whole, SCALE, G, kv_idx=torch.zeros((B, H, 0), dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("fmt", list(CODES))
def test_positions_at_the_ends_of_32_bits(fmt):
    """Entries that are padding: starts and counts at the ends of their type drop every row and leave the cache as it was."""
    B, T, N, H = 4, 9, 20, 2
    gen = torch.Generator().manual_seed(1)
    cache = ops.QuantCache.empty(B, N, H, CODES[fmt])
    k, v = (torch.randn((B, T, H, 128), generator=gen).half().cuda() for _ in range(2))
    ends = (2 ** 31 - 1, -2 ** 31)
    announce("kvq positions %s" % fmt)
    ops.kvq_write(cache, k, v, start=_i32([ends[0], ends[1], 3, 4]), count=_i32([T, T, ends[1], ends[0]]))
    assert all(int(x.contiguous().view(torch.uint8)[:3].count_nonzero()) == 0 for x in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale))
    assert torch.equal(cache.k_scale[3, 4:4 + T].cpu(), quantise64(k[3].cpu(), fmt)[1])
    got = [torch.full((B, T, H, 128), 3.0, dtype=torch.float16, device="cuda") for _ in range(2)]
    ops.KvqReadPlan(cache, got[0], got[1], start=_i32([ends[0], ends[1], 3, 4]), count=_i32([T, T, ends[1], ends[0]])).run()
    assert all((x[:3] == 3.0).all() and (x[3] != 3.0).any() for x in got)
    q = torch.randn((B, H, 128), generator=gen).half().cuda()
    out, lse = ops.kvq_flash_decode(q, cache, SCALE, 1, kv_len=_i32([ends[1], -1, 0, ends[0]]), return_lse=True)
    assert (out[:3] == 0).all() and (lse[:3] == -math.inf).all() and torch.isfinite(lse[3]).all()


def test_one_plan_made_and_run_on_another_stream():
    """Plans run on the stream that is current when they run, and functions leave nothing on another stream's memory."""
    gen = torch.Generator().manual_seed(5)
    held = [random_cache(gen, (2, 4000, 2, 128), "int8") for _ in range(2)]
    cache = ops.QuantCache(held[0][0].cuda(), held[1][0].cuda(), held[0][1].cuda(), held[1][1].cuda())
    q = torch.randn((2, 8, 128), generator=gen).bfloat16().cuda()
    want = ops.kvq_flash_decode(q, cache, SCALE, 4)
    plan = ops.KvqFlashDecodePlan(q, cache, SCALE, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    announce("kvq plan on a side stream")
    with torch.cuda.stream(side):
        for _ in range(5):
            plan.run()
            got = ops.kvq_flash_decode(q, cache, SCALE, 4)
            assert torch.equal(got, want) and torch.equal(plan.out, want)
