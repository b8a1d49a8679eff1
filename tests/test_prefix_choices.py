"""Which form tka_prefix_decode takes by itself, asserted through the workspace that it asks for, and each of these forms
against 64 bits; the launch that joins suffixes and partials for every group."""
import ctypes as C

import pytest
import torch

from kvq_util import CODES, DTYPES, SCALE, check_attention
from topk_attn_amd import _lib as L, ops
from util import announce

# format, batch, heads, group, prefix, suffix, sixteens of query rows that the call takes by itself, and those that would ask
# for another workspace (blocks of 32 and 64 query rows over 33 to 64 rows of 8 bits ask for the same)
CHOICES = [("16bit", 40, 1, 4, 16000, 40, 1, (2, 4)), ("16bit", 10, 1, 4, 100000, 40, 2, (1, 4)), ("16bit", 40, 1, 8, 60000, 40, 4, (1, 2)),
           ("e4m3", 25, 1, 4, 25000, 40, 1, (2, 4, 8, 16)), ("int8", 18, 1, 4, 60000, 40, 2, (1, 4, 8, 16)), ("e4m3", 16, 8, 4, 92000, 0, 4, (1, 8)),
           ("int8", 32, 1, 4, 380000, 40, 8, (1, 2, 4, 16)), ("e4m3", 38, 1, 8, 100000, 40, 16, (1, 2, 4, 8)),
           ("e4m3", 64, 8, 8, 8192, 100, 16, (1, 2, 4, 8)), ("int8", 33, 8, 8, 15000, 7, 16, (1, 2, 4, 8))]
JOINS = [("int8", 65, 4, 2, 1100, 129), ("e4m3", 130, 2, 1, 500, 1), ("e4m3", 64, 4, 1, 700, 33), ("int8", 33, 8, 4, 290, 260), ("int8", 17, 16, 8, 300, 40)]
FORMAT = {"16bit": L.TKA_KV_16BIT, "e4m3": L.TKA_KV_E4M3, "int8": L.TKA_KV_INT8}


def _need(args, row_tiles=0):
    assert L.lib().tka_kvq_test_row_tiles(row_tiles) == 0
    try:
        return L.lib().tka_prefix_decode_workspace_bytes(C.byref(args))
    finally:
        assert L.lib().tka_kvq_test_row_tiles(0) == 0


def _args(fmt, B, H, G, P, S):
    """An argument block for the checks alone: none of its pointers is looked at."""
    a = L.PrefixDecodeArgs()
    for c, batch, rows in ((a.prefix, 1, P), (a.suffix, B, S)):
        c.k, c.v, c.format, c.batch, c.num_kv_heads, c.head_dim, c.rows = 0x10000, 0x20000, FORMAT[fmt], batch, H, 128, rows
        c.stride_b, c.stride_n, c.stride_h = H * rows * 128, 128, rows * 128
        if fmt != "16bit":
            c.k_scale, c.v_scale, c.scale_stride_b, c.scale_stride_n, c.scale_stride_h = 0x30000, 0x40000, H * rows, 1, rows
    a.q, a.out, a.dtype, a.out_dtype, a.group, a.scale = 0x50000, 0x60000, L.TKA_BF16, L.TKA_BF16, G, SCALE
    a.q_stride_b = a.out_stride_b = H * G * 128
    return a


def _assert_choice(args, tiles, others):
    assert _need(args) == _need(args, tiles) > 256
    for other in others:
        assert _need(args) != _need(args, other), other


def _assert_join(args):
    """Blocks of 256 query rows whose suffixes are attended to by the joining launch: no partials of theirs in the workspace."""
    alone = L.PrefixDecodeArgs.from_buffer_copy(args)
    alone.suffix.rows = 0
    assert _need(args, 16) == _need(alone, 16) > 256


@pytest.mark.parametrize("fmt,B,H,G,P,S,tiles,others", CHOICES)
def test_choices(fmt, B, H, G, P, S, tiles, others):
    a = _args(fmt, B, H, G, P, S)
    _assert_choice(a, tiles, others)
    if tiles == 16 and H * B >= 256:
        _assert_join(a)


@pytest.mark.parametrize("fmt,B,H,G,P,S", JOINS)
def test_joins(fmt, B, H, G, P, S):
    _assert_join(_args(fmt, B, H, G, P, S))


def _source(gen, shape, dtype, fmt):
    """Rows on the GPU, head by head, any codes but NaN, scales (of 8 bits) of their own; and rows (entry, head) of them in 64 bits."""
    B, N, H, _ = shape
    if fmt == "16bit":
        k, v = (torch.randn((B, H, N, 128), generator=gen, device="cuda").to(DTYPES[dtype]).transpose(1, 2) for _ in range(2))
        return (k, v), lambda b, h, n: (k[b, :n, h].double().cpu(), v[b, :n, h].double().cpu())
    cache = ops.QuantCache.empty(B, N, H, CODES[fmt])
    for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
        x = torch.randint(0, 256, codes.shape, generator=gen, device="cuda", dtype=torch.int32).to(torch.uint8)
        if fmt == "e4m3":
            x = torch.where((x & 0x7F) == 0x7F, torch.zeros_like(x), x)
        codes.view(torch.uint8).copy_(x)
        scale.copy_(torch.exp(0.4 * torch.randn(scale.shape, generator=gen, device="cuda")) / 100)

    def rows(b, h, n):
        return tuple(c.view(torch.uint8)[b, :n, h].cpu().view(c.dtype).float().double() * s[b, :n, h].double().cpu()[:, None]
                     for c, s in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)))
    return cache, rows


def _check_call(fmt, dtype, B, H, G, P, S, seed, check_plan):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pre, pre_rows = _source(gen, (1, P, H, 128), dtype, fmt)
    suf, suf_rows = _source(gen, (B, S, H, 128), dtype, fmt) if S else (None, None)
    q = (0.3 * torch.randn((B, H * G, 128), generator=gen, device="cuda")).to(DTYPES[dtype])
    length = [(S, 0, 1, S // 2, S - 1)[b % 5] for b in range(B)]
    plan = ops.PrefixDecodePlan(q, pre, suf, SCALE, G, suffix_len=torch.tensor(length, dtype=torch.int32, device="cuda") if S else None, return_lse=True)
    check_plan(plan.args)
    plan.run()
    torch.cuda.synchronize()
    out, lse = plan.out.cpu(), plan.lse.cpu()
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    for h in sorted({0, H - 1}):
        kp, vp = pre_rows(0, h, P)
        for b in sorted({0, 1, 2, 3, 4, B // 2, B - 1}):
            k, v = kp, vp
            if S and length[b] > 0:
                ks, vs = suf_rows(b, h, length[b])
                k, v = torch.cat([kp, ks]), torch.cat([vp, vs])
            at = slice(h * G, (h + 1) * G)
            check_attention(out[b, at], lse[b, at], q[b, at].cpu(), k, v, out.dtype, fmt == "16bit" or dtype == "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt,B,H,G,P,S,tiles,others", CHOICES)
def test_what_the_call_chooses(fmt, B, H, G, P, S, tiles, others, dtype):
    announce("prefix choice %s %s B%d H%d G%d P%d S%d" % (dtype, fmt, B, H, G, P, S))
    _check_call(fmt, dtype, B, H, G, P, S, P, lambda a: _assert_choice(a, tiles, others))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt,B,H,G,P,S", JOINS)
def test_joining_launch_of_every_group(fmt, B, H, G, P, S, dtype):
    announce("prefix join %s %s B%d H%d G%d P%d S%d" % (dtype, fmt, B, H, G, P, S))
    assert L.lib().tka_kvq_test_row_tiles(16) == 0
    try:
        _check_call(fmt, dtype, B, H, G, P, S, P + S, lambda a: None)
    finally:
        assert L.lib().tka_kvq_test_row_tiles(0) == 0
