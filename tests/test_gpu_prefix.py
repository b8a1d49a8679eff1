"""Decode attention of a batch behind a shared prefix on the GPU, 16-bit and 8-bit caches, against 64-bit references."""
import math

import pytest
import torch

from kvq_util import CODES, DTYPES, SCALE, check_attention, laid, random_cache
from topk_attn_amd import _lib as L, ops
from util import announce

pytestmark = pytest.mark.gpu

KINDS = [(d, f) for d in DTYPES for f in ("16bit", "e4m3", "int8")]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _source(gen, shape, dtype, fmt, layout):
    """What PrefixDecodePlan takes for [B,N,H,128] rows, and the rows in 64 bits."""
    if fmt == "16bit":
        k, v = ((torch.randn(shape, generator=gen) * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen))).to(DTYPES[dtype]) for _ in range(2))
        return (laid(k, layout), laid(v, layout)), k.double(), v.double()
    held = [random_cache(gen, shape, fmt) for _ in range(2)]
    cache = ops.QuantCache(laid(held[0][0], layout), laid(held[1][0], layout), laid(held[0][1], "heads"), laid(held[1][1], "heads"))
    return cache, *(c.float().double() * s.double()[..., None] for c, s in held)


def _as_prefix(source):
    """[1,P,H,128] as the shared [P,H,128] form."""
    if isinstance(source, tuple):
        return source[0][0], source[1][0]
    return ops.QuantCache(source.k_codes[0], source.v_codes[0], source.k_scale[0], source.v_scale[0])


def _check(out, lse, q, pre, suf, length, G, dtype, fmt):
    B, H = q.shape[0], q.shape[1] // G
    none = torch.zeros((0, 128), dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            n = min(max(length[b], 0), suf[0].shape[1]) if suf else 0
            k, v = (torch.cat([pre[i][0, :, h] if pre else none, suf[i][b, :n, h] if suf else none]) for i in range(2))
            qs = slice(h * G, (h + 1) * G)
            check_attention(out[b, qs], None if lse is None else lse[b, qs], q[b, qs], k, v, out.dtype, fmt == "16bit" or dtype == "f16")


@pytest.mark.parametrize("dtype,fmt", KINDS)
@pytest.mark.parametrize("B,H,G,P,S,layout", [(1, 1, 1, 1, 1, "tokens"), (2, 2, 4, 31, 5, "heads"), (5, 1, 4, 200, 33, "gaps"),
                                              (9, 2, 2, 257, 40, "tokens"), (6, 1, 8, 1000, 130, "heads"), (17, 1, 4, 129, 3, "tokens"),
                                              (33, 1, 8, 160, 2, "heads")])
def test_prefix(dtype, fmt, B, H, G, P, S, layout):
    announce("prefix %s %s B%d H%d G%d P%d S%d %s" % (dtype, fmt, B, H, G, P, S, layout))
    gen = torch.Generator().manual_seed(B * P)
    pre, kp, vp = _source(gen, (1, P, H, 128), dtype, fmt, layout)
    suf, ks, vs = _source(gen, (B, S, H, 128), dtype, fmt, layout)
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    length = [(S, 0, 1, S // 2, S + 3)[b % 5] for b in range(B)]
    out, lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), suf, SCALE, G, suffix_len=_i32(length), return_lse=True)
    _check(out, lse, q, (kp, vp), (ks, vs), length, G, dtype, fmt)
    if B <= 6:
        for splits in (1, 3):
            out, lse = ops.prefix_decode(q.cuda(), pre, suf, SCALE, G, suffix_len=_i32(length), num_splits=splits, return_lse=True)
            _check(out, lse, q, (kp, vp), (ks, vs), length, G, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", KINDS)
@pytest.mark.parametrize("B,H,G,P,S", [(3, 2, 4, 600, 20), (7, 1, 4, 700, 40), (12, 1, 4, 900, 33), (24, 1, 4, 1100, 9), (40, 1, 8, 1300, 270),
                                       (130, 1, 1, 513, 1), (64, 1, 2, 384, 7)])
def test_prefix_blocks_of_query_rows(dtype, fmt, B, H, G, P, S):
    """Each form of the shared part (12, 28, 48, 96, 320, 130, 128 query rows of a head), several tiles of every wave."""
    announce("prefix blocks %s %s B%d H%d G%d P%d S%d" % (dtype, fmt, B, H, G, P, S))
    gen = torch.Generator().manual_seed(B * P + 1)
    pre, kp, vp = _source(gen, (1, P, H, 128), dtype, fmt, "heads")
    suf, ks, vs = _source(gen, (B, S, H, 128), dtype, fmt, "tokens")
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    length = [(S, 0, 1, S // 2)[b % 4] for b in range(B)]
    for splits in (0, 1, 2):
        out, lse = ops.prefix_decode(q.cuda(), pre, suf, SCALE, G, suffix_len=_i32(length), num_splits=splits, return_lse=True)
        _check(out, lse, q, (kp, vp), (ks, vs), length, G, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", [k for k in KINDS if k[1] != "16bit"])
@pytest.mark.parametrize("B", [2, 20, 40])
def test_prefix_scales_far_apart(dtype, fmt, B):
    """Value scales of a shared prefix that differ by 2^60, also between the tiles that share operands; NaN rows stay visible."""
    H, G, P = 1, 8, 900
    gen = torch.Generator().manual_seed(19)
    pre, kp, vp = _source(gen, (1, P, H, 128), dtype, fmt, "heads")
    far = torch.exp2(torch.randint(-50, 11, (1, P, H), generator=gen).float())
    far[:, 300:600] = torch.exp2(torch.tensor(-60.0))
    pre.v_scale.mul_(far.cuda())
    vp = vp * far.double()[..., None]
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    announce("prefix far scales %s %s B%d" % (dtype, fmt, B))
    out, lse = ops.prefix_decode(q.cuda(), pre, None, SCALE, G, out_dtype=torch.bfloat16, return_lse=True)
    _check(out, lse, q, (kp, vp), None, [0] * B, G, dtype, fmt)
    pre.v_scale[0, 700] = math.nan
    out, lse = ops.prefix_decode(q.cuda(), pre, None, SCALE, G, return_lse=True)
    assert torch.isnan(out).all() and torch.isfinite(lse).all()
    pre.k_scale[0, 5] = math.nan
    assert torch.isnan(ops.prefix_decode(q.cuda(), pre, None, SCALE, G, return_lse=True)[1]).all()


@pytest.mark.parametrize("dtype,fmt", KINDS)
def test_prefix_alone_and_suffix_alone(dtype, fmt):
    B, H, G = 4, 2, 2
    gen = torch.Generator().manual_seed(2)
    pre, kp, vp = _source(gen, (1, 100, H, 128), dtype, fmt, "tokens")
    suf, ks, vs = _source(gen, (B, 50, H, 128), dtype, fmt, "heads")
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    length = [50, 0, 1, 32]
    announce("prefix alone %s %s" % (dtype, fmt))
    out, lse = ops.prefix_decode(q.cuda(), pre, None, SCALE, G, return_lse=True)
    _check(out, lse, q, (kp, vp), None, length, G, dtype, fmt)
    out, lse = ops.prefix_decode(q.cuda(), None, suf, SCALE, G, suffix_len=_i32(length), return_lse=True)
    _check(out, lse, q, None, (ks, vs), length, G, dtype, fmt)
    out = ops.prefix_decode(q.cuda(), None, suf, SCALE, G)
    _check(out, None, q, None, (ks, vs), [50] * B, G, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", KINDS)
def test_masked_places_hold_anything(dtype, fmt):
    """NaN and infinities in the rows behind a suffix's length change nothing."""
    B, H, G = 3, 2, 4
    gen = torch.Generator().manual_seed(7)
    pre, _, _ = _source(gen, (1, 490, H, 128), dtype, fmt, "tokens")
    suf, _, _ = _source(gen, (B, 70, H, 128), dtype, fmt, "heads")
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype]).cuda()
    length = [70, 0, 37]
    announce("prefix masked %s %s" % (dtype, fmt))
    clean = ops.prefix_decode(q, pre, suf, SCALE, G, suffix_len=_i32(length))
    for b in range(B):
        for t in (suf if fmt == "16bit" else (suf.k_scale, suf.v_scale)):
            t[b, length[b]:] = math.nan if b == 2 else math.inf
    assert torch.equal(clean, ops.prefix_decode(q, pre, suf, SCALE, G, suffix_len=_i32(length)))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_extreme_16bit_rows(dtype):
    """Logits of -infinity for every key but one, and the largest values of the type."""
    B, H, G, P = 2, 1, 2, 64
    dt = DTYPES[dtype]
    k = torch.zeros((1, P, H, 128), dtype=dt)
    v = torch.full((1, P, H, 128), torch.finfo(dt).max, dtype=dt)
    q = torch.ones((B, H * G, 128), dtype=dt)
    k[0, :, 0, 0] = -math.inf
    k[0, 41] = 1.0
    v[0, 41] = -2.0
    announce("prefix extremes %s" % dtype)
    out, lse = ops.prefix_decode(q.cuda(), (k.cuda(), v.cuda()), None, SCALE, G, return_lse=True)
    assert (out == -2.0).all() and torch.allclose(lse.cpu(), torch.full((B, 2), 128 * SCALE), rtol=1e-6)
    k[0, 41] = -math.inf                    # nothing but -infinity: no weight anywhere, like a row without keys
    out, lse = ops.prefix_decode(q.cuda(), (k.cuda(), v.cuda()), None, SCALE, G, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    k.zero_()                               # equal weights over the largest numbers: their mean
    v.fill_(torch.finfo(dt).max)
    out = ops.prefix_decode(q.cuda(), (k.cuda(), v.cuda()), None, SCALE, G)
    assert (out == torch.finfo(dt).max).all()


def test_equals_attention_over_the_whole():
    """Prefix and suffix of an 8-bit cache against the decode over one cache that holds both, within both bounds."""
    B, H, G, P, S = 3, 2, 4, 500, 60
    gen = torch.Generator().manual_seed(17)
    pre, kp, vp = _source(gen, (1, P, H, 128), "bf16", "int8", "heads")
    suf, ks, vs = _source(gen, (B, S, H, 128), "bf16", "int8", "heads")
    q = torch.randn((B, H * G, 128), generator=gen).bfloat16()
    whole = ops.QuantCache(*(torch.cat([getattr(pre, n).expand(B, *getattr(pre, n).shape[1:]), getattr(suf, n)], 1).contiguous()
                             for n in ("k_codes", "v_codes", "k_scale", "v_scale")))
    length = [60, 0, 31]
    announce("prefix and whole")
    a = ops.prefix_decode(q.cuda(), pre, suf, SCALE, G, suffix_len=_i32(length), return_lse=True)
    b = ops.kvq_flash_decode(q.cuda(), whole, SCALE, G, kv_len=_i32([P + n for n in length]), return_lse=True)
    for out, lse in (a, b):
        _check(out, lse, q, (kp, vp), (ks, vs), length, G, "bf16", "int8")


@pytest.mark.parametrize("fmt", ["16bit", "int8"])
@pytest.mark.parametrize("B,G", [(5, 4), (19, 8)])
def test_graph_replays(fmt, B, G):
    """Two captured graphs and eager calls in turn: every replay gives what an eager call gives."""
    H = 2
    gen = torch.Generator().manual_seed(23)
    pre, _, _ = _source(gen, (1, 2000, H, 128), "bf16", fmt, "tokens")
    suf, _, _ = _source(gen, (B, 100, H, 128), "bf16", fmt, "heads")
    length = _i32([(100, 0, 50, 1, 99)[b % 5] for b in range(B)])
    qs = [torch.randn((B, H * G, 128), generator=gen).bfloat16().cuda() for _ in range(2)]
    plans = [ops.PrefixDecodePlan(q, pre, suf, SCALE, G, suffix_len=length, return_lse=True) for q in qs]
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    announce("prefix graphs %s B%d" % (fmt, B))
    torch.cuda.synchronize()
    for g, p in zip(graphs, plans):
        with torch.cuda.graph(g):
            p.run()
    for step in range(4):
        for q in qs:
            q.copy_(torch.randn(q.shape, generator=gen))
        for g in graphs:
            g.replay()
        want = [ops.prefix_decode(q, pre, suf, SCALE, G, suffix_len=length, return_lse=True) for q in qs]
        torch.cuda.synchronize()
        for p, (out, lse) in zip(plans, want):
            assert torch.equal(p.out, out) and torch.equal(p.lse, lse)
        length.sub_(1).clamp_(min=0)


def test_offsets_beyond_32_bits():
    """A prefix whose last rows lie beyond 4 GiB."""
    P, stride = 300, 1 << 23
    gen = torch.Generator().manual_seed(8)
    k, v = (torch.randn((1, P, 1, 128), generator=gen).half() for _ in range(2))
    far = []
    for x in (k, v):
        t = torch.zeros((P * stride,), dtype=torch.float16, device="cuda").as_strided((P, 1, 128), (stride, 128, 1))
        t.copy_(x[0])
        far.append(t)
    q = torch.randn((2, 4, 128), generator=gen).half()
    announce("prefix far offsets")
    out, lse = ops.prefix_decode(q.cuda(), tuple(far), None, SCALE, 4, return_lse=True)
    _check(out, lse, q, (k.double(), v.double()), None, [0, 0], 4, "f16", "16bit")


BLOCKS = [(4, 4), (8, 4), (16, 4), (16, 8), (40, 8)]      # query rows of a head: 16, 32, 64, 128 and more


@pytest.mark.parametrize("fmt", ["16bit", "e4m3", "int8"])
@pytest.mark.parametrize("B,G", BLOCKS)
def test_a_bad_query_stays_alone(fmt, B, G):
    """A query with a NaN or an infinity makes its own row NaN and no other row of its block."""
    gen = torch.Generator().manual_seed(31)
    pre, kp, vp = _source(gen, (1, 400, 1, 128), "bf16", fmt, "heads")
    suf, ks, vs = _source(gen, (B, 20, 1, 128), "bf16", fmt, "tokens")
    q = torch.randn((B, G, 128), generator=gen).bfloat16()
    announce("prefix bad query %s B%d G%d" % (fmt, B, G))
    clean, clean_lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), suf, SCALE, G, return_lse=True)
    _check(clean, clean_lse, q, (kp, vp), (ks, vs), [20] * B, G, "bf16", fmt)
    bad = q.clone()
    bad[1, 2, 5], bad[B - 1, G - 1, 100] = math.nan, math.inf
    out, lse = ops.prefix_decode(bad.cuda(), _as_prefix(pre), suf, SCALE, G, return_lse=True)
    hit = torch.zeros((B, G), dtype=torch.bool)
    hit[1, 2] = hit[B - 1, G - 1] = True
    hit = hit.cuda()
    assert torch.isnan(out[hit]).all() and torch.isnan(lse[hit]).all()
    _check(torch.where(hit[..., None], clean, out), torch.where(hit, clean_lse, lse), q, (kp, vp), (ks, vs), [20] * B, G, "bf16", fmt)


@pytest.mark.parametrize("dtype,fmt", KINDS)
@pytest.mark.parametrize("B,G", BLOCKS)
def test_prefix_any_number_of_splits(dtype, fmt, B, G):
    """One split, two and the most there may be; the scales of some value rows negative."""
    P = 1500
    gen = torch.Generator().manual_seed(37)
    pre, kp, vp = _source(gen, (1, P, 1, 128), dtype, fmt, "heads")
    if fmt != "16bit":
        pre.v_scale[:, ::3] *= -1
        vp[:, ::3] *= -1
    q = torch.randn((B, G, 128), generator=gen).to(DTYPES[dtype])
    announce("prefix splits %s %s B%d G%d" % (dtype, fmt, B, G))
    for splits in (1, 2, 512):
        out, lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), None, SCALE, G, num_splits=splits, return_lse=True)
        _check(out, lse, q, (kp, vp), None, [0] * B, G, dtype, fmt)


@pytest.mark.parametrize("dtype,fmt", KINDS)
@pytest.mark.parametrize("B,H,G,P,S", [(17, 16, 8, 300, 40), (65, 4, 2, 1100, 129), (130, 2, 1, 500, 1), (33, 8, 4, 290, 260)])
def test_many_short_suffixes(dtype, fmt, B, H, G, P, S):
    """More than 128 query rows of a head and 256 suffixes or more, of every length: empty ones, whole ones, and one that holds
    NaN behind its end."""
    announce("prefix many suffixes %s %s B%d H%d G%d P%d S%d" % (dtype, fmt, B, H, G, P, S))
    gen = torch.Generator().manual_seed(P + S)
    pre, kp, vp = _source(gen, (1, P, H, 128), dtype, fmt, "heads")
    suf, ks, vs = _source(gen, (B, S, H, 128), dtype, fmt, "tokens")
    length = [(S, 0, 1, S // 2, S - 1)[b % 5] for b in range(B)]
    for b in range(B):
        for x in (suf[0], suf[1]) if fmt == "16bit" else (suf.k_scale, suf.v_scale):
            x[b, length[b]:] = math.nan
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    for splits in (0, 1):
        out, lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), suf, SCALE, G, suffix_len=_i32(length), num_splits=splits, return_lse=True)
        some = [0, 1, 2, 3, B - 1]
        _check(out[some], lse[some], q[some], (kp, vp), (ks[some], vs[some]), [length[b] for b in some], G, dtype, fmt)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()


def test_many_short_suffixes_in_a_graph():
    """The form of many short suffixes captured before any eager call of its shape, replayed over changing queries and lengths."""
    B, H, G, P, S = 33, 8, 8, 700, 50
    gen = torch.Generator().manual_seed(41)
    pre, _, _ = _source(gen, (1, P, H, 128), "bf16", "e4m3", "heads")
    suf, _, _ = _source(gen, (B, S, H, 128), "bf16", "e4m3", "heads")
    q = torch.randn((B, H * G, 128), generator=gen).bfloat16().cuda()
    length = _i32([b % (S + 1) for b in range(B)])
    plan = ops.PrefixDecodePlan(q, pre, suf, SCALE, G, suffix_len=length, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    announce("prefix many suffixes graph")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan.run()
    for step in range(4):
        q.copy_(torch.randn(q.shape, generator=gen))
        graph.replay()
        out, lse = ops.prefix_decode(q, pre, suf, SCALE, G, suffix_len=length, return_lse=True)
        torch.cuda.synchronize()
        assert torch.equal(plan.out, out) and torch.equal(plan.lse, lse)
        length.sub_(7).clamp_(min=0)


@pytest.fixture(params=[1, 2, 4, 8, 16])
def row_tiles(request):
    """Blocks of 16 times as many query rows, whatever the call would choose."""
    assert L.lib().tka_kvq_test_row_tiles(request.param) == 0
    yield request.param
    assert L.lib().tka_kvq_test_row_tiles(0) == 0


def _kinds_of(row_tiles):
    return [(d, f) for d, f in KINDS if f != "16bit" or row_tiles <= 4]


@pytest.mark.parametrize("B,H,G,P,S,layout", [(1, 1, 1, 1, 1, "tokens"), (5, 2, 4, 31, 3, "heads"), (9, 1, 8, 161, 40, "gaps"), (19, 2, 8, 700, 33, "heads"),
                                              (40, 1, 8, 1301, 270, "tokens"), (65, 4, 4, 260, 30, "heads")])
def test_every_block_size(row_tiles, B, H, G, P, S, layout):
    """Blocks larger than the call, several blocks with a last one that is cut, prefixes shorter than a tile and cut ones."""
    for dtype, fmt in _kinds_of(row_tiles):
        announce("prefix blocks of %d: %s %s B%d H%d G%d P%d S%d %s" % (16 * row_tiles, dtype, fmt, B, H, G, P, S, layout))
        gen = torch.Generator().manual_seed(B + P)
        pre, kp, vp = _source(gen, (1, P, H, 128), dtype, fmt, layout)
        suf, ks, vs = _source(gen, (B, S, H, 128), dtype, fmt, layout)
        q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
        length = [(S, 0, 1, S // 2, S + 3)[b % 5] for b in range(B)]
        out, lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), suf, SCALE, G, suffix_len=_i32(length), return_lse=True)
        _check(out, lse, q, (kp, vp), (ks, vs), length, G, dtype, fmt)


def test_every_block_size_where_it_can_go_wrong(row_tiles):
    """The cases of the tests above with this block size: scales far apart, places that are masked, bad queries, any number of
    splits, prefix or suffix alone, many short suffixes, replays."""
    for dtype, fmt in _kinds_of(row_tiles):
        if fmt != "16bit":
            test_prefix_scales_far_apart(dtype, fmt, 20)
        test_masked_places_hold_anything(dtype, fmt)
        test_prefix_alone_and_suffix_alone(dtype, fmt)
        test_prefix_any_number_of_splits(dtype, fmt, 40, 8)
        test_many_short_suffixes(dtype, fmt, 33, 8, 4, 290, 260)
        if dtype == "bf16":
            test_a_bad_query_stays_alone(fmt, 19, 8)
    for dtype in DTYPES:
        test_extreme_16bit_rows(dtype)
    test_graph_replays("int8", 19, 8)
    test_many_short_suffixes_in_a_graph()


@pytest.mark.parametrize("fmt,B,G,P", [("16bit", 3, 8, 40000), ("16bit", 40, 8, 60000), ("e4m3", 6, 8, 60000), ("int8", 40, 4, 200000), ("e4m3", 64, 8, 60000),
                                       ("e4m3", 32, 4, 380000)])
def test_the_blocks_that_long_prefixes_choose(fmt, B, G, P):
    """Sizes at which the call itself takes blocks of 32, 64, 128 and 256 query rows; the output of a few entries is checked."""
    announce("prefix long %s B%d G%d P%d" % (fmt, B, G, P))
    gen = torch.Generator().manual_seed(P)
    pre, kp, vp = _source(gen, (1, P, 1, 128), "bf16", fmt, "heads")
    suf, ks, vs = _source(gen, (B, 40, 1, 128), "bf16", fmt, "heads")
    q = torch.randn((B, G, 128), generator=gen).bfloat16()
    out, lse = ops.prefix_decode(q.cuda(), _as_prefix(pre), suf, SCALE, G, return_lse=True)
    some = [0, B // 2, B - 1]
    _check(out[some], lse[some], q[some], (kp, vp), (ks[some], vs[some]), [40] * 3, G, "bf16", fmt)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
