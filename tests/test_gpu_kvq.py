"""8-bit K/V caches on the GPU: writing, reading back, scoring and attending, against 64-bit references."""
import math

import pytest
import torch

from kvq_util import CODES, DTYPES, SCALE, U, check_attention, laid, quantise64, random_cache
from topk_attn_amd import ops
from util import announce

pytestmark = pytest.mark.gpu

TYPES = [(d, f) for d in DTYPES for f in CODES]


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _filled_cache(B, N, H, fmt, layout):
    """A cache whose every byte is a mark: what is not written has to keep it."""
    codes = [laid(torch.full((B, N, H, 128), 0x2A, dtype=torch.uint8).view(CODES[fmt]), layout) for _ in range(2)]
    scales = [laid(torch.full((B, N, H), -7.0), layout) for _ in range(2)]
    return ops.QuantCache(codes[0], codes[1], scales[0], scales[1])


def _as_float(codes):
    return codes.float().cpu() if codes.dtype != torch.int8 else codes.cpu().float()


# ---- write ----------------------------------------------------------------------------------------


def _check_written(cache, k, v, start, count, fmt):
    B, N, H = cache.k_codes.shape[:3]
    T = k.shape[1]
    for codes, scale, x in ((cache.k_codes, cache.k_scale, k), (cache.v_codes, cache.v_scale, v)):
        want_c = torch.full((B, N, H, 128), 0x2A, dtype=torch.uint8).view(CODES[fmt]).float()
        want_s = torch.full((B, N, H), -7.0)
        for b in range(B):
            c, s = quantise64(x[b].cpu(), fmt)
            for t in range(min(max(count[b], 0), T)):
                if 0 <= start[b] + t < N:
                    want_c[b, start[b] + t], want_s[b, start[b] + t] = c[t].float(), s[t]
        assert torch.equal(torch.nan_to_num(scale.cpu(), nan=-1.0), torch.nan_to_num(want_s, nan=-1.0))
        assert torch.equal(_as_float(codes), want_c)


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("B,T,N,H,layout", [(1, 1, 1, 1, "tokens"), (3, 1, 40, 5, "heads"), (2, 7, 9, 3, "gaps"),
                                            (5, 33, 100, 2, "tokens"), (2, 70, 70, 8, "heads")])
def test_write(dtype, fmt, B, T, N, H, layout):
    announce("kvq write %s %s B%d T%d N%d H%d %s" % (dtype, fmt, B, T, N, H, layout))
    gen = torch.Generator().manual_seed(B * 1000 + T)
    k, v = ((torch.randn((B, T, H, 128), generator=gen) * torch.exp(3 * torch.randn((B, T, H, 1), generator=gen))).to(DTYPES[dtype]) for _ in range(2))
    start = [int(torch.randint(0, N - T + 1, (1,), generator=gen)) for _ in range(B)]
    count = [T] * B
    if B >= 2:
        count[1] = 0
    if B >= 5:
        count[2], count[3], start[4] = T // 2, T + 9, N - 1   # a count beyond the rows, rows that leave the cache
    cache = _filled_cache(B, N, H, fmt, layout)
    ops.kvq_write(cache, k.cuda(), v.cuda(), start=_i32(start), count=_i32(count))
    _check_written(cache, k, v, start, count, fmt)


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_write_special_rows(dtype, fmt):
    """Zeros, the smallest and the largest numbers, exact powers, ties, one huge element, infinities and NaN."""
    dt = DTYPES[dtype]
    info = torch.finfo(dt)
    x = torch.zeros((1, 16, 1, 128), dtype=torch.float64)
    x[0, 1, 0, 5] = info.smallest_normal * info.eps          # the smallest subnormal
    x[0, 2, 0, :] = info.max
    x[0, 3, 0, :] = torch.arange(128) - 64
    x[0, 4, 0, :] = (torch.arange(128) - 64) * 7.0 / 4
    x[0, 5, 0, 0], x[0, 5, 0, 1:] = 448.0, torch.linspace(-1, 1, 127).double()
    x[0, 6, 0, 0], x[0, 6, 0, 1:] = 450.0, 13.5
    x[0, 7, 0, 0], x[0, 7, 0, 1:] = -127.0, torch.arange(127) / 2.0      # ties of the whole numbers
    x[0, 8, 0, :] = math.inf
    x[0, 9, 0, 77] = math.nan
    x[0, 10, 0, 3], x[0, 10, 0, 4] = -math.inf, 1.0
    x[0, 11, 0, :] = info.smallest_normal
    x[0, 12, 0, 0], x[0, 12, 0, 1:] = 448.0 * 2.0 ** -4, 2.0 ** -14
    x[0, 13, 0, :] = -0.0
    x[0, 14, 0, :] = torch.arange(128) * 0.0625 + 1
    x = x.to(dt)
    announce("kvq write special %s %s" % (dtype, fmt))
    cache = _filled_cache(1, 16, 1, fmt, "tokens")
    ops.kvq_write(cache, x.cuda(), x.cuda())
    _check_written(cache, x, x, [0], [16], fmt)
    k, _ = ops.kvq_read(cache, 16, dtype=dt)
    assert torch.isnan(k[0, 8:11]).all() and torch.isfinite(k[0, :8]).all() and (k[0, 0] == 0).all()
    assert (k[0, 2] >= info.max * (1 - 2.0 ** -4)).all()      # the largest number may stand for more than there is: it reads as the largest


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_write_strided_inputs(dtype):
    """K and V as views of one fused projection, the sequence between other rows."""
    gen = torch.Generator().manual_seed(5)
    fused = torch.randn((2, 20, 3 * 4, 128), generator=gen).to(DTYPES[dtype]).cuda()
    k, v = fused[:, 3:14, 4:8], fused[:, 3:14, 8:12]
    cache = _filled_cache(2, 30, 4, "int8", "heads")
    announce("kvq write strided")
    ops.kvq_write(cache, k, v, start=_i32([2, -4]))      # (entry 1: four rows in front of the cache are dropped)
    _check_written(cache, k, v, [2, -4], [11, 11], "int8")


# ---- read -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("B,T,N,H,layout", [(1, 1, 1, 1, "tokens"), (3, 50, 64, 3, "heads"), (2, 33, 40, 2, "gaps")])
def test_read(dtype, fmt, B, T, N, H, layout):
    gen = torch.Generator().manual_seed(T)
    held = [random_cache(gen, (B, N, H, 128), fmt, spread=2.0) for _ in range(2)]
    cache = ops.QuantCache(laid(held[0][0], layout), laid(held[1][0], layout), laid(held[0][1], "heads"), laid(held[1][1], "heads"))
    start = [int(torch.randint(0, N - T + 1, (1,), generator=gen)) for _ in range(B)]
    count = [T, 0, T // 2][:B]
    if B == 3:
        start[2] = N - 5        # rows that the cache does not have
    k, v = (torch.full((B, T, H, 128), 3.0, dtype=DTYPES[dtype], device="cuda") for _ in range(2))
    announce("kvq read %s %s B%d T%d %s" % (dtype, fmt, B, T, layout))
    ops.KvqReadPlan(cache, k, v, start=_i32(start), count=_i32(count)).run()
    for got, (codes, scale) in ((k, held[0]), (v, held[1])):
        want = torch.full((B, T, H, 128), 3.0, dtype=DTYPES[dtype])
        for b in range(B):
            for t in range(count[b]):
                if start[b] + t < N:
                    want[b, t] = (codes[b, start[b] + t].float() * scale[b, start[b] + t][:, None]).to(DTYPES[dtype])
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_read_every_code(dtype, fmt):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 2, 1, 128).view(CODES[fmt])
    scale = torch.tensor([0.75, 2.0 ** -9]).view(1, 2, 1)
    cache = ops.QuantCache(codes.cuda(), codes.cuda(), scale.cuda(), scale.cuda())
    announce("kvq read codes")
    k, v = ops.kvq_read(cache, 2, dtype=DTYPES[dtype])
    want = (codes.float() * scale[..., None]).to(DTYPES[dtype])
    for got in (k, v):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=1e9), torch.nan_to_num(want.float(), nan=1e9))


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_round_trip(dtype, fmt):
    """What is read differs from what was written by half a step: 2^-4 of an e4m3 number (or half its smallest step,
    2^-10 of the scale), half a scale of an int8 one, and the rounding to 16 bits."""
    gen = torch.Generator().manual_seed(11)
    x = (torch.randn((2, 40, 3, 128), generator=gen) * 5).to(DTYPES[dtype])
    cache = ops.QuantCache.empty(2, 40, 3, CODES[fmt])
    announce("kvq round trip")
    ops.kvq_write(cache, x.cuda(), x.cuda())
    k, v = ops.kvq_read(cache, 40, dtype=DTYPES[dtype])
    scale = cache.k_scale.double().cpu()[..., None]
    step = 0.5 * scale * (1 + 2 ** -20) if fmt == "int8" else torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)
    bound = step + (x.double().abs() + step) * torch.finfo(DTYPES[dtype]).eps / 2
    assert ((k.double().cpu() - x.double()).abs() <= bound).all() and torch.equal(k, v)


# ---- scores ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("B,H,G,N,layout", [(1, 1, 1, 1, "tokens"), (2, 3, 4, 63, "heads"), (3, 2, 8, 257, "tokens"), (2, 4, 2, 1000, "gaps")])
def test_scores(dtype, fmt, B, H, G, N, layout):
    gen = torch.Generator().manual_seed(N)
    codes, scale = random_cache(gen, (B, N, H, 128), fmt)
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    cache = ops.QuantCache(laid(codes, layout), None, laid(scale, "heads"), None)
    length = [N, 0, N // 2][:B] if B > 1 else [N]
    announce("kvq scores %s %s B%d H%d G%d N%d" % (dtype, fmt, B, H, G, N))
    got = ops.kvq_scores(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length))
    # the canonical order, bit for bit: the codes as 16-bit keys through the scores of 16-bit caches
    dots = ops.gemv_scores(q.cuda(), codes.float().to(DTYPES[dtype]).cuda(), group=G, scale=1.0)
    want = (dots * scale.cuda().transpose(1, 2)) * torch.tensor(SCALE, dtype=torch.float32, device="cuda")
    kd = codes.double() * scale.double()[..., None]
    for b in range(B):
        n = length[b]
        assert torch.equal(got[b, :, :n], want[b, :, :n])
        assert (got[b, :, n:] == -math.inf).all()
        for h in range(H):
            qg = q[b, h * G:(h + 1) * G].double()
            exact = (kd[b, :n, h] @ qg.sum(0)) * SCALE
            bound = (8 + 8 + 4 + 3) * U * SCALE * (kd[b, :n, h].abs() @ qg.abs().sum(0))
            assert ((got[b, h, :n].double().cpu() - exact).abs() <= bound).all()


# ---- decode ---------------------------------------------------------------------------------------


def _decode_case(gen, B, H, G, N, dtype, fmt, layout, spread=0.5):
    held = [random_cache(gen, (B, N, H, 128), fmt, spread) for _ in range(2)]
    q = torch.randn((B, H * G, 128), generator=gen).to(DTYPES[dtype])
    cache = ops.QuantCache(laid(held[0][0], layout), laid(held[1][0], layout), laid(held[0][1], "heads"), laid(held[1][1], "heads"))
    k, v = (c.float().double() * s.double()[..., None] for c, s in held)
    return q, cache, k, v


def _check_decode(out, lse, q, k, v, rows_of, G, dtype):
    B, H = k.shape[0], k.shape[2]
    for b in range(B):
        for h in range(H):
            rows = rows_of(b, h)
            qs = slice(h * G, (h + 1) * G)
            check_attention(out[b, qs], lse[b, qs] if lse is not None else None, q[b, qs], k[b, rows, h], v[b, rows, h], out.dtype, dtype == "f16")


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("B,H,G,N,layout", [(1, 1, 1, 1, "tokens"), (2, 2, 2, 31, "heads"), (6, 2, 4, 129, "gaps"), (3, 1, 8, 700, "tokens"),
                                            (1, 2, 4, 5000, "heads")])
def test_decode_dense(dtype, fmt, B, H, G, N, layout):
    gen = torch.Generator().manual_seed(N + B)
    q, cache, k, v = _decode_case(gen, B, H, G, N, dtype, fmt, layout)
    length = [N, 0, 1, N - 1, N // 2, N + 5][:B]
    announce("kvq decode %s %s B%d H%d G%d N%d %s" % (dtype, fmt, B, H, G, N, layout))
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length), return_lse=True)
    _check_decode(out, lse, q, k, v, lambda b, h: slice(0, min(length[b], N)), G, dtype)
    for splits in (1, 3):
        out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length), num_splits=splits, return_lse=True)
        _check_decode(out, lse, q, k, v, lambda b, h: slice(0, min(length[b], N)), G, dtype)
    if B == 1:
        other = torch.bfloat16 if dtype == "f16" else torch.float16
        out = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, out_dtype=other)
        _check_decode(out, None, q, k, v, lambda b, h: slice(0, N), G, dtype)


@pytest.mark.parametrize("dtype,fmt", TYPES)
@pytest.mark.parametrize("L,splits", [(1, 0), (40, 0), (333, 0), (333, 2), (2100, 0)])
def test_decode_listed(dtype, fmt, L, splits):
    """Lists with skipped ids, repeated ids, ids behind the length and outside the cache, and an empty list."""
    B, H, G, N = 3, 2, 4, 900
    gen = torch.Generator().manual_seed(L)
    q, cache, k, v = _decode_case(gen, B, H, G, N, dtype, fmt, "tokens")
    ids = torch.randint(0, N, (B, H, L), generator=gen, dtype=torch.int32)
    ids[torch.rand((B, H, L), generator=gen) < 0.1] = -1
    ids[0, 0, L // 2], ids[1, 1, 0], ids[2, 0, L - 1] = N + 3, 2 ** 31 - 1, -2 ** 31
    count = torch.randint(1, L + 1, (B, H), generator=gen, dtype=torch.int32)
    count[1, 0], count[2, 1], count[0, 0] = 0, L + 7, L
    length = [N, 600, N]
    announce("kvq decode listed %s %s L%d splits %d" % (dtype, fmt, L, splits))
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, num_splits=splits, kv_len=_i32(length), kv_idx=ids.cuda(),
                                    kv_count=count.cuda(), return_lse=True)

    def rows(b, h):
        got = ids[b, h, :min(int(count[b, h]), L)].long()
        return got[(got >= 0) & (got < length[b])]

    _check_decode(out, lse, q, k, v, rows, G, dtype)


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_decode_masked_places_hold_anything(dtype, fmt):
    """NaN scales and the NaN / largest codes behind the length, and in rows that a list skips, change nothing."""
    B, H, G, N = 2, 2, 8, 200
    gen = torch.Generator().manual_seed(3)
    q, cache, k, v = _decode_case(gen, B, H, G, N, dtype, fmt, "heads")
    length = [77, 33]
    clean = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length))
    for b in range(B):
        for codes, scale in ((cache.k_codes, cache.k_scale), (cache.v_codes, cache.v_scale)):
            codes.view(torch.uint8)[b, length[b]:] = 0x7F
            scale[b, length[b]:] = math.nan if b else math.inf
    announce("kvq decode masked places")
    assert torch.equal(clean, ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length)))
    for row in (0, 50):      # row 0 stands in for a skipped id: it must not reach the sums either
        cache.k_scale[:, row] = math.nan
        cache.v_scale[:, row] = math.nan
        cache.v_codes.view(torch.uint8)[:, row] = 0x7F
    ids = torch.arange(100, dtype=torch.int32).repeat(B, H, 1)
    ids[ids % 50 == 0] = -1
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=G, kv_len=_i32(length), kv_idx=ids.cuda(), return_lse=True)
    _check_decode(out, lse, q, k, v, lambda b, h: torch.tensor([t for t in range(length[b]) if t % 50]), G, dtype)


@pytest.mark.parametrize("splits", [1, 4])
def test_decode_shows_nan_rows(splits):
    """A row that could not be quantised makes what attends to it NaN, never a finite number."""
    q, cache, _, _ = _decode_case(torch.Generator().manual_seed(9), 2, 2, 4, 600, "bf16", "e4m3", "heads")
    cache.k_scale[0, 411, 1] = math.nan
    cache.v_scale[1, 7, 0] = math.nan
    announce("kvq decode nan rows")
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, group=4, num_splits=splits, return_lse=True)
    assert torch.isnan(out[0, 4:]).all() and torch.isnan(lse[0, 4:]).all() and torch.isfinite(out[0, :4]).all()
    assert torch.isnan(out[1, :4]).all() and torch.isfinite(lse[1]).all() and torch.isfinite(out[1, 4:]).all()


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_decode_scales_far_apart(dtype, fmt):
    """Value rows whose sizes differ by powers of two up to 2^60 and logits that span hundreds."""
    B, H, G, N = 1, 2, 4, 400
    gen = torch.Generator().manual_seed(21)
    q, cache, k, v = _decode_case(gen, B, H, G, N, dtype, fmt, "heads", spread=1.5)
    far = torch.exp2(torch.randint(-50, 11, (B, N, H), generator=gen).float())
    cache.v_scale.mul_(far.cuda())
    v = v * far.double()[..., None]
    announce("kvq decode far scales")
    out, lse = ops.kvq_flash_decode((q * 4).cuda(), cache, SCALE, group=G, out_dtype=torch.bfloat16, return_lse=True)
    _check_decode(out, lse, q * 4, k, v, lambda b, h: slice(0, N), G, dtype)


@pytest.mark.parametrize("scale", [-0.3, 0.0])
def test_decode_score_factors(scale):
    """A negative factor turns the weights round, a factor of zero makes them equal; so does a negative scale of a row."""
    q, cache, k, v = _decode_case(torch.Generator().manual_seed(5), 1, 2, 4, 300, "bf16", "int8", "heads")
    cache.k_scale[:, ::3] *= -1
    cache.v_scale[:, ::5] *= -100
    k[:, ::3] *= -1
    v[:, ::5] *= -100
    announce("kvq decode factor %g" % scale)
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, scale, 4, return_lse=True)
    for h in range(2):
        check_attention(out[0, 4 * h:4 * h + 4], lse[0, 4 * h:4 * h + 4], q[0, 4 * h:4 * h + 4], k[0, :, h], v[0, :, h], out.dtype, False, scale)


@pytest.mark.parametrize("fmt", list(CODES))
def test_decode_shared_cache(fmt):
    """One cache [N,H,128] for the batch equals a copy for each entry, bit for bit."""
    gen = torch.Generator().manual_seed(4)
    q, cache, _, _ = _decode_case(gen, 1, 2, 2, 300, "f16", fmt, "tokens")
    q = torch.randn((3, 4, 128), generator=gen).half().cuda()
    shared = ops.QuantCache(cache.k_codes[0], cache.v_codes[0], cache.k_scale[0], cache.v_scale[0])
    copies = ops.QuantCache(*(x.view(torch.uint8).repeat(3, 1, 1, 1).view(x.dtype) for x in (cache.k_codes, cache.v_codes)),
                            *(x.repeat(3, 1, 1) for x in (cache.k_scale, cache.v_scale)))
    announce("kvq decode shared cache")
    length = _i32([300, 17, 0])
    assert torch.equal(ops.kvq_flash_decode(q, shared, SCALE, 2, kv_len=length), ops.kvq_flash_decode(q, copies, SCALE, 2, kv_len=length))
    assert torch.equal(ops.kvq_scores(q, shared, SCALE, 2, kv_len=length), ops.kvq_scores(q, copies, SCALE, 2, kv_len=length))


def test_offsets_beyond_32_bits():
    """A cache whose last rows lie beyond 4 GiB: written, read, scored, attended to."""
    N, stride = 300, 1 << 24
    gen = torch.Generator().manual_seed(8)
    codes = [torch.zeros((N * stride,), dtype=torch.int8, device="cuda").as_strided((1, N, 1, 128), (0, stride, 128, 1)) for _ in range(2)]
    scale = [torch.zeros((1, N, 1), device="cuda") for _ in range(2)]
    cache = ops.QuantCache(codes[0], codes[1], scale[0], scale[1])
    k, v = (torch.randn((1, N, 1, 128), generator=gen).bfloat16() for _ in range(2))
    announce("kvq far offsets")
    ops.kvq_write(cache, k.cuda(), v.cuda())
    qk, qv = quantise64(k, "int8"), quantise64(v, "int8")
    assert torch.equal(cache.k_codes.cpu().double(), qk[0]) and torch.equal(cache.v_scale.cpu(), qv[1])
    got = ops.kvq_read(cache, 5, start=_i32([N - 5]))[1]
    assert torch.equal(got.cpu(), (qv[0].float() * qv[1][..., None]).to(torch.bfloat16)[:, N - 5:])
    q = torch.randn((1, 4, 128), generator=gen).bfloat16()
    kd, vd = (c * s.double()[..., None] for c, s in (qk, qv))
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, 4, return_lse=True)
    _check_decode(out, lse, q, kd, vd, lambda b, h: slice(0, N), 4, "bf16")
    ids = torch.arange(N - 40, N, dtype=torch.int32).view(1, 1, 40).cuda()
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, 4, kv_idx=ids, return_lse=True)
    _check_decode(out, lse, q, kd, vd, lambda b, h: slice(N - 40, N), 4, "bf16")
    scores = ops.kvq_scores(q.cuda(), cache, SCALE, 4).double().cpu()[0, 0]
    exact = (kd[0, :, 0] @ q[0].double().sum(0)) * SCALE
    assert ((scores - exact).abs() <= 23 * U * SCALE * (kd[0, :, 0].abs() @ q[0].double().abs().sum(0))).all()


# ---- used together --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,fmt", TYPES)
def test_sparse_decode_steps_over_the_cache(dtype, fmt):
    """A ragged prompt, then decode steps: append the new token, score, select, unite with sink and window, attend; against
    64 bits over what the cache holds and the selected tokens."""
    B, H, G, N, k_sel, sink, local = 2, 2, 4, 700, 64, 4, 16
    dt = DTYPES[dtype]
    gen = torch.Generator().manual_seed(31)
    cache = ops.QuantCache.empty(B, N, H, CODES[fmt])
    prompt = [600, 431]
    announce("kvq steps %s %s" % (dtype, fmt))
    k, v = (torch.randn((B, 600, H, 128), generator=gen).to(dt).cuda() for _ in range(2))
    ops.kvq_write(cache, k, v, count=_i32(prompt))
    for step in range(3):
        k, v = (torch.randn((B, 1, H, 128), generator=gen).to(dt).cuda() for _ in range(2))
        q = torch.randn((B, H * G, 128), generator=gen).to(dt).cuda()
        now = [p + step for p in prompt]
        ops.kvq_write(cache, k, v, start=_i32(now))
        length = [n + 1 for n in now]
        scores = ops.kvq_scores(q, cache, SCALE, G, kv_len=_i32(length))
        idx, _ = ops.topk(scores.view(B * H, N), k_sel)
        idx = idx.view(B, H, k_sel)
        kd = cache.k_codes.float().double().cpu() * cache.k_scale.double().cpu()[..., None]
        vd = cache.v_codes.float().double().cpu() * cache.v_scale.double().cpu()[..., None]
        for b in range(B):
            union, count = ops.index_union(idx[b], sink, local, length[b])
            out, lse = ops.kvq_flash_decode(q[b:b + 1], ops.QuantCache(cache.k_codes[b:b + 1], cache.v_codes[b:b + 1], cache.k_scale[b:b + 1], cache.v_scale[b:b + 1]),
                                            SCALE, G, kv_len=_i32([length[b]]), kv_idx=union[None], kv_count=count[None], return_lse=True)
            for h in range(H):
                want = torch.topk(scores[b, h, :length[b]], k_sel).values
                assert torch.equal(torch.sort(scores[b, h][idx[b, h].long()], descending=True).values, want)
                rows = union[h, :int(count[h])].long().cpu()
                assert set(rows.tolist()) == set(idx[b, h].tolist()) | set(range(sink)) | set(range(length[b] - local, length[b]))
                check_attention(out[0, h * G:(h + 1) * G], lse[0, h * G:(h + 1) * G], q[b, h * G:(h + 1) * G].cpu(), kd[b, rows, h], vd[b, rows, h], dt, dtype == "f16")


def test_centre_selection_over_the_cache():
    """The centre-only selection names whole clusters of the 8-bit cache, the listed decode attends to them."""
    H, C, clen, top_c = 4, 16, 32, 5
    gen = torch.Generator().manual_seed(6)
    q, cache, k, v = _decode_case(gen, 1, H, 1, C * clen, "f16", "int8", "heads")
    centers = torch.randn((H, C, 128), generator=gen).half().cuda()
    announce("kvq centre selection")
    ids, _, _ = ops.center_topk_expand(q[0].cuda(), centers, top_c, clen)
    out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, 1, kv_idx=ids[None], return_lse=True)
    _check_decode(out, lse, q, k, v, lambda b, h: ids[h].long().cpu(), 1, "f16")


@pytest.mark.parametrize("fmt", list(CODES))
def test_graph_replays(fmt):
    """Write, scores and both decodes captured into one graph, replayed over changing inputs, with the program's own eager
    calls between: every replay gives what the eager calls give."""
    B, H, G, N = 2, 2, 4, 1500
    gen = torch.Generator().manual_seed(13)
    q, cache, _, _ = _decode_case(gen, B, H, G, N, "bf16", fmt, "heads")
    q = q.cuda()
    new = [torch.zeros((B, 1, H, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    start, length = _i32([700, 900]), _i32([701, 901])
    ids = torch.arange(0, 1200, 3, dtype=torch.int32).repeat(B, H, 1).cuda()
    write = ops.KvqWritePlan(cache, new[0], new[1], start=start)
    plans = [ops.KvqScoresPlan(q, cache, SCALE, G, kv_len=length), ops.KvqFlashDecodePlan(q, cache, SCALE, G, kv_len=length, return_lse=True),
             ops.KvqFlashDecodePlan(q, cache, SCALE, G, kv_len=length, kv_idx=ids, return_lse=True)]
    announce("kvq graph")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        write.run()
        for p in plans:
            p.run()
    for step in range(4):
        for x in new:
            x.copy_(torch.randn(x.shape, generator=gen))
        q.copy_(torch.randn(q.shape, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        got = [plans[0].scores.clone()] + [x.clone() for p in plans[1:] for x in (p.out, p.lse)]
        held = [cache.k_codes.view(torch.uint8).clone(), cache.v_scale.clone()]
        ops.kvq_write(cache, new[0], new[1], start=start)
        want = [ops.kvq_scores(q, cache, SCALE, G, kv_len=length), *ops.kvq_flash_decode(q, cache, SCALE, G, kv_len=length, return_lse=True),
                *ops.kvq_flash_decode(q, cache, SCALE, G, kv_len=length, kv_idx=ids, return_lse=True)]
        assert torch.equal(held[0], cache.k_codes.view(torch.uint8)) and torch.equal(held[1], cache.v_scale)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        start.add_(1)
        length.add_(1)


def test_two_streams():
    """Two plans of one cache on two streams at a time, each with its own workspace."""
    gen = torch.Generator().manual_seed(14)
    q, cache, _, _ = _decode_case(gen, 2, 2, 4, 3000, "f16", "e4m3", "heads")
    qs = [torch.randn((2, 8, 128), generator=gen).half().cuda() for _ in range(2)]
    want = [ops.kvq_flash_decode(x, cache, SCALE, 4) for x in qs]
    plans = [ops.KvqFlashDecodePlan(x, cache, SCALE, 4) for x in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    announce("kvq two streams")
    torch.cuda.synchronize()
    for _ in range(20):
        for s, p in zip(streams, plans):
            with torch.cuda.stream(s):
                p.run()
    torch.cuda.synchronize()
    assert all(torch.equal(p.out, w) for p, w in zip(plans, want))
