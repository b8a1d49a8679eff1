"""Value scales that tka_kvq_write does not make, in every form that reads an 8-bit cache: the readers accept any fp32 scale.
The bounds are those of kvq_util, derived there."""
import pytest
import torch

from kvq_util import DTYPES, SCALE, check_attention
from topk_attn_amd import _lib as L, ops
from util import announce

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[0, 1, 2, 4, 8, 16])
def row_tiles(request):
    """Blocks of 16 times as many query rows (0: what the call chooses)."""
    assert L.lib().tka_kvq_test_row_tiles(request.param) == 0
    yield request.param
    assert L.lib().tka_kvq_test_row_tiles(0) == 0


def _cache(codes, scale):
    """[N,H,128] and [N,H] on the CPU, keys then values -> the cache on the GPU, head by head, and the rows in 64 bits."""
    held = [c.cuda().transpose(0, 1).contiguous().transpose(0, 1) for c in codes], [s.cuda().t().contiguous().t() for s in scale]
    return ops.QuantCache(held[0][0], held[0][1], held[1][0], held[1][1]), *(c.float().double() * s.double()[..., None] for c, s in zip(codes, scale))


def _over_448(gen, shape):
    """Rows quantised with scale = max / 448, which is hardly ever a power of two."""
    x = torch.randn(shape, generator=gen) * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=gen))
    scale = x.abs().amax(-1) / 448
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _check(out, lse, q, k, v, G, two_parts):
    for b in range(q.shape[0]):
        for h in range(k.shape[1]):
            at = slice(h * G, (h + 1) * G)
            check_attention(out[b, at], lse[b, at], q[b, at], k[:, h], v[:, h], out.dtype, two_parts)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("P", [3, 70, 500])
@pytest.mark.parametrize("kinds", ["others", "mixed"])
def test_e4m3_scales_between_powers_of_two(row_tiles, dtype, P, kinds):
    """Small queries, so that the bound is little more than the rounding of the output.  mixed: some tiles have powers of two
    alone, some scales are negative or zero."""
    B, H, G = 19, 2, 8
    gen = torch.Generator().manual_seed(P)
    codes, scale = zip(*(_over_448(gen, (P, H, 128)) for _ in range(2)))
    if kinds == "mixed":
        s = scale[1]
        s[:64] = torch.exp2(torch.round(torch.log2(s[:64])))
        s[1::7] *= -1
        s[100::50] = 0.0
    cache, k, v = _cache(codes, scale)
    q = (0.05 * torch.randn((B, H * G, 128), generator=gen)).to(DTYPES[dtype])
    announce("kvq scales of others: blocks of %d, %s, P%d %s" % (16 * row_tiles, dtype, P, kinds))
    out, lse = ops.prefix_decode(q.cuda(), cache, None, SCALE, G, return_lse=True)
    _check(out, lse, q, k, v, G, dtype == "f16")


def _far_end(gen, fmt, N, H, top, rest):
    """Keys of zeros but for one row in 32 from row 512 on, whose logit lies 5.5 / log2 e above: its weight grows by 2^5.5 over
    the reference that the first tiles set, just less than what moves it.  Those value rows have the scale `top`, the others `rest`."""
    dt = torch.float8_e4m3fn if fmt == "e4m3" else torch.int8
    special = (torch.arange(N) >= 512) & (torch.arange(N) % 32 == 13)
    kc = torch.where(special[:, None, None], torch.ones(N, H, 128), torch.zeros(N, H, 128))
    ks = torch.full((N, H), 5.5 / 1.4426950408889634 / (128 * SCALE))
    vc = torch.randint(0, 2, (N, H, 128), generator=gen).float() * 2 - 1
    vs = torch.where(special[:, None], torch.full((N, H), top), torch.full((N, H), rest))
    return _cache([kc.to(dt), vc.to(dt)], [ks, vs])


FAR = [(2.0 ** 127.9, 2.0 ** 126), (2.0 ** 127, 2.0 ** 127), (2.0 ** 125.5, 2.0 ** 20), (2.0 ** -126, 2.0 ** -126), (2.0 ** -115, 2.0 ** -140), (2.0 ** -111, 2.0 ** -112)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("top,rest", FAR)
def test_prefix_scales_at_the_ends_of_the_range(row_tiles, dtype, fmt, top, rest):
    """Values near the largest number there is, and near the smallest."""
    B, H, G, N = 19, 2, 8, 1000
    gen = torch.Generator().manual_seed(3)
    cache, k, v = _far_end(gen, fmt, N, H, top, rest)
    q = torch.ones((B, H * G, 128), dtype=DTYPES[dtype])
    announce("kvq far scales: blocks of %d, %s %s %g %g" % (16 * row_tiles, dtype, fmt, top, rest))
    for splits in (0, 1):
        out, lse = ops.prefix_decode(q.cuda(), cache, None, SCALE, G, num_splits=splits, out_dtype=torch.bfloat16, return_lse=True)
        _check(out[:2], lse[:2], q[:2], k, v, G, dtype == "f16")
        assert torch.equal(out, out[:1].expand_as(out))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("top,rest", FAR)
def test_decode_scales_at_the_ends_of_the_range(dtype, fmt, top, rest):
    """The same through the decode over all rows, over listed rows, and over so few that one launch takes them."""
    H, G, N = 2, 4, 1000
    gen = torch.Generator().manual_seed(4)
    cache, k, v = _far_end(gen, fmt, N, H, top, rest)
    q = torch.ones((1, H * G, 128), dtype=DTYPES[dtype])
    announce("kvq far scales: decode %s %s %g %g" % (dtype, fmt, top, rest))
    for splits in (0, 1):
        out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, G, num_splits=splits, out_dtype=torch.bfloat16, return_lse=True)
        _check(out, lse, q, k, v, G, dtype == "f16")
    for ids in (torch.arange(N), torch.arange(400, 650)):
        listed = ids.to(torch.int32).repeat(1, H, 1).cuda()
        out, lse = ops.kvq_flash_decode(q.cuda(), cache, SCALE, G, kv_idx=listed, out_dtype=torch.bfloat16, return_lse=True)
        _check(out, lse, q, k[ids], v[ids], G, dtype == "f16")
