"""Shared by the tests of the 8-bit caches and the shared prefix: inputs, the definitions in 64 bits, error bounds.

Bounds of the decode outputs.  With u = 2^-24 (half a step of fp32), per query row and output element d:
  logits     the products are exact, their fp32 sum of 128 terms and the three factors behind it are off by at most
             140 * 2u * S, S = max over tokens of scale * sum |q k| (2u: the matrix unit need not round to nearest);
             in the exponent of 2 a logit has rounding |x| * 2u and the exponential 2^-21 of its own: a weight is off by at
             most e_w = 140 * 2u * S + |x|max * 2u + 2^-21 of itself, S and x in the base that makes them larger (log2 e);
  weights    in two parts (bf16 rows of 16 bits; every case of fp16 queries): 2^-16 of themselves.  One fp16 number (8-bit rows,
             bf16 queries): 2^-11, and twice that again where value rows carry their scales in fp16 (a factor and a
             product): 3 * 2^-11.  Below the normal range a weight is off by 2^-25, held times 2^9 over a cap of at most four
             times the largest scale, whose row holds a code of at least half the largest one: 2^-34 * 4 * 2 of max |v|,
             against a sum of weights of at least that of the reference, which lags by 2^6 at most: below 2^-31 of max |v|;
  sums       fp32 sums of n terms: n * 2u;
  output     rounded to its type: eps / 2 of itself.
So |error| <= eps_out / 2 * |o| + (2 e_w + w + 2 n * 2u) * sum p |v| + n * 2^-31 * max |v|, p the normalised weights; lse is off by
e_w + n * 2u + |lse| * 4u."""
import math

import torch

U = 2.0 ** -24
SCALE = 1.0 / math.sqrt(128.0)
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def quantise64(x, fmt):
    """Rows in 64 bits -> (codes, scales), from the definition in topk_attn_kvq.h (ties are decided on exact values)."""
    x = x.double()
    top = x.abs().amax(-1)
    if fmt == "int8":
        # fp32 quotients, as the definition says; a product of two fp32 numbers is exact in 64 bits, then rounded to fp32
        # (tensor by tensor: torch computes a number divided by a tensor as a rounded reciprocal times the number)
        t32 = top.float()
        most = torch.full_like(t32, 127.0)
        scale = (t32 / most).clamp(min=2.0 ** -126)
        inv = torch.where(t32 > 0, (most / t32).clamp(max=2.0 ** 126), torch.full_like(t32, 2.0 ** 126))
        codes = torch.round((x * inv.double()[..., None]).float().double())
    else:
        k = torch.full_like(top, -126.0)
        some = top > 0
        e = torch.floor(torch.log2(torch.where(some, top, torch.ones_like(top)))) - 10
        for _ in range(3):   # the smallest power whose 448-fold reaches the top, found by trying
            e = torch.where(448 * 2.0 ** e < top, e + 1, e)
        k = torch.where(some, e.clamp(min=-126), k)
        scale = 2.0 ** k
        y = x / scale[..., None]
        step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        codes = torch.round(y / step) * step
        scale = scale.float()
    bad = ~torch.isfinite(x).all(-1)
    scale = torch.where(bad, torch.full_like(scale, math.nan), scale)
    codes = torch.where(bad[..., None], torch.zeros_like(codes), codes)
    return codes, scale


def random_cache(gen, shape, fmt, spread=0.5):
    """Codes [..., 128] and scales [...] as they come from quantised rows, the scale of a row its own (on the CPU)."""
    x = torch.randn(shape, generator=gen) * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=gen))
    codes, scale = quantise64(x, fmt)
    return codes.float().to(CODES[fmt]), scale


def attention64(q, k, v, scale=SCALE):
    """q [R,128], k, v [n,128] in 64 bits -> out, lse, sum p|v|, S, |x|max; zeros and -inf without a row."""
    R = q.shape[0]
    if k.shape[0] == 0:
        z = torch.zeros(R, 128, dtype=torch.float64)
        return z, torch.full((R,), -math.inf, dtype=torch.float64), z, 0.0, 0.0
    s = (q @ k.T) * scale
    p = torch.softmax(s, -1)
    big = float(((q.abs() @ k.abs().T) * abs(scale)).max())
    return p @ v, torch.logsumexp(s, -1), p @ v.abs(), big, float(s.abs().max())


def check_attention(out, lse, q, k, v, dtype16, two_parts, scale=SCALE):
    """out [R,128] (16 bits), lse [R] of one head against 64 bits; k, v: the rows that count, in 64 bits."""
    o, l, pv, big, top = attention64(q.double(), k.double(), v.double(), scale)
    n = k.shape[0]
    log2e = 1.4426950408889634
    e_w = 140 * 2 * U * big * log2e + top * log2e * 2 * U + 2.0 ** -21
    w = 2.0 ** -16 if two_parts else 3 * 2.0 ** -11
    vmax = float(v.abs().max()) if n else 0.0
    bound = torch.finfo(dtype16).eps / 2 * o.abs() + (2 * e_w + w + 4 * n * U) * pv + n * 2.0 ** -31 * vmax + torch.finfo(dtype16).smallest_normal * torch.finfo(dtype16).eps
    err = (out.double().cpu() - o).abs()
    assert bool((err <= bound).all()), "out of bounds by a factor of %.3g (n %d)" % (float((err / bound.clamp(min=1e-300)).max()), n)
    if lse is not None:
        got = lse.double().cpu()
        if n == 0:
            assert bool((got == -math.inf).all())
        else:
            assert bool(((got - l).abs() <= e_w + 2 * n * U + l.abs() * 4 * U).all()), "lse off by %.3g" % float((got - l).abs().max())


def laid(t, layout):
    """[B,N,H,...] on the GPU, held token by token or head by head, or with gaps between the rows."""
    t = t.cuda()
    if layout == "heads":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "gaps":   # room for one more head and a wider row
        B, N, H = t.shape[:3]
        wide = torch.zeros((B, N, H + 1) + ((160,) if t.dim() == 4 else ()), dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device="cuda")
        if t.element_size() == 1:
            wide = wide.view(t.dtype)
        view = wide[:, :, :H, :128] if t.dim() == 4 else wide[:, :, :H]
        view.view(torch.int8 if t.element_size() == 1 else t.dtype).copy_(t.view(torch.int8) if t.element_size() == 1 else t)
        return view
    return t.contiguous()
