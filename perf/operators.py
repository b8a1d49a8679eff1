"""The operators of 8-bit K/V caches and of shared prefixes as a decoding program calls them: what a pass reads, computes
and returns, in plain torch (`own` false) and through topk_attn_amd.ops (`own` true).

  write    new K and V rows are quantised into the cache (one step of a batch, a ragged prompt)
  read     rows of the cache as 16-bit numbers again
  scores   q . K^T over the 8-bit keys, the input of the top-k selection
  decode   one decode step of attention over the 8-bit cache, all rows or the listed ones
  prefix   one decode step of a batch whose sequences share a long prefix and have a suffix each

A row is the 128 elements of one (sequence, token, KV head); it is held as 128 codes and one fp32 scale and stands for
code * scale.  e4m3: scale = the smallest power of two (2^-126 at least) with max|x| <= 448 * scale, code = x / scale
rounded to the nearest even e4m3 number.  int8: scale = max(max|x| / 127, 2^-126), code = x * (1 / scale') rounded to the
nearest even whole number, 1 / scale' = 127 / max|x| (2^126 at most), each step in fp32."""
import math

import numpy as np
import torch

own = False

HEAD_DIM = 128
_DT = {"f16": torch.float16, "bf16": torch.bfloat16}
_SCALE = 1.0 / math.sqrt(HEAD_DIM)


def listed():
    return [
        # one token of 32 sequences is appended, every sequence at a position of its own: the write of every decode step
        {"name": "write step", "op": "write", "dtype": "bf16", "fmt": "e4m3", "batch": 32, "heads": 8, "tokens": 1, "rows": 4096, "layout": "heads"},
        # three prompts of different lengths go into a cache whose layout is [token][head], padded to the longest
        {"name": "write prompts", "op": "write", "dtype": "f16", "fmt": "int8", "batch": 3, "heads": 8, "tokens": 16385, "rows": 16500, "layout": "tokens"},
        # a window of a short cache goes back to 16 bits
        {"name": "read window", "op": "read", "dtype": "f16", "fmt": "e4m3", "batch": 4, "heads": 8, "tokens": 129, "rows": 2000, "layout": "tokens"},
        # whole prompts go back to 16 bits, to be handed to an operator of 16-bit caches
        {"name": "read prompts", "op": "read", "dtype": "bf16", "fmt": "int8", "batch": 2, "heads": 8, "tokens": 32768, "rows": 32768, "layout": "heads"},
        # the scores of a short context on a few heads
        {"name": "scores short", "op": "scores", "dtype": "f16", "fmt": "int8", "batch": 1, "heads": 4, "group": 8, "rows": 4099, "layout": "heads"},
        # the scores of a sparse decode step on long contexts, what its top-k selects from
        {"name": "scores long", "op": "scores", "dtype": "bf16", "fmt": "e4m3", "batch": 4, "heads": 8, "group": 4, "rows": 131072, "layout": "heads"},
        # one sequence, one GPU's head of a model that is sharded by its heads
        {"name": "decode short", "op": "decode", "dtype": "f16", "fmt": "int8", "batch": 1, "heads": 1, "group": 8, "rows": 1000, "picked": 0, "layout": "heads"},
        # four sequences of up to 32768 tokens, all of them attended to
        {"name": "decode dense", "op": "decode", "dtype": "bf16", "fmt": "e4m3", "batch": 4, "heads": 8, "group": 4, "rows": 32768, "picked": 0, "layout": "heads"},
        # the attention of a sparse decode step: 2048 selected tokens with the first 16 and the last 64 of each head
        {"name": "decode listed", "op": "decode", "dtype": "bf16", "fmt": "int8", "batch": 8, "heads": 8, "group": 4, "rows": 32768, "picked": 2128, "layout": "heads"},
        # a few requests behind one system prompt
        {"name": "prefix short", "op": "prefix", "dtype": "f16", "fmt": "16bit", "batch": 4, "heads": 2, "group": 4, "rows": 1000, "suffix": 33, "layout": "tokens"},
        # a batch of requests about one long document
        {"name": "prefix document", "op": "prefix", "dtype": "bf16", "fmt": "16bit", "batch": 16, "heads": 8, "group": 4, "rows": 32768, "suffix": 500, "layout": "tokens"},
        # a large batch behind a shared prefix in 8 bits: the matrix products outweigh the bytes
        {"name": "prefix large batch", "op": "prefix", "dtype": "bf16", "fmt": "e4m3", "batch": 64, "heads": 8, "group": 8, "rows": 32768, "suffix": 256, "layout": "heads"},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _price(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1e15)


def draw(rng):
    """One more case of the ranges above."""
    most = max(_price(c) for c in listed())
    while True:
        op = rng.choice(("write", "read", "scores", "decode", "decode", "prefix", "prefix"))
        case = {"op": op, "dtype": rng.choice(("f16", "bf16")), "fmt": rng.choice(("e4m3", "int8")), "heads": rng.choice((1, 2, 4, 8, 8, 16)),
                "layout": rng.choice(("heads", "tokens"))}
        if op in ("write", "read"):
            case["batch"] = _spread(rng, 1, 64)
            case["tokens"] = 1 if op == "write" and rng.random() < 0.3 else _spread(rng, 2, 32768)
            case["rows"] = case["tokens"] + _spread(rng, 1, 512)
        elif op == "scores":
            case["batch"], case["group"], case["rows"] = _spread(rng, 1, 16), rng.choice((1, 2, 4, 8)), _spread(rng, 100, 131072)
        elif op == "decode":
            case["batch"], case["group"], case["rows"] = _spread(rng, 1, 32), rng.choice((1, 2, 4, 8)), _spread(rng, 100, 131072)
            case["picked"] = 0 if rng.random() < 0.5 else min(case["rows"], _spread(rng, 32, 4200))
        else:
            case["batch"], case["group"], case["rows"] = _spread(rng, 2, 64), rng.choice((1, 2, 4, 8)), _spread(rng, 100, 65536)
            case["suffix"] = _spread(rng, 1, 1024)
            case["fmt"] = rng.choice(("16bit", "16bit", "e4m3", "int8"))
        cells = case["batch"] * case["heads"] * case["rows"] if op != "prefix" else case["heads"] * (case["rows"] + case["batch"] * case["suffix"])
        if _price(case) <= most and cells <= 4 * 8 * 131072:
            return case


# ---- inputs -------------------------------------------------------------------------------------


def _quantise(x, fmt):
    """fp32 rows [..., 128] -> (codes as fp32 numbers, fp32 scales [...]), the definition at the head of this file."""
    top = x.abs().amax(-1, keepdim=True)
    if fmt == "e4m3":
        m, e = torch.frexp(top)
        scale = torch.ldexp(torch.ones_like(top), torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126))  # 448 = 0.875 * 2^9
        scale = torch.where(top > 0, scale, torch.full_like(top, 2.0 ** -126))
        y = x / scale
        ulp = torch.ldexp(torch.ones_like(y), torch.frexp(y)[1].clamp(min=-5) - 4)    # 4 bits of significand, least exponent -6
        return torch.round(y / ulp) * ulp, scale.squeeze(-1)
    most = torch.full_like(top, 127.0)   # (a tensor: torch divides by a number, and a number by a tensor, through a rounded reciprocal)
    scale = (top / most).clamp(min=2.0 ** -126)
    inverse = (most / top).clamp(max=2.0 ** 126)
    return torch.round(x * inverse), scale.squeeze(-1)


def _stored(codes, fmt):
    return codes.to(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8)


def _laid(x, layout):
    """[B, N, H, ...] held head by head or token by token, the same shape either way."""
    return x.transpose(1, 2).contiguous().transpose(1, 2) if layout == "heads" else x.contiguous()


def _rows(gen, shape):
    """Rows as a model makes them: normal elements, some channels larger, the size of a row its own."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x *= torch.exp(0.4 * torch.randn(shape[-1], generator=gen, device="cuda"))
    x *= torch.exp(0.3 * torch.randn(shape[:-1] + (1,), generator=gen, device="cuda"))
    return x


def _cache(gen, batch, rows, heads, fmt, layout, dtype, values=True):
    """Tensors of a cache: codes and scales, or 16-bit rows (fmt "16bit"); keys, then values."""
    got = []
    for _ in range(2 if values else 1):
        x = _rows(gen, (batch, rows, heads, HEAD_DIM)).to(dtype)
        if fmt == "16bit":
            got.append((_laid(x, layout),))
        else:
            codes, scale = _quantise(x.float(), fmt)
            got.append((_laid(_stored(codes, fmt), layout), _laid(scale, "heads")))
            del codes
        del x
    return got


def _lengths(rs, batch, most):
    """Ragged lengths: the first sequence is full, one of five and more is empty."""
    n = rs.randint((most + 1) // 2, most + 1, batch)
    n[0] = most
    if batch >= 5:
        n[3] = 0
    return torch.from_numpy(n.astype(np.int32)).cuda()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) % (1 << 62))
    rs = np.random.RandomState(int(seed) % (1 << 31))
    op, dtype, B, H = case["op"], _DT[case["dtype"]], case["batch"], case["heads"]
    s = {"case": case}
    if op == "write":
        T, N = case["tokens"], case["rows"]
        s["k"], s["v"] = (_rows(gen, (B, T, H, HEAD_DIM)).to(dtype) for _ in range(2))
        s["count"] = _lengths(rs, B, T)
        s["start"] = torch.from_numpy(rs.randint(0, N - T + 1, B).astype(np.int32)).cuda()
        for kind in ("k", "v"):
            s[kind + "_codes"] = _laid(torch.zeros((B, N, H, HEAD_DIM), device="cuda").to(torch.float8_e4m3fn if case["fmt"] == "e4m3" else torch.int8), case["layout"])
            s[kind + "_scale"] = _laid(torch.zeros((B, N, H), device="cuda"), "heads")
        return s
    if op == "prefix":
        s["q"] = torch.randn((B, H * case["group"], HEAD_DIM), generator=gen, device="cuda").to(dtype)
        s["prefix"] = [tuple(t[0] for t in x) for x in _cache(gen, 1, case["rows"], H, case["fmt"], case["layout"], dtype)]
        s["suffix"] = _cache(gen, B, case["suffix"], H, case["fmt"], case["layout"], dtype)
        s["length"] = _lengths(rs, B, case["suffix"])
        return s
    (s["k_codes"], s["k_scale"]), *rest = _cache(gen, B, case["rows"], H, case["fmt"], case["layout"], dtype, values=op != "scores")
    if rest:
        s["v_codes"], s["v_scale"] = rest[0]
    if op == "read":
        s["count"] = _lengths(rs, B, case["tokens"])
        s["start"] = torch.from_numpy(rs.randint(0, case["rows"] - case["tokens"] + 1, B).astype(np.int32)).cuda()
        s["k"], s["v"] = (torch.zeros((B, case["tokens"], H, HEAD_DIM), dtype=dtype, device="cuda") for _ in range(2))
        return s
    s["q"] = torch.randn((B, H * case["group"], HEAD_DIM), generator=gen, device="cuda").to(dtype)
    if op == "decode" and case["picked"]:
        N, L = case["rows"], case["picked"]
        draws = torch.rand((B, H, N), generator=gen, device="cuda")
        ids = draws.topk(L, dim=-1).indices.sort(dim=-1).values.to(torch.int32)
        s["ids_count"] = torch.from_numpy(rs.randint((L + 1) // 2, L + 1, (B, H)).astype(np.int32)).cuda()
        s["ids"] = torch.where(torch.arange(L, device="cuda") < s["ids_count"][..., None], ids, torch.full_like(ids, -1))
    else:
        s["length"] = _lengths(rs, B, case["rows"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        from topk_attn_amd import ops
        op = case["op"]
        if op == "prefix":
            quantised = case["fmt"] != "16bit"
            prefix, suffix = ((ops.QuantCache(x[0][0], x[1][0], x[0][1], x[1][1]) if quantised else (x[0][0], x[1][0])) for x in (s["prefix"], s["suffix"]))
            s["plan"] = ops.PrefixDecodePlan(s["q"], prefix, suffix, _SCALE, group=case["group"], suffix_len=s["length"], return_lse=True)
            return s
        cache = ops.QuantCache(s["k_codes"], s.get("v_codes"), s["k_scale"], s.get("v_scale"))
        if op == "write":
            s["plan"] = ops.KvqWritePlan(cache, s["k"], s["v"], start=s["start"], count=s["count"])
        elif op == "read":
            s["plan"] = ops.KvqReadPlan(cache, s["k"], s["v"], start=s["start"], count=s["count"])
        elif op == "scores":
            s["plan"] = ops.KvqScoresPlan(s["q"], cache, _SCALE, group=case["group"], kv_len=s["length"])
        else:
            s["plan"] = ops.KvqFlashDecodePlan(s["q"], cache, _SCALE, group=case["group"], kv_len=s.get("length"), kv_idx=s.get("ids"),
                                               kv_count=s.get("ids_count"), return_lse=True)
    return s


# ---- the operators in plain torch ---------------------------------------------------------------


def _heads(codes, scale=None):
    """[B, N, H, 128] codes and [B, N, H] scales -> fp32 [B, H, N, 128]."""
    x = codes.transpose(1, 2).float()
    return x if scale is None else x * scale.transpose(1, 2)[..., None]


def _softmax_parts(logits):
    """Row maxima (0 where a row has nothing), exponentials and their sums."""
    top = logits.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = torch.exp(logits - top)
    return top, p, p.sum(-1, keepdim=True)


def _finish(out, top, total, dtype, shape):
    some = total > 0
    out = torch.where(some, out / torch.where(some, total, torch.ones_like(total)), torch.zeros_like(out))
    lse = torch.where(some, top + torch.log(torch.where(some, total, torch.ones_like(total))), torch.full_like(top, -math.inf))
    return out.reshape(shape).to(dtype), lse.reshape(shape[:2])


def _plain_write(s):
    B, T, _, _ = s["k"].shape
    t = torch.arange(T, device="cuda")
    kept = (t < s["count"][:, None]).nonzero(as_tuple=True)      # (sequence, token) pairs that there are
    to = (s["start"][kept[0]] + kept[1]).long()
    for kind in ("k", "v"):
        codes, scale = _quantise(s[kind][kept].float(), s["case"]["fmt"])
        held = s[kind + "_codes"]
        held.view(torch.int8)[kept[0], to] = _stored(codes, s["case"]["fmt"]).view(torch.int8)
        s[kind + "_scale"][kept[0], to] = scale
    return [s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"]]


def _plain_read(s):
    B, T, _, _ = s["k"].shape
    t = torch.arange(T, device="cuda")
    there = (t < s["count"][:, None])[..., None, None]
    rows = (s["start"][:, None] + t).long()
    which = torch.arange(B, device="cuda")[:, None]
    for kind in ("k", "v"):
        held = s[kind + "_codes"]
        codes = held.view(torch.int8)[which, rows].view(held.dtype).float()
        s[kind] = torch.where(there, (codes * s[kind + "_scale"][which, rows][..., None]).to(s[kind].dtype), s[kind])
    return [s["k"], s["v"]]


def _plain_scores(s):
    c = s["case"]
    B, H, G = c["batch"], c["heads"], c["group"]
    q = s["q"].float().reshape(B, H, G, HEAD_DIM).sum(2, keepdim=True)
    dot = (_heads(s["k_codes"]) @ q.transpose(2, 3)).squeeze(-1)
    scores = dot * s["k_scale"].transpose(1, 2) * _SCALE
    there = torch.arange(c["rows"], device="cuda") < s["length"][:, None, None]
    return torch.where(there, scores, torch.full_like(scores, -math.inf))


def _plain_decode(s):
    c = s["case"]
    B, H, G = c["batch"], c["heads"], c["group"]
    q = s["q"].float().reshape(B, H, G, HEAD_DIM)
    if c["picked"]:
        ids = s["ids"].clamp(min=0).long()
        at = (torch.arange(B, device="cuda")[:, None, None], ids, torch.arange(H, device="cuda")[None, :, None])
        k, v = ((s[x + "_codes"].view(torch.int8)[at].view(s[x + "_codes"].dtype).float() * s[x + "_scale"][at][..., None]) for x in ("k", "v"))
        there = (torch.arange(c["picked"], device="cuda") < s["ids_count"][..., None]) & (s["ids"] >= 0)
    else:
        k, v = _heads(s["k_codes"], s["k_scale"]), _heads(s["v_codes"], s["v_scale"])
        there = (torch.arange(c["rows"], device="cuda") < s["length"][:, None, None]).expand(B, H, -1)
    logits = (q @ k.transpose(2, 3)) * _SCALE
    logits = torch.where(there[:, :, None], logits, torch.full_like(logits, -math.inf))
    top, p, total = _softmax_parts(logits)
    return _finish(p @ v, top, total, s["q"].dtype, (B, H * G, HEAD_DIM))


def _plain_prefix(s):
    c = s["case"]
    B, H, G, P = c["batch"], c["heads"], c["group"], c["rows"]
    q = s["q"].float().reshape(B, H, G, HEAD_DIM)
    kp, vp = (_heads(*(t[None] for t in x))[0] for x in s["prefix"])                 # [H, P, 128]
    ks, vs = (_heads(*x) for x in s["suffix"])                                       # [B, H, S, 128]
    shared = (q.transpose(0, 1).reshape(H, B * G, HEAD_DIM) @ kp.transpose(1, 2)).reshape(H, B, G, P).transpose(0, 1)
    rest = q @ ks.transpose(2, 3)
    there = torch.arange(c["suffix"], device="cuda") < s["length"][:, None, None, None]
    rest = torch.where(there, rest, torch.full_like(rest, -math.inf))
    top, p, total = _softmax_parts(torch.cat([shared, rest], dim=-1) * _SCALE)
    out = (p[..., :P].transpose(0, 1).reshape(H, B * G, P) @ vp).reshape(H, B, G, HEAD_DIM).transpose(0, 1) + p[..., P:] @ vs
    return _finish(out, top, total, s["q"].dtype, (B, H * G, HEAD_DIM))


_PLAIN = {"write": _plain_write, "read": _plain_read, "scores": _plain_scores, "decode": _plain_decode, "prefix": _plain_prefix}


def run(state):
    if not own:
        return _PLAIN[state["case"]["op"]](state)
    plan, op = state["plan"].run(), state["case"]["op"]
    if op == "write":
        return [state["k_codes"], state["v_codes"], state["k_scale"], state["v_scale"]]
    if op == "read":
        return [state["k"], state["v"]]
    if op == "scores":
        return plan.scores
    return plan.out, plan.lse


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    """Lengths are taken as the mean of what _lengths draws: three quarters of the longest."""
    op, B, H = case["op"], case["batch"], case["heads"]
    mean = lambda most, n: most * (0.25 + 0.75 * n) / n   # noqa: E731  the first is full
    row = 2 * HEAD_DIM if case["fmt"] == "16bit" else HEAD_DIM + 4
    if op in ("write", "read"):
        rows = B * H * mean(case["tokens"], B) * 2
        return {"bytes": rows * (2 * HEAD_DIM + row), "flops": rows * 3 * HEAD_DIM}
    G = case["group"]
    if op == "scores":
        rows = B * H * mean(case["rows"], B)
        return {"bytes": rows * row + B * H * (case["rows"] * 4 + G * HEAD_DIM * 2), "flops": rows * 2 * HEAD_DIM}
    ends = B * H * G * (HEAD_DIM * 2 * 2 + 4)
    if op == "decode":
        rows = B * H * (0.75 * case["picked"] if case["picked"] else mean(case["rows"], B))
        return {"bytes": 2 * rows * row + ends + (rows * 4 if case["picked"] else 0), "flops": rows * G * 4 * HEAD_DIM}
    own_rows = B * H * mean(case["suffix"], B)
    return {"bytes": 2 * (H * case["rows"] + own_rows) * row + ends, "flops": (H * case["rows"] * B + own_rows) * G * 4 * HEAD_DIM}


# ---- the definitions in 64 bits -----------------------------------------------------------------


def _nearest(x, fmt):
    """Rows in 64 bits -> (codes, scales), by the definition and not by the steps above."""
    top = x.abs().max(-1).values
    if fmt == "int8":
        scale = top / 127
        return torch.where(top[..., None] > 0, torch.round(x * 127 / top[..., None]), torch.zeros_like(x)), scale.clamp(min=2.0 ** -126)
    power = torch.ceil(torch.log2(top.clamp(min=1e-60) / 448)).clamp(min=-126)
    scale = 2.0 ** power
    y = x / scale[..., None]
    grid = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / grid) * grid, scale


def exact(case, seed):
    s = _inputs(case, seed)
    op, B, H = case["op"], case["batch"], case["heads"]
    if op == "write":
        got = [torch.zeros(s["k_codes"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        scales = [torch.zeros(s["k_scale"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b in range(B):
            n, to = int(s["count"][b]), int(s["start"][b])
            for i, kind in enumerate(("k", "v")):
                if n:
                    got[i][b, to:to + n], scales[i][b, to:to + n] = _nearest(s[kind][b, :n].double(), case["fmt"])
        if case["fmt"] == "int8":
            got = [g.to(torch.int8) for g in got]
        return got + scales
    if op == "read":
        got = [torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b in range(B):
            n, at = int(s["count"][b]), int(s["start"][b])
            for i, kind in enumerate(("k", "v")):
                got[i][b, :n] = s[kind + "_codes"][b, at:at + n].double() * s[kind + "_scale"][b, at:at + n].double()[..., None]
        return got
    G = case["group"]
    q = s["q"].double().reshape(B, H, G, HEAD_DIM)
    if op == "scores":
        scores = torch.full((B, H, case["rows"]), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = int(s["length"][b])
            for h in range(H):
                k = s["k_codes"][b, :n, h].double() * s["k_scale"][b, :n, h].double()[:, None]
                scores[b, h, :n] = (k * q[b, h].sum(0)).sum(-1) * _SCALE
        return scores
    out = torch.zeros((B, H, G, HEAD_DIM), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, G), -math.inf, dtype=torch.float64, device="cuda")

    def rows(held, *at):
        x = held[0][at] if held[0].element_size() > 1 else held[0].view(torch.int8)[at].view(held[0].dtype)
        return x.double() if len(held) == 1 else x.double() * held[1][at].double()[..., None]

    for h in range(H):
        if op == "prefix":
            kp, vp = (rows(x, slice(None), h) for x in s["prefix"])
        for b in range(B):
            if op == "prefix":
                n = int(s["length"][b])
                k, v = (torch.cat([p, rows(x, b, slice(0, n), h)]) for p, x in zip((kp, vp), s["suffix"]))
            else:
                if case["picked"]:
                    at = s["ids"][b, h, :int(s["ids_count"][b, h])].long()
                else:
                    at = slice(0, int(s["length"][b]))
                k, v = (rows((s[x + "_codes"], s[x + "_scale"]), b, at, h) for x in ("k", "v"))
            if len(k):
                logits = (q[b, h] @ k.T) * _SCALE
                lse[b, h] = torch.logsumexp(logits, -1)
                out[b, h] = torch.softmax(logits, -1) @ v
    return out.reshape(B, H * G, HEAD_DIM), lse.reshape(B, H * G)
