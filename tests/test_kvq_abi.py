"""The C boundary of include/topk_attn_kvq.h without a GPU: symbols, struct layouts, and refusals before any HIP call."""
import ctypes as C
import os
import re
import subprocess
import tempfile

import pytest
import torch

from topk_attn_amd import _lib as L
from topk_attn_amd import ops

INCLUDE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
STRUCTS = {"tka_kv_cache": L.KvCache, "tka_kvq_write_args": L.KvqWriteArgs, "tka_kvq_read_args": L.KvqReadArgs,
           "tka_kvq_scores_args": L.KvqScoresArgs, "tka_kvq_flash_decode_args": L.KvqFlashDecodeArgs,
           "tka_prefix_decode_args": L.PrefixDecodeArgs}


def test_symbols_match_the_header():
    with open(os.path.join(INCLUDE, "topk_attn_kvq.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    declared = set(re.findall(r"^\s*(?:int|size_t)\s+(tka_\w+)\s*\(", text, flags=re.M))
    assert declared == set(L.KVQ_PROTOTYPES) and not declared & set(L.PROTOTYPES)
    for name in declared:
        assert hasattr(L.lib(), name)


def test_ctypes_structs_match_the_c_layout():
    lines = ['#include <stdio.h>', '#include "topk_attn_kvq.h"', 'int main(void) {']
    for cname, cls in STRUCTS.items():
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (cname, cname))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (cname, f, cname, f) for f, _ in cls._fields_]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "layout.c"), os.path.join(d, "layout")
        with open(src, "w") as f:
            f.write("\n".join(lines + ["return 0; }"]))
        subprocess.check_call(["gcc", "-std=c11", "-Wall", "-Werror", "-I", INCLUDE, "-o", exe, src])
        got = dict(line.split() for line in subprocess.check_output([exe], text=True).strip().splitlines())
    for cname, cls in STRUCTS.items():
        assert int(got[cname]) == C.sizeof(cls), cname
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (cname, f)]) == getattr(cls, f).offset, (cname, f)


def _cache(fmt=L.TKA_KV_E4M3, batch=2, rows=100, heads=4):
    c = L.KvCache()
    c.k, c.v, c.format, c.batch, c.num_kv_heads, c.head_dim, c.rows = 0x10000, 0x20000, fmt, batch, heads, 128, rows
    c.stride_b, c.stride_n, c.stride_h = rows * heads * 128, heads * 128, 128
    if fmt != L.TKA_KV_16BIT:
        c.k_scale, c.v_scale = 0x30000, 0x40000
        c.scale_stride_b, c.scale_stride_n, c.scale_stride_h = heads * rows, 1, rows
    return c


def _copy(cls):
    a = cls()
    a.cache, a.k, a.v, a.dtype, a.num_tokens = _cache(), 0x50000, 0x60000, L.TKA_BF16, 10
    a.stride_b, a.stride_n, a.stride_h = 10 * 4 * 128, 4 * 128, 128
    return a


def _scores():
    a = L.KvqScoresArgs()
    a.cache, a.q, a.dtype, a.group, a.q_stride_b, a.scale, a.out_scores = _cache(), 0x50000, L.TKA_F16, 4, 16 * 128, 1.0, 0x70000
    return a


def _decode():
    a = L.KvqFlashDecodeArgs()
    a.cache, a.q, a.out, a.dtype, a.out_dtype, a.group, a.scale = _cache(), 0x50000, 0x60000, L.TKA_F16, L.TKA_BF16, 4, 0.1
    a.q_stride_b = a.out_stride_b = 16 * 128
    return a


def _prefix(fmt=L.TKA_KV_16BIT):
    a = L.PrefixDecodeArgs()
    a.prefix, a.suffix, a.q, a.out, a.dtype, a.out_dtype, a.group, a.scale = _cache(fmt, 1), _cache(fmt), 0x50000, 0x60000, L.TKA_F16, L.TKA_F16, 4, 0.1
    a.q_stride_b = a.out_stride_b = 16 * 128
    return a


INVALID, UNSUPPORTED = L.TKA_EINVAL, L.TKA_EUNSUPPORTED
CACHE_REFUSALS = [("format", 0, UNSUPPORTED), ("format", 7, UNSUPPORTED), ("head_dim", 64, UNSUPPORTED), ("batch", 0, INVALID),
                  ("num_kv_heads", 0, INVALID), ("rows", 0, INVALID), ("rows", -1, INVALID), ("rows", 1 << 31, UNSUPPORTED), ("k", None, INVALID),
                  ("k", 0x10008, INVALID), ("k_scale", None, INVALID), ("k_scale", 0x30002, INVALID), ("stride_n", 64, INVALID),
                  ("stride_n", 520, INVALID), ("stride_h", 136, INVALID), ("stride_b", -128, INVALID), ("stride_b", 1 << 62, INVALID),
                  ("scale_stride_n", -1, INVALID), ("batch", 70000, UNSUPPORTED), ("num_kv_heads", 70000, UNSUPPORTED)]


def _refused(fn, make, changes, where=None):
    for field, value, want in changes:
        a = make()
        setattr(getattr(a, where) if where else a, field, value)
        assert fn(C.byref(a)) == want, (field, value)


@pytest.mark.parametrize("name,make", [("tka_kvq_write", lambda: _copy(L.KvqWriteArgs)), ("tka_kvq_read", lambda: _copy(L.KvqReadArgs)),
                                       ("tka_kvq_scores", _scores), ("tka_kvq_flash_decode", _decode)])
def test_caches_are_checked(name, make):
    fn = getattr(L.lib(), name)
    assert fn(None) == INVALID
    _refused(fn, make, CACHE_REFUSALS, "cache")
    if name != "tka_kvq_scores":
        _refused(fn, make, [("v", None, INVALID), ("v_scale", None, INVALID), ("v", 0x20001, INVALID)], "cache")


@pytest.mark.parametrize("name,cls", [("tka_kvq_write", L.KvqWriteArgs), ("tka_kvq_read", L.KvqReadArgs)])
def test_copies_are_checked(name, cls):
    fn = getattr(L.lib(), name)
    _refused(fn, lambda: _copy(cls), [("k", None, INVALID), ("v", None, INVALID), ("v", 0x60008, INVALID), ("dtype", 5, UNSUPPORTED),
                                      ("num_tokens", 0, INVALID), ("num_tokens", -3, INVALID), ("stride_n", 516, INVALID),
                                      ("stride_b", -8, INVALID), ("num_tokens", 0x7fffffff, UNSUPPORTED if name == "tka_kvq_write" else UNSUPPORTED)])


def test_writes_into_overlapping_rows_are_refused():
    """Two rows of a written cache (or of the output of a read) may not share bytes: a race otherwise."""
    lib = L.lib()
    for field, value in (("stride_b", 0), ("stride_h", 0), ("stride_n", 256), ("scale_stride_b", 0), ("scale_stride_h", 50), ("scale_stride_n", 0),
                         ("stride_b", 99 * 512)):
        a = _copy(L.KvqWriteArgs)
        setattr(a.cache, field, value)
        assert lib.tka_kvq_write(C.byref(a)) == INVALID, field
    for field, value in (("stride_b", 0), ("stride_h", 0), ("stride_n", 256)):
        a = _copy(L.KvqReadArgs)
        setattr(a, field, value)
        assert lib.tka_kvq_read(C.byref(a)) == INVALID, field


def test_scores_are_checked():
    _refused(L.lib().tka_kvq_scores, _scores, [("q", None, INVALID), ("q", 0x50004, INVALID), ("dtype", 3, UNSUPPORTED), ("group", 3, UNSUPPORTED),
                                               ("group", 16, UNSUPPORTED), ("q_stride_b", 128, INVALID), ("q_stride_b", 2052, INVALID),
                                               ("out_scores", None, INVALID), ("reserved0", 1, INVALID)])


def test_decode_is_checked():
    lib = L.lib()
    a = _decode()
    need = lib.tka_kvq_flash_decode_workspace_bytes(C.byref(a))
    assert need > 0 and lib.tka_kvq_flash_decode(C.byref(a)) == L.TKA_EWORKSPACE
    a.workspace, a.workspace_bytes = 0x100000, need - 1
    assert lib.tka_kvq_flash_decode(C.byref(a)) == L.TKA_EWORKSPACE
    changes = [("q", None, INVALID), ("out", None, INVALID), ("out", 0x60004, INVALID), ("dtype", 3, UNSUPPORTED), ("out_dtype", 2, UNSUPPORTED),
               ("group", 5, UNSUPPORTED), ("num_splits", -1, INVALID), ("num_splits", 1025, INVALID), ("q_stride_b", 1024, INVALID),
               ("out_stride_b", 1024, INVALID), ("kv_count", 0x80000, INVALID), ("idx_len", 4, INVALID), ("kv_idx", 0x80000, INVALID)]
    _refused(lib.tka_kvq_flash_decode, _decode, changes)
    for field, value, _ in changes:
        b = _decode()
        setattr(b, field, value)
        assert lib.tka_kvq_flash_decode_workspace_bytes(C.byref(b)) == 0
    b = _decode()      # more partials than a launch takes: refused, not wrapped around
    b.cache.batch, b.cache.num_kv_heads, b.num_splits, b.cache.rows = 60000, 16, 1024, 1 << 20
    b.cache.stride_b, b.cache.scale_stride_b, b.q_stride_b, b.out_stride_b = 1 << 30, 1 << 24, 64 * 128, 64 * 128
    assert lib.tka_kvq_flash_decode(C.byref(b)) == UNSUPPORTED


@pytest.mark.parametrize("fmt", [L.TKA_KV_16BIT, L.TKA_KV_E4M3, L.TKA_KV_INT8])
def test_prefix_is_checked(fmt):
    lib = L.lib()
    fn, make = lib.tka_prefix_decode, lambda: _prefix(fmt)
    assert fn(None) == INVALID
    assert lib.tka_prefix_decode_workspace_bytes(C.byref(make())) > 0 and fn(C.byref(make())) == L.TKA_EWORKSPACE
    for side in ("prefix", "suffix"):
        _refused(fn, make, [(f, v, w) for f, v, w in CACHE_REFUSALS if f not in ("format", "batch", "num_kv_heads", "rows")
                            and not (fmt == L.TKA_KV_16BIT and "scale" in f) and not (f == "stride_b" and side == "prefix" and v > 0)
                            and not (fmt == L.TKA_KV_16BIT and v in (520, 136))], side)
        _refused(fn, make, [("format", 9, INVALID), ("num_kv_heads", 3, INVALID), ("rows", -1, INVALID), ("v", None, INVALID)], side)
    _refused(fn, make, [("batch", 2, INVALID)], "prefix")
    _refused(fn, make, [("batch", 0, INVALID)], "suffix")
    _refused(fn, make, [("q", None, INVALID), ("out", None, INVALID), ("dtype", 3, UNSUPPORTED), ("out_dtype", 3, UNSUPPORTED), ("group", 6, UNSUPPORTED),
                        ("num_splits", 513, INVALID), ("num_splits", -1, INVALID), ("q_stride_b", 128, INVALID), ("out_stride_b", 128, INVALID),
                        ("reserved0", 1, INVALID)])
    a = make()
    a.prefix.rows = a.suffix.rows = 0
    assert fn(C.byref(a)) == INVALID
    for side in ("prefix", "suffix"):        # one of the two may be empty, its pointers are then not looked at
        a = make()
        c = getattr(a, side)
        c.rows, c.k, c.v = 0, None, None
        assert fn(C.byref(a)) == L.TKA_EWORKSPACE
    a = make()
    a.prefix.format = a.suffix.format = 9
    assert fn(C.byref(a)) == UNSUPPORTED


def test_ops_refuse_cpu_tensors():
    q, k = torch.zeros(1, 8, 128, dtype=torch.float16), torch.zeros(1, 64, 8, 128, dtype=torch.float16)
    codes, scale = torch.zeros(1, 64, 8, 128, dtype=torch.int8), torch.zeros(1, 64, 8)
    with pytest.raises(ValueError):
        ops.QuantCache(codes, codes, scale, scale)
    with pytest.raises(ValueError):
        ops.prefix_decode(q, (k[0], k[0]), (k, k), 1.0)


def test_launches_stay_within_the_limit():
    """Calls whose rows would take more than 2^32 - 1 threads are refused before anything is launched."""
    lib = L.lib()
    a = _copy(L.KvqWriteArgs)      # 2^29 rows: 2^24 workgroups of 256 threads
    a.cache.batch, a.cache.num_kv_heads, a.num_tokens, a.stride_b, a.stride_n, a.stride_h = 1, 1, 1 << 29, 0, 0, 0
    assert lib.tka_kvq_write(C.byref(a)) == UNSUPPORTED
    a = _scores()                  # 2^32 rows of a shared cache
    a.cache.batch, a.cache.num_kv_heads, a.cache.rows, a.cache.stride_b, a.cache.scale_stride_b = 4096, 4, 1 << 18, 0, 0
    assert lib.tka_kvq_scores(C.byref(a)) == UNSUPPORTED
    for rows in (200, 1000):       # 2^23 query heads, one launch or two
        a = _decode()
        a.cache.batch, a.cache.num_kv_heads, a.cache.rows, a.group, a.cache.stride_b, a.cache.scale_stride_b = 32768, 256, rows, 1, 0, 0
        a.q_stride_b = a.out_stride_b = 256 * 128
        assert lib.tka_kvq_flash_decode(C.byref(a)) == UNSUPPORTED
        a.cache.batch = 32767
        assert lib.tka_kvq_flash_decode(C.byref(a)) == L.TKA_EWORKSPACE
        a = _prefix()
        a.prefix.rows, a.suffix.rows, a.suffix.batch, a.group = rows, 0, 32768, 1
        a.prefix.num_kv_heads = a.suffix.num_kv_heads = 256
        a.q_stride_b = a.out_stride_b = 256 * 128
        assert lib.tka_prefix_decode(C.byref(a)) == L.TKA_EWORKSPACE      # (blocks of query rows: fewer workgroups)
        a.suffix.batch, a.group = 32768, 4
        a.q_stride_b = a.out_stride_b = 1024 * 128
        assert lib.tka_prefix_decode(C.byref(a)) == UNSUPPORTED


def test_the_hook_is_checked():
    for n in (-1, 3, 5, 32):
        assert L.lib().tka_kvq_test_row_tiles(n) == INVALID
    assert L.lib().tka_kvq_test_row_tiles(0) == 0
