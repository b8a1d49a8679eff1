"""Torch-facing wrappers of the C ABI: device tensors in, device tensors out, nothing computed in Python.

PyTorch is used for device memory and the current stream only.  Every function raises if libtka.so is
missing or a call is rejected; there is no CPU or eager fallback.
"""
import ctypes as C

import torch

from . import _lib as L

_DT = {torch.float16: L.TKA_F16, torch.bfloat16: L.TKA_BF16}
_workspaces = {}


def _dtype_code(t):
    if t.dtype not in _DT:
        raise TypeError("expected float16 or bfloat16, got %s" % t.dtype)
    return _DT[t.dtype]


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _workspace(nbytes, device):
    """Workspace of the one-shot wrappers: one growing byte buffer per (device, stream), looked up by the stream the
    call is about to be launched on; calls on one stream are ordered, so they may share it.  Never grown during a
    graph capture (the allocation would belong to the capture's pool and be handed to later eager calls)."""
    key = (device.index, torch.cuda.current_stream().cuda_stream)
    buf = _workspaces.get(key)
    if buf is None or buf.numel() < nbytes:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the workspace of this stream must exist before a graph capture: call once eagerly, "
                               "or use a plan object (it owns its workspace)")
        buf = torch.empty(max(int(nbytes), 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[key] = buf
    return buf


def _own_workspace(nbytes, device):
    """Workspace of a plan object: its own buffer, so that plans run on different streams never share one."""
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


def _need_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("tensors must live on the GPU")


def _kv_strides(kv, batch):
    """kv is [N, H, 128] (shared by the batch) or [B, N, H, 128]; returns (stride_b, stride_n, stride_h, N, H)."""
    if kv.stride(-1) != 1 or kv.shape[-1] != 128:
        raise ValueError("last dim must be 128 and contiguous")
    if kv.dim() == 3:
        return 0, kv.stride(0), kv.stride(1), kv.shape[0], kv.shape[1]
    if kv.dim() == 4:
        if kv.shape[0] != batch:
            raise ValueError("batch mismatch")
        return kv.stride(0), kv.stride(1), kv.stride(2), kv.shape[1], kv.shape[2]
    raise ValueError("keys/values must be [N,H,128] or [B,N,H,128]")


def _q3(q):
    if q.dim() == 2:
        q = q.unsqueeze(0)
    if q.dim() != 3 or q.shape[-1] != 128 or q.stride(-1) != 1 or q.stride(1) != 128:
        raise ValueError("q must be [B,Hq,128] with contiguous heads")
    return q


class GemvTopkPlan:
    """Argument block, outputs and workspace of one fused GEMV + top-k configuration; run() is one C call."""

    def __init__(self, q, keys, k, group=1, scale=1.0, num_chunks=1, return_scores=False, score_mode=L.TKA_SCORE_CANONICAL):
        _need_cuda(q, keys)
        q = _q3(q)
        B = q.shape[0]
        sb, sn, sh, N, H = _kv_strides(keys, B)
        if q.shape[1] != H * group:
            raise ValueError("q heads != kv heads * group")
        self.q, self.keys = q, keys
        self.idx = torch.empty((B, H, num_chunks * k), dtype=torch.int32, device=q.device)
        self.val = torch.empty((B, H, num_chunks * k), dtype=torch.float32, device=q.device)
        self.scores = torch.empty((B, H, N), dtype=torch.float32, device=q.device) if return_scores else None
        a = L.GemvTopkArgs()
        a.q, a.keys = q.data_ptr(), keys.data_ptr()
        a.dtype, a.batch, a.num_kv_heads, a.group, a.head_dim = _dtype_code(keys), B, H, group, 128
        a.k, a.num_chunks, a.seq_len, a.score_mode = k, num_chunks, N, score_mode
        a.q_stride_b, a.key_stride_b, a.key_stride_n, a.key_stride_h = q.stride(0), sb, sn, sh
        a.scale = scale
        a.out_idx, a.out_val = self.idx.data_ptr(), self.val.data_ptr()
        a.out_scores = self.scores.data_ptr() if self.scores is not None else None
        need = L.lib().tka_gemv_topk_workspace_bytes(C.byref(a))
        self.ws = _own_workspace(need, q.device)
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        self.args = a
        self._fn = L.lib().tka_gemv_topk

    def run(self):
        self.args.stream = torch.cuda.current_stream().cuda_stream
        L.check(self._fn(C.byref(self.args)), "tka_gemv_topk")
        return self

    def redone_segments(self):
        """Diagnostic: segments of the last run() that the selection kernel had to redo from the keys."""
        n = C.c_int32(0)
        L.check(L.lib().tka_gemv_topk_redone_segments(C.byref(self.args), C.byref(n)), "tka_gemv_topk_redone_segments")
        return n.value

    def gave_up_slices(self):
        """Diagnostic: candidate slices of the last run() whose workgroup ran out of its wait for the threshold."""
        n = C.c_int32(0)
        L.check(L.lib().tka_gemv_topk_gave_up_slices(C.byref(self.args), C.byref(n)), "tka_gemv_topk_gave_up_slices")
        return n.value


def gemv_topk(q, keys, k, group=1, scale=1.0, num_chunks=1, return_scores=False, score_mode=L.TKA_SCORE_CANONICAL):
    """Fused GEMV + top-k.  Returns (idx int32 [B,Hkv,num_chunks*k], val fp32 same shape[, scores fp32 [B,Hkv,N]])."""
    plan = GemvTopkPlan(q, keys, k, group, scale, num_chunks, return_scores, score_mode).run()
    return (plan.idx, plan.val, plan.scores) if return_scores else (plan.idx, plan.val)


def gemv_scores(q, keys, group=1, scale=1.0, score_mode=L.TKA_SCORE_CANONICAL):
    """GEMV phase alone: fp32 scores [B,Hkv,N]."""
    _need_cuda(q, keys)
    q = _q3(q)
    B = q.shape[0]
    sb, sn, sh, N, H = _kv_strides(keys, B)
    scores = torch.empty((B, H, N), dtype=torch.float32, device=q.device)
    a = L.GemvTopkArgs()
    a.q, a.keys = q.data_ptr(), keys.data_ptr()
    a.dtype, a.batch, a.num_kv_heads, a.group, a.head_dim = _dtype_code(keys), B, H, group, 128
    a.k, a.num_chunks, a.seq_len, a.score_mode = 1, 1, N, score_mode
    a.q_stride_b, a.key_stride_b, a.key_stride_n, a.key_stride_h = q.stride(0), sb, sn, sh
    a.scale = scale
    a.out_scores = scores.data_ptr()
    a.stream = _stream()
    L.check(L.lib().tka_gemv_scores(C.byref(a)), "tka_gemv_scores")
    return scores


def topk(scores, k):
    """Selection phase alone on fp32 scores [S, N] (row stride free).  Returns (idx int32 [S,k], val fp32 [S,k])."""
    _need_cuda(scores)
    if scores.dim() == 1:
        scores = scores.unsqueeze(0)
    if scores.dtype != torch.float32 or scores.dim() != 2 or scores.stride(1) != 1:
        raise ValueError("scores must be fp32 [S,N] with contiguous rows")
    S, N = scores.shape
    idx = torch.empty((S, k), dtype=torch.int32, device=scores.device)
    val = torch.empty((S, k), dtype=torch.float32, device=scores.device)
    a = L.TopkArgs()
    a.scores, a.num_segments, a.k, a.seg_len = scores.data_ptr(), S, k, N
    a.seg_stride = scores.stride(0) if S > 1 else N
    a.out_idx, a.out_val = idx.data_ptr(), val.data_ptr()
    need = L.lib().tka_topk_workspace_bytes(C.byref(a))
    ws = _workspace(need, scores.device)
    a.workspace, a.workspace_bytes, a.stream = ws.data_ptr(), ws.numel(), _stream()
    L.check(L.lib().tka_topk_f32(C.byref(a)), "tka_topk_f32")
    return idx, val


class CenterTopkPlan:
    """Argument block, outputs and workspace of one centre-only selection; run() is one C call."""

    def __init__(self, q, centers, top_c, cluster_len, scale=1.0):
        _need_cuda(q, centers)
        if not centers.is_contiguous() or not q.is_contiguous():
            raise ValueError("q and centers must be contiguous")
        H, Cn, _ = centers.shape
        self.q, self.centers = q, centers
        self.out = torch.empty((H, top_c * cluster_len), dtype=torch.int32, device=q.device)
        self.cen = torch.empty((H, top_c), dtype=torch.int32, device=q.device)
        self.val = torch.empty((H, top_c), dtype=torch.float32, device=q.device)
        a = self.args = L.CenterTopkArgs()
        a.q, a.centers, a.dtype = q.data_ptr(), centers.data_ptr(), _dtype_code(centers)
        a.num_heads, a.num_centers, a.top_c, a.cluster_len, a.head_dim = H, Cn, top_c, cluster_len, 128
        a.scale = scale
        a.out_idx, a.out_centers, a.out_center_val = self.out.data_ptr(), self.cen.data_ptr(), self.val.data_ptr()
        need = L.lib().tka_center_topk_expand_workspace_bytes(C.byref(a))
        self.ws = _own_workspace(need, q.device)
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()

    def run(self):
        self.args.stream = _stream()
        L.check(L.lib().tka_center_topk_expand(C.byref(self.args)), "tka_center_topk_expand")
        return self


def center_topk_expand(q, centers, top_c, cluster_len, scale=1.0):
    """Centre-only selection.  q [H,128], centers [H,C,128] contiguous.
    Returns (token ids int32 [H, top_c*cluster_len], centre ids int32 [H,top_c], centre scores fp32 [H,top_c])."""
    plan = CenterTopkPlan(q, centers, top_c, cluster_len, scale).run()
    return plan.out, plan.cen, plan.val


def cluster_gemv_topk(q, centers, keys, top_c, cluster_len, k, scale=1.0):
    """Two-level selection.  q [H,128], centers [H,C,128], keys [C*cluster_len, H, 128].  Returns int32 [H, top_c*k]."""
    _need_cuda(q, centers, keys)
    H, Cn, _ = centers.shape
    out = torch.empty((H, top_c * k), dtype=torch.int32, device=q.device)
    a = L.ClusterTopkArgs()
    a.q, a.centers, a.keys, a.dtype = q.data_ptr(), centers.data_ptr(), keys.data_ptr(), _dtype_code(keys)
    a.num_heads, a.num_centers, a.top_c, a.cluster_len, a.k, a.head_dim = H, Cn, top_c, cluster_len, k, 128
    a.scale = scale
    a.key_stride_n, a.key_stride_h = keys.stride(0), keys.stride(1)
    a.out_idx = out.data_ptr()
    need = L.lib().tka_cluster_gemv_topk_workspace_bytes(C.byref(a))
    ws = _workspace(need, q.device)
    a.workspace, a.workspace_bytes, a.stream = ws.data_ptr(), ws.numel(), _stream()
    L.check(L.lib().tka_cluster_gemv_topk(C.byref(a)), "tka_cluster_gemv_topk")
    return out


def index_union(idx, sink, local, seq_len):
    """idx int32 [..., k] -> (union int32 [..., k+sink+local] ascending, -1 padded; count int32 [...])."""
    _need_cuda(idx)
    idx = idx.contiguous()
    k = idx.shape[-1]
    S = idx.numel() // k
    out = torch.empty(idx.shape[:-1] + (k + sink + local,), dtype=torch.int32, device=idx.device)
    cnt = torch.empty(idx.shape[:-1], dtype=torch.int32, device=idx.device)
    a = L.IndexUnionArgs()
    a.idx, a.num_segments, a.k, a.sink, a.local, a.seq_len = idx.data_ptr(), S, k, sink, local, seq_len
    a.out_idx, a.out_count, a.stream = out.data_ptr(), cnt.data_ptr(), _stream()
    L.check(L.lib().tka_index_union(C.byref(a)), "tka_index_union")
    return out, cnt


class FlashDecodePlan:
    """Argument block, output and workspace of one split-K decode configuration; run() is one C call."""

    def __init__(self, q, keys, values, scale, group=1, num_splits=0, kv_idx=None, kv_count=None, kv_logit=None,
                 out_dtype=None, return_lse=False, softmax_mode=L.TKA_SOFTMAX_SCALED):
        _need_cuda(q, keys, values, kv_idx, kv_count, kv_logit)
        q = _q3(q)
        B = q.shape[0]
        sb, sn, sh, N, H = _kv_strides(keys, B)
        if _kv_strides(values, B) != (sb, sn, sh, N, H):
            raise ValueError("keys and values must share shape and strides")
        out_dtype = out_dtype or q.dtype
        self.q, self.keys, self.values = q, keys, values
        self.out = torch.empty((B, H * group, 128), dtype=out_dtype, device=q.device)
        self.lse = torch.empty((B, H * group), dtype=torch.float32, device=q.device) if return_lse else None
        a = L.FlashDecodeArgs()
        a.q, a.keys, a.values, a.out = q.data_ptr(), keys.data_ptr(), values.data_ptr(), self.out.data_ptr()
        a.dtype, a.out_dtype = _dtype_code(keys), _DT[out_dtype]
        a.batch, a.num_kv_heads, a.group, a.head_dim = B, H, group, 128
        a.num_splits, a.softmax_mode = num_splits, softmax_mode
        a.seq_len, a.q_stride_b, a.out_stride_b = N, q.stride(0), self.out.stride(0)
        a.kv_stride_b, a.kv_stride_n, a.kv_stride_h = sb, sn, sh
        a.scale = scale
        if kv_idx is not None:
            self.kv_idx = kv_idx.contiguous()
            a.idx_len, a.kv_idx = self.kv_idx.shape[-1], self.kv_idx.data_ptr()
            if kv_count is not None:
                self.kv_count = kv_count.contiguous()
                a.kv_count = self.kv_count.data_ptr()
            if kv_logit is not None:
                self.kv_logit = kv_logit.contiguous()
                a.kv_logit = self.kv_logit.data_ptr()
        a.out_lse = self.lse.data_ptr() if self.lse is not None else None
        need = L.lib().tka_flash_decode_workspace_bytes(C.byref(a))
        self.ws = _own_workspace(need, q.device)
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        self.args = a
        self._fn = L.lib().tka_flash_decode

    def run(self):
        self.args.stream = torch.cuda.current_stream().cuda_stream
        L.check(self._fn(C.byref(self.args)), "tka_flash_decode")
        return self


def flash_decode(q, keys, values, scale, group=1, num_splits=0, kv_idx=None, kv_count=None, kv_logit=None,
                 out_dtype=None, return_lse=False, softmax_mode=L.TKA_SOFTMAX_SCALED):
    """Split-K decode attention (dense, or over kv_idx [B,Hkv,L]).  Returns out [B,Hq,128] (and LSE fp32 [B,Hq])."""
    plan = FlashDecodePlan(q, keys, values, scale, group, num_splits, kv_idx, kv_count, kv_logit, out_dtype,
                           return_lse, softmax_mode).run()
    return (plan.out, plan.lse) if return_lse else plan.out


def lse_combine(part_m, part_l, part_acc, out_dtype=torch.float16, return_lse=False):
    """part_m, part_l fp32 [R,S]; part_acc fp32 [R,S,128] -> out [R,128]."""
    _need_cuda(part_m, part_l, part_acc)
    part_m, part_l, part_acc = part_m.contiguous(), part_l.contiguous(), part_acc.contiguous()
    R, S = part_m.shape
    out = torch.empty((R, 128), dtype=out_dtype, device=part_m.device)
    lse = torch.empty((R,), dtype=torch.float32, device=part_m.device) if return_lse else None
    a = L.LseCombineArgs()
    a.part_m, a.part_l, a.part_acc = part_m.data_ptr(), part_l.data_ptr(), part_acc.data_ptr()
    a.rows, a.num_splits, a.out_dtype = R, S, _DT[out_dtype]
    a.out = out.data_ptr()
    a.out_lse = lse.data_ptr() if lse is not None else None
    a.stream = _stream()
    L.check(L.lib().tka_lse_combine(C.byref(a)), "tka_lse_combine")
    return (out, lse) if return_lse else out


def retrieval_attention(q, k, v, out, topk, num_chunks=4, scale=1.0, softmax_mode=L.TKA_SOFTMAX_RAW_EXP,
                        bench_print=False, score_mode=L.TKA_SCORE_CANONICAL):
    """The reference op, general form: q [B,H,128], k/v [N,H,128] contiguous, writes out [B,H,128] in place."""
    _need_cuda(q, k, v, out)
    for t in (q, k, v, out):
        if not t.is_contiguous():
            raise ValueError("retrieval_attention expects contiguous tensors")
    if out.dtype != q.dtype or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k, v, out must share one dtype")
    B, H, _ = q.shape
    a = L.RaArgs()
    a.q, a.keys, a.values, a.out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
    a.dtype, a.batch, a.num_heads, a.head_dim = _dtype_code(q), B, H, 128
    a.topk_per_chunk, a.num_chunks, a.softmax_mode, a.bench_print = topk, num_chunks, softmax_mode, int(bench_print)
    a.seq_len, a.scale, a.score_mode = k.shape[0], scale, score_mode
    need = L.lib().tka_retrieval_attention_workspace_bytes(C.byref(a))
    ws = _workspace(need, q.device)
    a.workspace, a.workspace_bytes, a.stream = ws.data_ptr(), ws.numel(), _stream()
    L.check(L.lib().tka_retrieval_attention(C.byref(a)), "tka_retrieval_attention")
    return out


class SparseDecodePlan:
    """Holds the argument block, outputs and workspace of one end-to-end decode configuration so that
    a step is a single C call (used by the benchmark and by callers that decode repeatedly)."""

    def __init__(self, q, keys, values, k, sink, local, scale, group, out_dtype=None, num_splits=0,
                 want_topk=True, want_union=True):
        _need_cuda(q, keys, values)
        q = _q3(q)
        B = q.shape[0]
        sb, sn, sh, N, H = _kv_strides(keys, B)
        if _kv_strides(values, B) != (sb, sn, sh, N, H):
            raise ValueError("keys and values must share shape and strides")
        out_dtype = out_dtype or q.dtype
        self.q, self.keys, self.values = q, keys, values
        self.out = torch.empty((B, H * group, 128), dtype=out_dtype, device=q.device)
        a = L.SparseDecodeArgs()
        a.q, a.keys, a.values, a.out = q.data_ptr(), keys.data_ptr(), values.data_ptr(), self.out.data_ptr()
        a.dtype, a.out_dtype = _dtype_code(keys), _DT[out_dtype]
        a.batch, a.num_kv_heads, a.group, a.head_dim = B, H, group, 128
        a.k, a.sink, a.local, a.num_splits = k, sink, local, num_splits
        a.seq_len, a.q_stride_b, a.out_stride_b = N, q.stride(0), self.out.stride(0)
        a.kv_stride_b, a.kv_stride_n, a.kv_stride_h = sb, sn, sh
        a.scale = scale
        self.topk_idx = self.topk_val = self.union_idx = self.union_count = None
        if want_topk:  # rank-ordered selection: costs a sort per KV head, not needed by the attention
            self.topk_idx = torch.empty((B, H, k), dtype=torch.int32, device=q.device)
            self.topk_val = torch.empty((B, H, k), dtype=torch.float32, device=q.device)
            a.out_topk_idx, a.out_topk_val = self.topk_idx.data_ptr(), self.topk_val.data_ptr()
        if want_union:
            self.union_idx = torch.empty((B, H, k + sink + local), dtype=torch.int32, device=q.device)
            self.union_count = torch.empty((B, H), dtype=torch.int32, device=q.device)
            a.out_union_idx, a.out_union_count = self.union_idx.data_ptr(), self.union_count.data_ptr()
        need = L.lib().tka_sparse_decode_workspace_bytes(C.byref(a))
        if need == 0:
            L.check(L.lib().tka_sparse_decode_step(C.byref(a)), "tka_sparse_decode_step")
        self.ws = torch.empty(need, dtype=torch.uint8, device=q.device)
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        self.args = a
        self._fn = L.lib().tka_sparse_decode_step

    def step(self):
        self.args.stream = torch.cuda.current_stream().cuda_stream
        rc = self._fn(C.byref(self.args))
        if rc != L.TKA_OK:
            L.check(rc, "tka_sparse_decode_step")
        return self.out

    def redone_segments(self):
        """Diagnostic: segments of the last step() that the selection kernel had to redo from the keys."""
        n = C.c_int32(0)
        L.check(L.lib().tka_sparse_decode_redone_segments(C.byref(self.args), C.byref(n)), "tka_sparse_decode_redone_segments")
        return n.value


def sparse_decode_step(q, keys, values, k, sink, local, scale, group, out_dtype=None, num_splits=0, want_topk=True):
    """End-to-end decode step.  Returns (out, topk_idx, topk_val, union_idx, union_count); without want_topk the
    rank-ordered selection is not produced (None)."""
    plan = SparseDecodePlan(q, keys, values, k, sink, local, scale, group, out_dtype, num_splits, want_topk=want_topk)
    plan.step()
    return plan.out, plan.topk_idx, plan.topk_val, plan.union_idx, plan.union_count


# ---- 8-bit K/V caches and shared prefixes (include/topk_attn_kvq.h) --------------------------------

_KV_FORMAT = {torch.float8_e4m3fn: L.TKA_KV_E4M3, torch.int8: L.TKA_KV_INT8}


def _one_device(*tensors):
    """Index of the GPU that all the tensors (None aside) live on."""
    _need_cuda(*tensors)
    devices = {t.device for t in tensors if t is not None}
    if len(devices) != 1:
        raise ValueError("tensors must live on one GPU, got %s" % sorted(map(str, devices)))
    return devices.pop().index


# The handle of a device's current stream: torch.cuda.current_stream() makes an object of it (2.6 us), the call it is made
# from takes 0.1 us, where this torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _call(fn, args, device, where):
    """One C call on the current stream of `device` (which need not be the current device)."""
    args.stream = _raw_stream(device)
    if torch.cuda.current_device() == device:
        rc = fn(C.byref(args))
    else:
        with torch.cuda.device(device):
            rc = fn(C.byref(args))
    if rc != L.TKA_OK:
        L.check(rc, where)


def _need_workspace(need, fn, args, where):
    """The C side's reason for a workspace size of zero (its checks come before any launch)."""
    if need == 0:
        L.check(fn(C.byref(args)) or L.TKA_EINVAL, where)


def _strides(t, dims):
    """Strides of a tensor's dims in elements; a dim of size 1 has none that matters."""
    return [0 if t.shape[d] == 1 else t.stride(d) for d in dims]


def _alike(a, b):
    """Same shape, and the same strides where they matter."""
    return a.shape == b.shape and _strides(a, range(a.dim())) == _strides(b, range(b.dim()))


def _int32(t, shape, name):
    if t is None:
        return None
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError("%s must be int32 %s, contiguous" % (name, list(shape)))
    return t


def _rows4(t, name):
    """[N,H,128] (shared by a batch) or [B,N,H,128] with contiguous rows -> the 4-dim view."""
    if t.dim() not in (3, 4) or t.shape[-1] != 128 or t.stride(-1) != 1:
        raise ValueError("%s must be [N,H,128] or [B,N,H,128] with a contiguous last dim" % name)
    return t if t.dim() == 4 else t.unsqueeze(0)


def _fill_cache(c, fmt, k, v, batch, shared):
    """tka_kv_cache of 4-dim tensors; `shared`: entry 0 serves every entry of the batch."""
    c.k, c.v, c.format = k.data_ptr(), (v.data_ptr() if v is not None else None), fmt
    c.batch, c.rows, c.num_kv_heads, c.head_dim = batch, k.shape[1], k.shape[2], 128
    c.stride_b, c.stride_n, c.stride_h = _strides(k, (0, 1, 2))
    if shared:
        c.stride_b = 0


class QuantCache:
    """K/V cache of 8-bit rows: codes [B,N,H,128] (or [N,H,128], one cache that a batch shares) in torch.float8_e4m3fn or
    torch.int8 - the dtype names the format - and one fp32 scale per row, [B,N,H] (or [N,H]).  Any strides with 16-byte
    aligned rows; keys and values share theirs.  v_codes / v_scale may be None where only scores are taken."""

    def __init__(self, k_codes, v_codes, k_scale, v_scale):
        self.device = _one_device(k_codes, v_codes, k_scale, v_scale)
        if k_codes.dtype not in _KV_FORMAT:
            raise TypeError("codes must be float8_e4m3fn or int8, got %s" % k_codes.dtype)
        self.shared = k_codes.dim() == 3
        if (v_codes is None) != (v_scale is None):
            raise ValueError("v_codes and v_scale go together")
        for codes, scale, name in ((k_codes, k_scale, "k"), (v_codes, v_scale, "v")):
            if codes is None:
                continue
            _rows4(codes, name + "_codes")
            if codes.dtype != k_codes.dtype or not _alike(codes, k_codes):
                raise ValueError("keys and values must share dtype, shape and strides")
            if scale.dtype != torch.float32 or scale.shape != codes.shape[:-1]:
                raise ValueError("%s_scale must be float32 %s" % (name, list(codes.shape[:-1])))
            if not _alike(scale, k_scale):
                raise ValueError("the scales of keys and values must share strides")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.format = _KV_FORMAT[k_codes.dtype]
        self.batch = 1 if self.shared else k_codes.shape[0]
        self.rows, self.heads = k_codes.shape[-3], k_codes.shape[-2]

    @classmethod
    def empty(cls, batch, rows, heads, dtype=torch.float8_e4m3fn, device="cuda"):
        """A cache of zeros for `batch` entries of `rows` tokens, head by head (a head's rows and scales are contiguous:
        the layout that the kernels stream best).  batch None: one cache [N,H,128] that a batch shares."""
        n = 1 if batch is None else batch
        codes = [torch.zeros((n, heads, rows, 128), dtype=torch.uint8, device=device).view(dtype).transpose(1, 2) for _ in range(2)]
        scale = [torch.zeros((n, heads, rows), dtype=torch.float32, device=device).transpose(1, 2) for _ in range(2)]
        if batch is None:
            codes, scale = [c[0] for c in codes], [s[0] for s in scale]
        return cls(codes[0], codes[1], scale[0], scale[1])

    def _fill(self, c, batch):
        """The C description for a call of `batch` entries."""
        if not self.shared and self.batch != batch:
            raise ValueError("batch mismatch: cache %d, call %d" % (self.batch, batch))
        k, ks = (self.k_codes, self.k_scale) if not self.shared else (self.k_codes.unsqueeze(0), self.k_scale.unsqueeze(0))
        _fill_cache(c, self.format, k, self.v_codes, batch, self.shared)
        c.k_scale, c.v_scale = ks.data_ptr(), (self.v_scale.data_ptr() if self.v_scale is not None else None)
        c.scale_stride_b, c.scale_stride_n, c.scale_stride_h = _strides(ks, (0, 1, 2))
        if self.shared:
            c.scale_stride_b = 0

    def _need_values(self):
        if self.v_codes is None:
            raise ValueError("this call needs the values of the cache")


class _KvqCopyPlan:
    """What the write and the read plan share: rows k, v [B,T,H,128] on the 16-bit side."""

    def __init__(self, args, fn, where, cache, k, v, start, count):
        cache._need_values()
        self._device = _one_device(cache.k_codes, k, v, start, count)
        for t in (k, v):
            if t.dim() != 4 or t.shape[-1] != 128 or t.stride(-1) != 1:
                raise ValueError("k and v must be [B,T,H,128] with a contiguous last dim")
        B, T, H, _ = k.shape
        if v.dtype != k.dtype or not _alike(k, v):
            raise ValueError("k and v must share dtype, shape and strides")
        if H != cache.heads or B != cache.batch:
            raise ValueError("k and v do not match the cache's batch entries or heads")
        self.cache, self.k, self.v = cache, k, v
        self.start, self.count = _int32(start, (B,), "start"), _int32(count, (B,), "count")
        a = self.args = args
        cache._fill(a.cache, B)
        a.k, a.v, a.dtype, a.num_tokens = k.data_ptr(), v.data_ptr(), _dtype_code(k), T
        a.stride_b, a.stride_n, a.stride_h = _strides(k, (0, 1, 2))
        a.start = start.data_ptr() if start is not None else None
        a.count = count.data_ptr() if count is not None else None
        self._fn, self._where = fn, where

    def run(self):
        _call(self._fn, self.args, self._device, self._where)
        return self


class KvqWritePlan(_KvqCopyPlan):
    """Quantises rows k, v [B,T,H,128] into a QuantCache: row t of entry b goes to row start[b] + t (start None: 0) for
    t < count[b] (None: T); start and count are int32 [B] on the GPU.  run() is one C call; what k, v, start and count
    hold when it runs counts."""

    def __init__(self, cache, k, v, start=None, count=None):
        super().__init__(L.KvqWriteArgs(), L.lib().tka_kvq_write, "tka_kvq_write", cache, k, v, start, count)


class KvqReadPlan(_KvqCopyPlan):
    """The other way: rows start[b] + t of a QuantCache as 16-bit numbers in k, v [B,T,H,128]; rows behind count[b], and
    rows that the cache does not have, keep what they hold."""

    def __init__(self, cache, k, v, start=None, count=None):
        super().__init__(L.KvqReadArgs(), L.lib().tka_kvq_read, "tka_kvq_read", cache, k, v, start, count)


def kvq_write(cache, k, v, start=None, count=None):
    """Quantise k, v [B,T,H,128] into a QuantCache (see KvqWritePlan)."""
    KvqWritePlan(cache, k, v, start, count).run()
    return cache


def kvq_read(cache, num_tokens, start=None, count=None, dtype=torch.bfloat16):
    """Rows of a QuantCache as 16-bit numbers: (k, v) [B,num_tokens,H,128], zeros where there is no row."""
    cache._need_values()
    shape = (cache.batch, num_tokens, cache.heads, 128)
    k, v = (torch.zeros(shape, dtype=dtype, device=cache.k_codes.device) for _ in range(2))
    KvqReadPlan(cache, k, v, start, count).run()
    return k, v


class KvqScoresPlan:
    """Stage-1 scores over the keys of a QuantCache: scores fp32 [B,Hkv,N], -inf behind kv_len[b] (int32 [B] on the GPU;
    None: all rows).  What topk() selects from; run() is one C call."""

    def __init__(self, q, cache, scale=1.0, group=1, kv_len=None):
        self._device = _one_device(q, cache.k_codes, kv_len)
        q = _q3(q)
        B = q.shape[0]
        if q.shape[1] != cache.heads * group:
            raise ValueError("q heads != kv heads * group")
        self.q, self.cache, self.kv_len = q, cache, _int32(kv_len, (B,), "kv_len")
        a = self.args = L.KvqScoresArgs()
        cache._fill(a.cache, B)
        a.q, a.dtype, a.group, a.q_stride_b, a.scale = q.data_ptr(), _dtype_code(q), group, _strides(q, (0,))[0], scale
        a.kv_len = kv_len.data_ptr() if kv_len is not None else None
        self.scores = torch.empty((B, cache.heads, cache.rows), dtype=torch.float32, device=q.device)
        a.out_scores = self.scores.data_ptr()
        self._fn = L.lib().tka_kvq_scores

    def run(self):
        _call(self._fn, self.args, self._device, "tka_kvq_scores")
        return self


def kvq_scores(q, cache, scale=1.0, group=1, kv_len=None):
    """Scores fp32 [B,Hkv,N] over a QuantCache's keys (see KvqScoresPlan)."""
    return KvqScoresPlan(q, cache, scale, group, kv_len).run().scores


class _DecodeOutputs:
    """Outputs and workspace of a decode plan."""

    def _finish(self, a, q, out_dtype, return_lse, need, fn, where):
        B, Hq, _ = q.shape
        if out_dtype not in _DT:
            raise TypeError("expected float16 or bfloat16, got %s" % out_dtype)
        self.out = torch.empty((B, Hq, 128), dtype=out_dtype, device=q.device)
        self.lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device) if return_lse else None
        a.out, a.out_dtype, a.out_stride_b = self.out.data_ptr(), _DT[out_dtype], Hq * 128
        a.out_lse = self.lse.data_ptr() if return_lse else None
        size = need(C.byref(a))
        _need_workspace(size, fn, a, where)
        self.ws = _own_workspace(size, q.device)
        a.workspace, a.workspace_bytes = self.ws.data_ptr(), self.ws.numel()
        self._fn, self._where = fn, where

    def run(self):
        _call(self._fn, self.args, self._device, self._where)
        return self


class KvqFlashDecodePlan(_DecodeOutputs):
    """Argument block, output and workspace of one decode step of attention over a QuantCache: over its first kv_len[b]
    rows (int32 [B]; None: all), or over the rows listed in kv_idx int32 [B,Hkv,L] (the first kv_count[b,h] entries of
    each list; ids outside the cache or behind kv_len are skipped).  A query without a row gets zeros, its lse is -inf.
    run() is one C call; a plan runs on one stream at a time."""

    def __init__(self, q, cache, scale, group=1, num_splits=0, kv_len=None, kv_idx=None, kv_count=None, out_dtype=None,
                 return_lse=False):
        cache._need_values()
        self._device = _one_device(q, cache.k_codes, kv_len, kv_idx, kv_count)
        q = _q3(q)
        B, H = q.shape[0], cache.heads
        if q.shape[1] != H * group:
            raise ValueError("q heads != kv heads * group")
        if kv_idx is not None and (kv_idx.dim() != 3 or kv_idx.shape[-1] < 1):
            raise ValueError("kv_idx must be int32 [B,Hkv,L]")
        self.q, self.cache = q, cache
        self.kv_len = _int32(kv_len, (B,), "kv_len")
        self.kv_idx = _int32(kv_idx, (B, H, kv_idx.shape[-1] if kv_idx is not None else 0), "kv_idx")
        self.kv_count = _int32(kv_count, (B, H), "kv_count")
        a = self.args = L.KvqFlashDecodeArgs()
        cache._fill(a.cache, B)
        a.q, a.dtype, a.group, a.q_stride_b = q.data_ptr(), _dtype_code(q), group, _strides(q, (0,))[0]
        a.num_splits, a.scale = num_splits, scale
        a.kv_len = kv_len.data_ptr() if kv_len is not None else None
        if kv_idx is not None:
            a.kv_idx, a.idx_len = kv_idx.data_ptr(), kv_idx.shape[-1]
        a.kv_count = kv_count.data_ptr() if kv_count is not None else None
        self._finish(a, q, out_dtype or q.dtype, return_lse, L.lib().tka_kvq_flash_decode_workspace_bytes,
                     L.lib().tka_kvq_flash_decode, "tka_kvq_flash_decode")


def kvq_flash_decode(q, cache, scale, group=1, num_splits=0, kv_len=None, kv_idx=None, kv_count=None, out_dtype=None,
                     return_lse=False):
    """Decode attention over a QuantCache (see KvqFlashDecodePlan).  Returns out [B,Hq,128] (and lse fp32 [B,Hq])."""
    plan = KvqFlashDecodePlan(q, cache, scale, group, num_splits, kv_len, kv_idx, kv_count, out_dtype, return_lse).run()
    return (plan.out, plan.lse) if return_lse else plan.out


class PrefixDecodePlan(_DecodeOutputs):
    """One decode step of a batch whose sequences share a prefix and go on with a suffix each: the prefix is read once for
    the batch.  prefix and suffix are QuantCaches of one dtype, or pairs (keys, values) of 16-bit tensors of q's dtype:
    the prefix [P,H,128] (or a batch of one), the suffix [B,S,H,128].  Either may be None.  suffix_len: int32 [B], the rows
    of each suffix (None: S).  run() is one C call; a plan runs on one stream at a time."""

    def __init__(self, q, prefix, suffix, scale, group=1, suffix_len=None, num_splits=0, out_dtype=None, return_lse=False):
        q = _q3(q)
        B = q.shape[0]
        a = self.args = L.PrefixDecodeArgs()
        if prefix is None and suffix is None:
            raise ValueError("neither a prefix nor a suffix")
        tensors, formats = [q, suffix_len], set()
        for source, c, name, batch in ((prefix, a.prefix, "prefix", 1), (suffix, a.suffix, "suffix", B)):
            if source is None:
                continue
            if isinstance(source, QuantCache):
                source._need_values()
                if name == "suffix" and source.shared:
                    raise ValueError("the suffix must be [B,S,H,128]")
                source._fill(c, batch)
                tensors += [source.k_codes, source.v_codes]
            else:
                k, v = source
                if k.dtype != q.dtype or v.dtype != q.dtype:
                    raise TypeError("16-bit caches must have q's dtype")
                if not _alike(k, v):
                    raise ValueError("keys and values must share shape and strides")
                if name == "suffix" and k.dim() != 4:
                    raise ValueError("the suffix must be [B,S,H,128]")
                k4 = _rows4(k, name)
                if k4.shape[0] != batch:
                    raise ValueError("%s: batch mismatch" % name)
                _fill_cache(c, L.TKA_KV_16BIT, k4, v, batch, False)
                tensors += [k, v]
            if q.shape[1] != c.num_kv_heads * group:
                raise ValueError("q heads != kv heads * group")
            formats.add(c.format)
        if len(formats) != 1:
            raise ValueError("prefix and suffix must have one format")
        for source, c, batch in ((prefix, a.prefix, 1), (suffix, a.suffix, B)):
            if source is None:
                c.format, c.batch, c.rows, c.num_kv_heads, c.head_dim = formats.copy().pop(), batch, 0, q.shape[1] // group, 128
        self._device = _one_device(*tensors)
        self.q, self.prefix, self.suffix, self.suffix_len = q, prefix, suffix, _int32(suffix_len, (B,), "suffix_len")
        a.q, a.dtype, a.group, a.q_stride_b = q.data_ptr(), _dtype_code(q), group, _strides(q, (0,))[0]
        a.num_splits, a.scale = num_splits, scale
        a.suffix_len = suffix_len.data_ptr() if suffix_len is not None else None
        self._finish(a, q, out_dtype or q.dtype, return_lse, L.lib().tka_prefix_decode_workspace_bytes,
                     L.lib().tka_prefix_decode, "tka_prefix_decode")


def prefix_decode(q, prefix, suffix, scale, group=1, suffix_len=None, num_splits=0, out_dtype=None, return_lse=False):
    """Decode attention of a batch behind a shared prefix (see PrefixDecodePlan).  Returns out [B,Hq,128] (and lse)."""
    plan = PrefixDecodePlan(q, prefix, suffix, scale, group, suffix_len, num_splits, out_dtype, return_lse).run()
    return (plan.out, plan.lse) if return_lse else plan.out


def set_test_hooks(force_segment_redo=0, tau_spin_limit=0, tau_withhold_mod=0, tau_withhold_rem=0, tau_withhold_mode=0,
                   union_handoff_order=0, fused_tail=0):
    """Testing hooks (see tka_test_hooks in include/topk_attn.h); no arguments = defaults."""
    h = L.TestHooks(force_segment_redo, tau_spin_limit, tau_withhold_mod, tau_withhold_rem, tau_withhold_mode, union_handoff_order,
                    fused_tail)
    L.check(L.lib().tka_set_test_hooks(C.byref(h)), "tka_set_test_hooks")


class ReadProbe:
    """A kernel that only reads a KV cache in the access pattern of the long-segment GEMV (`stream`) or of the gathered
    attention (`gather`, over idx [B,H,L]): what the memory system gives to that pattern (tka_probe_read)."""

    def __init__(self, keys, values=None, idx=None, threads=512, rounds=2, nontemporal=True, tokens_per_wg=256):
        _need_cuda(keys)
        B = keys.shape[0] if keys.dim() == 4 else 1
        sb, sn, sh, N, H = _kv_strides(keys, B)
        self.keep = (keys, values, idx)
        self.sink = torch.zeros(1, dtype=torch.int32, device=keys.device)
        a = L.ProbeArgs()
        a.keys, a.sink = keys.data_ptr(), self.sink.data_ptr()
        a.kind = L.TKA_PROBE_STREAM if idx is None else L.TKA_PROBE_GATHER
        a.batch, a.num_kv_heads, a.seq_len = B, H, N
        a.kv_stride_b, a.kv_stride_n, a.kv_stride_h = sb, sn, sh
        a.threads, a.rounds, a.nontemporal, a.tokens_per_wg = threads, rounds, int(nontemporal), tokens_per_wg
        if idx is not None:
            if values is None or _kv_strides(values, B) != (sb, sn, sh, N, H) or idx.dtype != torch.int32 or not idx.is_contiguous():
                raise ValueError("gather probe: values like keys, idx int32 [B,H,L] contiguous")
            a.values, a.idx, a.idx_len = values.data_ptr(), idx.data_ptr(), idx.shape[-1]
        self.args = a

    def run(self):
        self.args.stream = _stream()
        L.check(L.lib().tka_probe_read(C.byref(self.args)), "tka_probe_read")
        return self


def profile_enable(on=True):
    L.lib().tka_profile_enable(int(on))


def profile_reset():
    L.lib().tka_profile_reset()


def profile_read():
    """{kernel name: (total_ms, launches)} since the last reset (synchronises the recorded events)."""
    cap = 64
    names = (C.c_char_p * cap)()
    ms = (C.c_double * cap)()
    n_l = (C.c_int64 * cap)()
    n = L.lib().tka_profile_read(names, ms, n_l, cap)
    return {names[i].decode(): (ms[i], n_l[i]) for i in range(n)}
