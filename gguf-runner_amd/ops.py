"""Device-pointer entry points of libgr_attn for torch tensors resident in HBM.

torch is used only for device memory and the stream handle; every computation
is a HIP kernel of libgr_attn.so reached through the C ABI (see ffi.py).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import ffi

_DT = {torch.float32: ffi.DTYPE_F32, torch.float16: ffi.DTYPE_F16, torch.bfloat16: ffi.DTYPE_BF16,
       torch.int8: ffi.DTYPE_Q8}


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("libgr_attn device entry points take device tensors")
    return t.data_ptr()


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _workspace(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256) + 256, dtype=torch.uint8, device=device)


def _aligned(ws: torch.Tensor) -> int:
    p = ws.data_ptr()
    return (p + 255) // 256 * 256


def _set_gate(a, gate, row_stride, head_stride) -> None:
    """The optional Qwen3.5 output gate (an f32 device tensor, or None): element
    (row r, head h, i) at r * row_stride + h * head_stride + i of gate's storage."""
    if gate is None:
        return
    assert gate.dtype == torch.float32 and gate.is_cuda
    a.out_gate = _ptr(gate)
    a.out_gate_row_stride = int(row_stride)
    a.out_gate_head_stride = int(head_stride)


class DecodeCall:
    """A prepared gr_decode_attention call (args + workspace), reusable for timing.

    q [n_seq][Hq][d] f32; k_cache/v_cache [n_seq][seq_len][Hkv][d] (f32/f16/bf16, or
    int8 Q8 codes with f32 k_scale/v_scale [n_seq][seq_len] (one per row) or
    [n_seq][seq_len][Hkv*d/32] (q8_block: one per 32 elements));
    kv_start/kv_end int32 [n_seq]; out [n_seq][Hq][d] f32.
    """

    def __init__(self, q, k_cache, v_cache, kv_start, kv_end, out, *, max_kv_len,
                 score_scale=None, split_keys=0, k_scale=None, v_scale=None, q8_block=False,
                 out_gate=None, out_gate_row_stride=0, out_gate_head_stride=0):
        n_seq, n_heads, d = q.shape
        _, seq_len, n_kv, d2 = k_cache.shape
        assert d2 == d and v_cache.shape == k_cache.shape and out.shape == q.shape
        assert q.dtype == torch.float32 and out.dtype == torch.float32
        assert kv_start.dtype == torch.int32 and kv_end.dtype == torch.int32
        assert k_cache.is_contiguous() and v_cache.is_contiguous() and q.is_contiguous()
        self._keep = (q, k_cache, v_cache, kv_start, kv_end, out, k_scale, v_scale)
        a = ffi.DecodeArgs()
        a.n_seq, a.n_heads, a.n_kv_heads, a.head_dim = n_seq, n_heads, n_kv, d
        a.kv_dtype = _DT[k_cache.dtype]
        a.split_keys = split_keys
        a.max_kv_len = int(max_kv_len)
        a.score_scale = 1.0 / math.sqrt(d) if score_scale is None else float(score_scale)
        a.q, a.k_cache, a.v_cache = _ptr(q), _ptr(k_cache), _ptr(v_cache)
        a.seq_stride = seq_len * n_kv * d
        a.row_stride = n_kv * d
        a.kv_start, a.kv_end, a.out = _ptr(kv_start), _ptr(kv_end), _ptr(out)
        if k_cache.dtype == torch.int8:
            per_row = n_kv * d // 32 if q8_block else 1
            for t in (k_scale, v_scale):
                assert t is not None and t.dtype == torch.float32 and t.is_contiguous()
                assert t.numel() == n_seq * seq_len * per_row
            a.k_scale, a.v_scale = _ptr(k_scale), _ptr(v_scale)
            a.scale_seq_stride = seq_len * per_row
            a.scale_row_stride = per_row
            a.q8_block = int(bool(q8_block))
        _set_gate(a, out_gate, out_gate_row_stride, out_gate_head_stride)
        self._keep = self._keep + (out_gate,)
        L = ffi.lib()
        nbytes = L.gr_decode_workspace_size(ctypes.byref(a))
        self.ws = _workspace(nbytes, q.device)
        a.workspace = _aligned(self.ws)
        self.args = a

    def __call__(self, stream=None) -> None:
        ffi.check(ffi.lib().gr_decode_attention(ctypes.byref(self.args), _stream(stream)))


def turbo_sign_table(n_layers: int, n_kv_heads: int, head_size: int):
    """gr_turbo_sign_table: host uint8 [4][n_layers][n_kv_heads][ceil(head_size/8)]."""
    import numpy as np
    t = np.zeros((4, n_layers, n_kv_heads, (head_size + 7) // 8), np.uint8)
    ffi.check(ffi.lib().gr_turbo_sign_table(n_layers, n_kv_heads, head_size, t.ctypes.data))
    return t


class TurboDecodeCall:
    """gr_decode_attention over a Turbo cache (device tensors):
    codes k_base/v_base uint8 [n_seq][seq_len][Hkv*d/4], signs k_sign/v_sign uint8
    [n_seq][seq_len][Hkv*d/8], sigma k_scale/v_scale and gamma k_rnorm/v_rnorm f32
    [n_seq][seq_len][Hkv], signs_dev uint8 [4][n_layers][Hkv][d/8] (the whole table)
    and the layer index; q / out as DecodeCall."""

    def __init__(self, q, k_base, v_base, k_sign, v_sign, k_scale, v_scale, k_rnorm, v_rnorm,
                 signs_dev, layer, kv_start, kv_end, out, *, max_kv_len, score_scale=None,
                 split_keys=0):
        n_seq, n_heads, d = q.shape
        _, seq_len, nb = k_base.shape
        n_kv = nb * 4 // d
        _, n_layers, n_kv2, sb = signs_dev.shape
        assert n_kv2 == n_kv and sb == d // 8 and k_sign.shape == (n_seq, seq_len, n_kv * d // 8)
        for t in (k_scale, v_scale, k_rnorm, v_rnorm):
            assert t.shape == (n_seq, seq_len, n_kv) and t.dtype == torch.float32 and t.is_contiguous()
        self._keep = (q, k_base, v_base, k_sign, v_sign, k_scale, v_scale, k_rnorm, v_rnorm, signs_dev,
                      kv_start, kv_end, out)
        a = ffi.DecodeArgs()
        a.n_seq, a.n_heads, a.n_kv_heads, a.head_dim = n_seq, n_heads, n_kv, d
        a.kv_dtype = ffi.DTYPE_TURBO
        a.split_keys = split_keys
        a.max_kv_len = int(max_kv_len)
        a.score_scale = 1.0 / math.sqrt(d) if score_scale is None else float(score_scale)
        a.q, a.k_cache, a.v_cache = _ptr(q), _ptr(k_base), _ptr(v_base)
        a.seq_stride = seq_len * n_kv * d
        a.row_stride = n_kv * d
        a.kv_start, a.kv_end, a.out = _ptr(kv_start), _ptr(kv_end), _ptr(out)
        a.k_scale, a.v_scale, a.k_rnorm, a.v_rnorm = _ptr(k_scale), _ptr(v_scale), _ptr(k_rnorm), _ptr(v_rnorm)
        a.k_sign, a.v_sign = _ptr(k_sign), _ptr(v_sign)
        a.scale_seq_stride = seq_len * n_kv
        a.scale_row_stride = n_kv
        a.turbo_signs = signs_dev.data_ptr() + layer * n_kv * sb
        a.turbo_slot_stride = n_layers * n_kv * sb
        L = ffi.lib()
        self.ws = _workspace(L.gr_decode_workspace_size(ctypes.byref(a)), q.device)
        a.workspace = _aligned(self.ws)
        self.args = a

    def __call__(self, stream=None) -> None:
        ffi.check(ffi.lib().gr_decode_attention(ctypes.byref(self.args), _stream(stream)))


def decode_attention(q, k_cache, v_cache, kv_start, kv_end, *, max_kv_len=None, score_scale=None,
                     split_keys=0, out=None, k_scale=None, v_scale=None, q8_block=False):
    if out is None:
        out = torch.empty_like(q)
    if max_kv_len is None:
        max_kv_len = int((kv_end - kv_start).max().item())
    DecodeCall(q, k_cache, v_cache, kv_start, kv_end, out, max_kv_len=max_kv_len,
               score_scale=score_scale, split_keys=split_keys, k_scale=k_scale, v_scale=v_scale,
               q8_block=q8_block)()
    return out


def rope_freqs(theta: float, rope_dim: int) -> list[float]:
    """Host-computed RoPE frequency table (gr_rope_freqs, inference.rs:1590-1609)."""
    buf = (ctypes.c_float * (rope_dim // 2))()
    ffi.check(ffi.lib().gr_rope_freqs(float(theta), int(rope_dim), ctypes.cast(buf, ctypes.c_void_p)))
    return list(buf)


class PrefillCall:
    """A prepared gr_prefill_attention call.

    q [m][Hq][d], k/v [m][Hkv][d] (f16 or bf16, pre-norm, pre-RoPE);
    k_cache/v_cache [rows][Hkv][d] of the same dtype (rows >= base_pos + m);
    out [m][Hq][d] f32.  rope_freqs is a device f32 tensor [rope_dim/2].
    """

    def __init__(self, q, k, v, k_cache, v_cache, out, *, base_pos=0, window=0,
                 rope_mode=ffi.ROPE_NONE, rope_dim=0, rope_scale=1.0, rope_freqs=None,
                 q_norm=None, k_norm=None, norm_eps=1e-6, is_gemma3=False, bidirectional=False,
                 out_gate=None, out_gate_row_stride=0, out_gate_head_stride=0, q_bias=None, k_bias=None,
                 v_bias=None):
        m, n_heads, d = q.shape
        _, n_kv, d2 = k.shape
        assert d2 == d and v.shape == k.shape and out.shape == (m, n_heads, d)
        assert q.dtype == k.dtype == v.dtype == k_cache.dtype == v_cache.dtype
        assert out.dtype == torch.float32
        for t in (q, k, v, k_cache, v_cache, out):
            assert t.is_contiguous()
        self._keep = (q, k, v, k_cache, v_cache, out, rope_freqs, q_norm, k_norm, out_gate, q_bias, k_bias, v_bias)
        a = ffi.PrefillArgs()
        a.n_tokens, a.base_pos, a.n_heads, a.n_kv_heads, a.head_dim = m, base_pos, n_heads, n_kv, d
        a.dtype = _DT[q.dtype]
        a.window = int(window)
        a.rope_mode, a.rope_dim, a.rope_scale = int(rope_mode), int(rope_dim), float(rope_scale)
        a.rope_freqs = _ptr(rope_freqs)
        a.q_norm, a.k_norm = _ptr(q_norm), _ptr(k_norm)
        a.q_bias, a.k_bias, a.v_bias = _ptr(q_bias), _ptr(k_bias), _ptr(v_bias)
        a.norm_eps = float(norm_eps)
        a.is_gemma3 = int(bool(is_gemma3))
        a.bidirectional = int(bool(bidirectional))
        a.q, a.k, a.v = _ptr(q), _ptr(k), _ptr(v)
        a.k_cache, a.v_cache = _ptr(k_cache), _ptr(v_cache)
        a.cache_row_stride = n_kv * d
        a.out = _ptr(out)
        _set_gate(a, out_gate, out_gate_row_stride, out_gate_head_stride)
        nbytes = ffi.lib().gr_prefill_workspace_size(ctypes.byref(a))
        self.ws = _workspace(nbytes, q.device)
        a.workspace = _aligned(self.ws)
        self.args = a

    def __call__(self, stream=None) -> None:
        ffi.check(ffi.lib().gr_prefill_attention(ctypes.byref(self.args), _stream(stream)))


def prefill_attention(q, k, v, k_cache, v_cache, **kw):
    out = torch.empty(q.shape, dtype=torch.float32, device=q.device)
    PrefillCall(q, k, v, k_cache, v_cache, out, **kw)()
    return out


def encoder_self_attention(q, k, v, *, n_seq, tokens, heads, head_dim, out=None, stream=None):
    """gr_encoder_self_attention (encoder_self_attention, multimodal/mod.rs:145-256):
    f32 device rows [n_seq*tokens][heads*head_dim]; returns out of the same shape."""
    for t in (q, k, v):
        assert t.dtype == torch.float32 and t.is_contiguous()
    if out is None:
        out = torch.empty_like(q)
    ffi.check(ffi.lib().gr_encoder_self_attention(_ptr(out), _ptr(q), _ptr(k), _ptr(v), int(n_seq),
                                                  int(tokens), int(heads), int(head_dim),
                                                  _stream(stream)))
    return out


class DeltaNetCall:
    """A prepared gr_deltanet_attention call.

    q/k/v [T][H][d] (f32/f16/bf16); gate/beta [T][H] f32; state [H][d][d] f32
    (updated in place); out [T][H][d] f32.
    """

    def __init__(self, q, k, v, gate, beta, state, out, *, l2norm=True, eps=1e-6,
                 algo=ffi.DELTANET_AUTO):
        T, H, d = q.shape
        assert k.shape == v.shape == q.shape and q.dtype == k.dtype == v.dtype
        assert gate.shape == beta.shape == (T, H) and gate.dtype == beta.dtype == torch.float32
        assert state.shape == (H, d, d) and state.dtype == torch.float32
        assert out.shape == (T, H, d) and out.dtype == torch.float32
        for t in (q, k, v, gate, beta, state, out):
            assert t.is_contiguous()
        self._keep = (q, k, v, gate, beta, state, out)
        a = ffi.DeltaNetArgs()
        a.n_tokens, a.n_heads, a.head_dim = T, H, d
        a.in_dtype = _DT[q.dtype]
        a.l2norm = int(bool(l2norm))
        a.algo = int(algo)
        a.eps = float(eps)
        a.q, a.k, a.v = _ptr(q), _ptr(k), _ptr(v)
        a.gate, a.beta, a.state, a.out = _ptr(gate), _ptr(beta), _ptr(state), _ptr(out)
        nbytes = ffi.lib().gr_deltanet_workspace_size(ctypes.byref(a))
        self.ws = _workspace(nbytes, q.device) if nbytes else None
        a.workspace = _aligned(self.ws) if nbytes else None
        self.args = a

    def __call__(self, stream=None) -> None:
        ffi.check(ffi.lib().gr_deltanet_attention(ctypes.byref(self.args), _stream(stream)))


# ---------------------------------------------------------------- paged cache, packed batches

def _need(ok, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(device, *tensors) -> None:
    for t in tensors:
        _need(t.is_cuda, "libgr_attn device entry points take device tensors")
        _need(t.device == device, f"every tensor of a call lives on one device: {t.device} and {device}")


def _ints(t, shape, name) -> None:
    _need(t.dtype == torch.int32 and tuple(t.shape) == shape and t.is_contiguous(),
          f"{name} is a contiguous int32 tensor of shape {shape}")


class _DeviceCall:
    """A prepared call on tensors of one device; enqueued on `stream` (a stream of that
    device) or on the device's current one."""

    device: torch.device

    def _enqueue(self, stream, fn, *args) -> None:
        index = self.device.index
        if stream is None:
            raw = torch._C._cuda_getCurrentRawStream(index)
        else:
            _need(stream.device == self.device, f"the call's tensors live on {self.device}, the stream on {stream.device}")
            raw = stream.cuda_stream
        if torch._C._cuda_getDevice() == index:
            rc = fn(*args, raw)
        else:
            with torch.cuda.device(index):
                rc = fn(*args, raw)
        if rc:
            ffi.check(rc)


class PagedCache:
    """The K and V pages of one layer (gr_paged_cache).

    k_pages / v_pages [n_pages][page_size][Hkv][d] (f16, bf16, or int8 Q8 codes), the same
    strides, dims contiguous: a [n_pages][Hkv][page_size][d] buffer goes in as its
    transpose(1, 2).  Q8: f32 k_scale / v_scale [n_pages][page_size][Hkv].
    """

    def __init__(self, k_pages, v_pages, k_scale=None, v_scale=None):
        _need(k_pages.dim() == 4 and k_pages.shape == v_pages.shape and k_pages.dtype == v_pages.dtype
              and k_pages.stride() == v_pages.stride() and k_pages.stride(3) == 1,
              "k_pages and v_pages: [n_pages][page_size][n_kv_heads][head_dim] of one type and one set of strides, "
              "dims contiguous")
        _need(k_pages.dtype in (torch.float16, torch.bfloat16, torch.int8), "pages are f16, bf16 or int8")
        self.device = k_pages.device
        _on(self.device, k_pages, v_pages)
        self._keep = (k_pages, v_pages, k_scale, v_scale)
        c = ffi.PagedCacheDesc()
        c.n_pages, c.page_size, c.n_kv_heads, c.head_dim = k_pages.shape
        c.kv_dtype = _DT[k_pages.dtype]
        c.k_pages, c.v_pages = _ptr(k_pages), _ptr(v_pages)
        c.page_stride, c.row_stride, c.head_stride = _strides(k_pages, 3)
        if k_pages.dtype == torch.int8:
            _need(k_scale is not None and v_scale is not None, "Q8 pages need k_scale and v_scale")
            _need(all(t.dtype == torch.float32 and t.shape == k_pages.shape[:3] for t in (k_scale, v_scale))
                  and k_scale.stride() == v_scale.stride(),
                  "k_scale and v_scale: f32 [n_pages][page_size][n_kv_heads] of one set of strides")
            _on(self.device, k_scale, v_scale)
            c.k_scale, c.v_scale = _ptr(k_scale), _ptr(v_scale)
            c.scale_page_stride, c.scale_row_stride, c.scale_head_stride = _strides(k_scale, 3, 1)
        else:
            _need(k_scale is None and v_scale is None, "k_scale and v_scale belong to Q8 pages")
        self.desc = c


def _strides(t, n: int, least: int | None = None):
    """The first n strides; that of a dimension of size 1 is never used and becomes a valid one."""
    least = t.shape[-1] if least is None else least
    return [least if t.shape[i] == 1 else s for i, s in enumerate(t.stride()[:n])]


class PagedBatch:
    """The rows of a step (gr_paged_batch): row_start int32 [n_seq + 1], kv_len int32
    [n_seq], page_table int32 [n_seq][pages] (rows may be strided), all on the device and
    read when a call's kernels run.  n_rows: rows of the step's row arrays; max_rows,
    max_len: upper bounds of a sequence's rows and length."""

    def __init__(self, row_start, kv_len, page_table, *, n_rows, max_rows, max_len):
        _need(page_table.dim() == 2 and page_table.dtype == torch.int32
              and (page_table.shape[1] == 1 or page_table.stride(1) == 1),
              "page_table is an int32 tensor [n_seq][pages], pages contiguous")
        n_seq, pages = page_table.shape
        _ints(row_start, (n_seq + 1,), "row_start")
        _ints(kv_len, (n_seq,), "kv_len")
        self.device = row_start.device
        _on(self.device, row_start, kv_len, page_table)
        self._keep = (row_start, kv_len, page_table)
        b = ffi.PagedBatchDesc()
        b.n_seq, b.n_rows, b.max_rows, b.max_len = n_seq, int(n_rows), int(max_rows), int(max_len)
        b.row_start, b.kv_len, b.page_table = _ptr(row_start), _ptr(kv_len), _ptr(page_table)
        b.table_stride, b.table_pages = max(page_table.stride(0), pages) if n_seq == 1 else page_table.stride(0), pages
        self.desc = b


class _PagedKvCall(_DeviceCall):
    _fn = ""

    def __init__(self, cache: PagedCache, batch: PagedBatch, k, v):
        _need(k.dim() == 3 and k.shape == v.shape and k.dtype == v.dtype and k.stride() == v.stride()
              and k.stride(2) == 1, "k and v: rows [n_rows][n_kv_heads][head_dim] of one type and one set of strides")
        _need(k.dtype in (torch.float32, torch.float16, torch.bfloat16), "rows are f32, f16 or bf16")
        c, b = cache.desc, batch.desc
        _need(tuple(k.shape) == (b.n_rows, c.n_kv_heads, c.head_dim),
              f"rows of shape {tuple(k.shape)}: the batch and the cache say {(b.n_rows, c.n_kv_heads, c.head_dim)}")
        self.device = cache.device
        _on(self.device, k, v, batch._keep[0])
        r = ffi.PagedRows()
        r.dtype, r.k, r.v = _DT[k.dtype], _ptr(k), _ptr(v)
        r.row_stride, r.head_stride = _strides(k, 2)
        self._keep = (cache, batch, k, v)
        self.args = r
        self._call = (getattr(ffi.lib(), self._fn), ctypes.byref(c), ctypes.byref(b), ctypes.byref(r))

    def __call__(self, stream=None) -> None:
        self._enqueue(stream, *self._call)


class PagedWriteCall(_PagedKvCall):
    """A prepared gr_paged_kv_write: the batch's K / V rows [n_rows][Hkv][d] (f32, f16 or
    bf16) go to their pages, rounded or quantised to the cache's type."""

    _fn = "gr_paged_kv_write"


class PagedReadCall(_PagedKvCall):
    """A prepared gr_paged_kv_read: the batch's positions read out of their pages into k and
    v [n_rows][Hkv][d] (f32, f16 or bf16)."""

    _fn = "gr_paged_kv_read"


def _check_qo(q, out) -> None:
    _need(q.dim() == 3 and out.shape == q.shape and out.dtype == q.dtype and q.stride(2) == 1 and out.stride(2) == 1,
          "q and out: rows [n_rows][n_heads][head_dim] of one type, dims contiguous")
    _need(q.dtype in (torch.float16, torch.bfloat16), "q and out are f16 or bf16")


class PagedAttentionCall(_DeviceCall):
    """A prepared gr_paged_attention (args + workspace): q / out [n_rows][Hq][d] (f16 or bf16,
    the pages' type unless they are Q8); the pages hold the batch's rows already.  Calls that
    may overlap (other streams, graphs replayed side by side) are prepared separately: each
    has its own workspace."""

    def __init__(self, cache: PagedCache, batch: PagedBatch, q, out, *, window=0, score_scale=None):
        _check_qo(q, out)
        c, b = cache.desc, batch.desc
        _need(q.shape[0] == b.n_rows and q.shape[2] == c.head_dim,
              f"q of shape {tuple(q.shape)}: the batch has {b.n_rows} rows, the cache head_dim {c.head_dim}")
        self.device = cache.device
        _on(self.device, q, out, batch._keep[0])
        a = ffi.PagedAttentionArgs()
        a.n_heads, a.dtype, a.window = q.shape[1], _DT[q.dtype], int(window)
        a.score_scale = 1.0 / math.sqrt(c.head_dim) if score_scale is None else float(score_scale)
        a.q, a.out = _ptr(q), _ptr(out)
        a.q_row_stride, a.q_head_stride = _strides(q, 2)
        a.out_row_stride, a.out_head_stride = _strides(out, 2)
        args = (ctypes.byref(c), ctypes.byref(b), ctypes.byref(a))
        self.ws = _workspace(ffi.lib().gr_paged_attention_workspace_size(*args), self.device)
        a.workspace = _aligned(self.ws)
        self._keep = (cache, batch, q, out)
        self.args = a
        self._call = (ffi.lib().gr_paged_attention, *args)

    def __call__(self, stream=None) -> None:
        self._enqueue(stream, *self._call)


def paged_attention(cache: PagedCache, batch: PagedBatch, q, *, out=None, window=0, score_scale=None):
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)  # rows of no sequence stay zero
    PagedAttentionCall(cache, batch, q, out, window=window, score_scale=score_scale)()
    return out


class PackedAttentionCall(_DeviceCall):
    """A prepared gr_packed_attention (args + workspace): causal attention inside each of the
    prompts that lie one after another in q [n_rows][Hq][d], k and v [n_rows][Hkv][d] (f16
    or bf16); seq_start int32 [n_seq + 1]; out as q; max_rows an upper bound of the longest
    prompt.  Calls that may overlap are prepared separately, as PagedAttentionCall."""

    def __init__(self, q, k, v, seq_start, out, *, max_rows, window=0, score_scale=None):
        _check_qo(q, out)
        n_rows, n_heads, d = q.shape
        _need(k.dim() == 3 and k.shape == v.shape and k.stride() == v.stride() and k.stride(2) == 1
              and k.dtype == v.dtype == q.dtype and k.shape[0] == n_rows and k.shape[2] == d,
              "k and v: rows [n_rows][n_kv_heads][head_dim] of q's type and of one set of strides")
        _need(seq_start.dim() == 1 and seq_start.numel() >= 1, "seq_start has n_seq + 1 entries")
        _ints(seq_start, (seq_start.numel(),), "seq_start")
        self.device = q.device
        _on(self.device, q, k, v, seq_start, out)
        a = ffi.PackedArgs()
        a.n_seq, a.n_rows, a.max_rows = seq_start.numel() - 1, n_rows, int(max_rows)
        a.n_heads, a.n_kv_heads, a.head_dim, a.dtype = n_heads, k.shape[1], d, _DT[q.dtype]
        a.window = int(window)
        a.score_scale = 1.0 / math.sqrt(d) if score_scale is None else float(score_scale)
        a.seq_start, a.q, a.k, a.v, a.out = _ptr(seq_start), _ptr(q), _ptr(k), _ptr(v), _ptr(out)
        a.q_row_stride, a.q_head_stride = _strides(q, 2)
        a.kv_row_stride, a.kv_head_stride = _strides(k, 2)
        a.out_row_stride, a.out_head_stride = _strides(out, 2)
        self.ws = _workspace(ffi.lib().gr_packed_attention_workspace_size(ctypes.byref(a)), self.device)
        a.workspace = _aligned(self.ws)
        self._keep = (q, k, v, seq_start, out)
        self.args = a

    def __call__(self, stream=None) -> None:
        self._enqueue(stream, ffi.lib().gr_packed_attention, ctypes.byref(self.args))


def packed_attention(q, k, v, seq_start, *, max_rows, out=None, window=0, score_scale=None):
    if out is None:
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)  # rows of no prompt stay zero
    PackedAttentionCall(q, k, v, seq_start, out, max_rows=max_rows, window=window, score_scale=score_scale)()
    return out
