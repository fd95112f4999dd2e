"""Refusals of the paged-cache and packed-batch calls (every check runs before a launch: no
GPU), the Python wrappers' checks, and the Rust and ctypes copies of gr_paged.h.  CPU only."""
from __future__ import annotations

import ctypes
import pathlib
import re

import pytest
import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]


def cache(ffi, **kw):
    c = ffi.PagedCacheDesc()
    c.n_pages, c.page_size, c.n_kv_heads, c.head_dim, c.kv_dtype = 8, 16, 4, 128, ffi.DTYPE_F16
    c.k_pages, c.v_pages = 1 << 20, 1 << 21
    c.page_stride, c.row_stride, c.head_stride = 16 * 512, 512, 128
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def batch(ffi, **kw):
    b = ffi.PagedBatchDesc()
    b.n_seq, b.n_rows, b.max_rows, b.max_len = 2, 10, 5, 64
    b.row_start, b.kv_len, b.page_table, b.table_stride, b.table_pages = 4096, 8192, 12288, 4, 4
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def rows(ffi, **kw):
    r = ffi.PagedRows()
    r.dtype, r.k, r.v, r.row_stride, r.head_stride = ffi.DTYPE_F32, 1 << 22, 1 << 23, 512, 128
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def attn(ffi, **kw):
    a = ffi.PagedAttentionArgs()
    a.n_heads, a.dtype, a.window, a.score_scale = 8, ffi.DTYPE_F16, 0, 0.1
    a.q, a.q_row_stride, a.q_head_stride = 1 << 24, 1024, 128
    a.out, a.out_row_stride, a.out_head_stride = 1 << 25, 1024, 128
    a.workspace = 1 << 26
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def packed(ffi, **kw):
    a = ffi.PackedArgs()
    a.n_seq, a.n_rows, a.max_rows, a.n_heads, a.n_kv_heads, a.head_dim = 2, 10, 6, 8, 4, 128
    a.dtype, a.score_scale, a.seq_start = ffi.DTYPE_BF16, 0.1, 4096
    a.q, a.q_row_stride, a.q_head_stride = 1 << 20, 1024, 128
    a.k, a.v, a.kv_row_stride, a.kv_head_stride = 1 << 21, 1 << 22, 512, 128
    a.out, a.out_row_stride, a.out_head_stride, a.workspace = 1 << 23, 1024, 128, 1 << 24
    for k, v in kw.items():
        setattr(a, k, v)
    return a


CACHE_BAD = [
    (dict(head_dim=96), "head_dim 96 unsupported"), (dict(n_kv_heads=0), "n_kv_heads 0"), (dict(n_pages=0), "n_pages 0"),
    (dict(page_size=8), "power of two"), (dict(page_size=48), "power of two"), (dict(page_size=-16), "power of two"),
    (dict(kv_dtype=0), "kv_dtype 0 unsupported"), (dict(kv_dtype=4), "kv_dtype 4 unsupported"),
    (dict(k_pages=None), "null k_pages"), (dict(v_pages=(1 << 21) + 8), "16-byte aligned"),
    (dict(row_stride=508), "multiples of 16 bytes"), (dict(head_stride=64), "at least head_dim"),
    (dict(page_stride=-512), "at least head_dim"), (dict(row_stride=(1 << 22) + 8), "above 2^22"),
    (dict(k_scale=4096), "belong to Q8 pages"), (dict(kv_dtype=3), "need k_scale and v_scale"),
    (dict(kv_dtype=3, k_scale=4096, v_scale=8192), "scale strides must be positive"),
    (dict(kv_dtype=3, row_stride=520), "multiples of 16 bytes"),
]
BATCH_BAD = [
    (dict(n_seq=-1), "negative sizes"), (dict(n_rows=-2), "negative sizes"), (dict(max_rows=0), "must be positive"),
    (dict(max_len=0), "must be positive"), (dict(row_start=None), "null row_start"), (dict(kv_len=None), "null row_start, kv_len"),
    (dict(page_table=None), "page_table"), (dict(table_pages=0), "table_pages 0"), (dict(table_pages=5), "table_pages 5"),
    (dict(table_pages=1 << 27, table_stride=1 << 27), "above 2^30"), (dict(n_seq=1 << 30), "n_seq"),
]
ROWS_BAD = [
    (dict(dtype=3), "rows dtype 3"), (dict(k=None), "null k or v"), (dict(v=(1 << 23) + 4), "16-byte aligned"),
    (dict(row_stride=514), "multiples of 16 bytes"), (dict(head_stride=64), "at least head_dim"),
    (dict(dtype=1, head_stride=132), "multiples of 16 bytes"),
]
ATTN_BAD = [
    (dict(n_heads=6), "multiple of n_kv_heads"), (dict(n_heads=0), "multiple of n_kv_heads"), (dict(dtype=0), "dtype 0 unsupported"),
    (dict(dtype=2), "over pages of dtype"), (dict(window=-1), "negative window"), (dict(score_scale=0.0), "finite and positive"),
    (dict(score_scale=float("nan")), "finite and positive"), (dict(score_scale=float("inf")), "finite and positive"),
    (dict(q=None), "null q or out"), (dict(out=(1 << 25) + 2), "16-byte aligned"), (dict(q_row_stride=1028), "multiples of 8"),
    (dict(out_head_stride=120), "at least head_dim"),
]
PACKED_BAD = [
    (dict(head_dim=80), "head_dim 80"), (dict(n_seq=-1), "negative sizes"), (dict(max_rows=0), "max_rows 0"),
    (dict(n_heads=10), "multiple of n_kv_heads"), (dict(n_kv_heads=0), "multiple of n_kv_heads"), (dict(dtype=3), "dtype 3"),
    (dict(window=-4), "negative window"), (dict(score_scale=-1.0), "finite and positive"), (dict(seq_start=None), "null seq_start"),
    (dict(k=None), "null k or v"), (dict(v=(1 << 22) + 8), "16-byte aligned"), (dict(kv_row_stride=130), "multiples of 8"),
    (dict(kv_row_stride=1 << 23), "above 2^22"), (dict(q_head_stride=100), "multiples of 8"), (dict(n_rows=1 << 28), "above 2^30"),
]


def refused(ffi, rc, msg):
    assert rc == ffi.GR_ERR_ARG
    assert msg in ffi.lib().gr_last_error().decode(), ffi.lib().gr_last_error()


@pytest.mark.parametrize("kw,msg", CACHE_BAD)
def test_bad_caches(pkg, kw, msg):
    from gguf_runner_amd import ffi
    L, c, b = ffi.lib(), cache(ffi, **kw), batch(ffi)
    for call in (L.gr_paged_kv_write, L.gr_paged_kv_read):
        refused(ffi, call(c, b, rows(ffi), None), msg)
    refused(ffi, L.gr_paged_attention(c, b, attn(ffi), None), msg)
    assert L.gr_paged_attention_workspace_size(c, b, attn(ffi)) == 0


@pytest.mark.parametrize("kw,msg", BATCH_BAD)
def test_bad_batches(pkg, kw, msg):
    from gguf_runner_amd import ffi
    L, c, b = ffi.lib(), cache(ffi), batch(ffi, **kw)
    for call in (L.gr_paged_kv_write, L.gr_paged_kv_read):
        refused(ffi, call(c, b, rows(ffi), None), msg)
    refused(ffi, L.gr_paged_attention(c, b, attn(ffi), None), msg)


@pytest.mark.parametrize("kw,msg", ROWS_BAD)
def test_bad_rows(pkg, kw, msg):
    from gguf_runner_amd import ffi
    for call in (ffi.lib().gr_paged_kv_write, ffi.lib().gr_paged_kv_read):
        refused(ffi, call(cache(ffi), batch(ffi), rows(ffi, **kw), None), msg)


@pytest.mark.parametrize("kw,msg", ATTN_BAD)
def test_bad_attention_args(pkg, kw, msg):
    from gguf_runner_amd import ffi
    L = ffi.lib()
    refused(ffi, L.gr_paged_attention(cache(ffi), batch(ffi), attn(ffi, **kw), None), msg)
    assert L.gr_paged_attention_workspace_size(cache(ffi), batch(ffi), attn(ffi, **kw)) == 0


@pytest.mark.parametrize("kw,msg", PACKED_BAD)
def test_bad_packed_args(pkg, kw, msg):
    from gguf_runner_amd import ffi
    L = ffi.lib()
    refused(ffi, L.gr_packed_attention(packed(ffi, **kw), None), msg)
    assert L.gr_packed_attention_workspace_size(packed(ffi, **kw)) == 0


def test_more_work_than_can_be_numbered(pkg):
    from gguf_runner_amd import ffi
    L = ffi.lib()
    big = dict(n_seq=1 << 20, n_rows=1 << 20, table_pages=1 << 20, table_stride=1 << 20)
    refused(ffi, L.gr_paged_attention(cache(ffi), batch(ffi, **big), attn(ffi), None), "divide the batch")
    assert L.gr_paged_attention_workspace_size(cache(ffi), batch(ffi, **big), attn(ffi)) == 0
    # the limit is the one of the kernel that the call takes: the places of a stream where blocks
    # are cut (max_rows 1), the threads of a launch where they are not
    rows_of = dict(n_seq=1 << 12, n_rows=1 << 21, table_pages=1 << 14, table_stride=1 << 14, max_len=4096)
    refused(ffi, L.gr_paged_attention(cache(ffi), batch(ffi, max_rows=1, **rows_of), attn(ffi), None), "divide the batch")
    assert L.gr_paged_attention_workspace_size(cache(ffi), batch(ffi, max_rows=4096, **rows_of), attn(ffi)) == 256
    for fn in (L.gr_paged_kv_write, L.gr_paged_kv_read):
        refused(ffi, fn(cache(ffi), batch(ffi, n_rows=(1 << 26) + 1), rows(ffi), None), "divide the batch")


def test_null_and_workspace(pkg):
    from gguf_runner_amd import ffi
    L, c, b, a = ffi.lib(), cache(ffi), batch(ffi), attn(ffi)
    refused(ffi, L.gr_paged_kv_write(None, b, rows(ffi), None), "null cache")
    refused(ffi, L.gr_paged_kv_write(c, None, rows(ffi), None), "null batch")
    refused(ffi, L.gr_paged_kv_read(c, b, None, None), "null rows")
    refused(ffi, L.gr_paged_attention(c, b, None, None), "null args")
    refused(ffi, L.gr_packed_attention(None, None), "null args")
    for ws, msg in ((None, "null workspace"), ((1 << 26) + 16, "256-byte aligned")):
        refused(ffi, L.gr_paged_attention(c, b, attn(ffi, workspace=ws), None), msg)
        refused(ffi, L.gr_packed_attention(packed(ffi, workspace=ws), None), msg)
    assert L.gr_paged_attention_workspace_size(c, b, a) > 0 and L.gr_packed_attention_workspace_size(packed(ffi)) > 0
    # nothing to do: no pointer is looked at
    none = batch(ffi, n_rows=0, row_start=None, kv_len=None, page_table=None)
    assert L.gr_paged_kv_write(c, none, None, None) == ffi.GR_OK
    assert L.gr_paged_attention(c, none, None, None) == ffi.GR_OK
    assert L.gr_packed_attention(packed(ffi, n_seq=0, q=None, workspace=None), None) == ffi.GR_OK


def test_wrappers_refuse(pkg):
    """The Python side's own checks: shapes, types, strides, devices."""
    from gguf_runner_amd import ops
    k = torch.zeros((4, 16, 2, 64), dtype=torch.float16)
    for bad, msg in (((k, k[:2]), "one type and one set of strides"), ((k, k.float()), "one type"),
                     ((k.float(), k.float()), "f16, bf16 or int8"), ((k[..., ::2], k[..., ::2]), "dims contiguous"),
                     ((k, k), "device tensors")):
        with pytest.raises(ValueError, match=msg):
            ops.PagedCache(*bad)
    one = torch.zeros(3, dtype=torch.int32)
    for bad, msg in (((one, one[:2], torch.zeros((2, 4))), "page_table"), ((one, one, torch.zeros((2, 4), dtype=torch.int32)), "kv_len"),
                     ((one[:2], one[:2], torch.zeros((2, 4), dtype=torch.int32)), "row_start"),
                     ((one.long(), one[:2], torch.zeros((2, 4), dtype=torch.int32)), "row_start"),
                     ((one, one[:2], torch.zeros((2, 8), dtype=torch.int32)[:, ::2]), "pages contiguous")):
        with pytest.raises(ValueError, match=msg):
            ops.PagedBatch(*bad, n_rows=2, max_rows=1, max_len=4)
    q = torch.zeros((5, 4, 64), dtype=torch.float16)
    for bad, msg in (((q, q.bfloat16(), q, one, q), "of q's type"), ((q, q[:4], q[:4], one, q), "n_rows"),
                     ((q, q, q, one, q[:4]), "q and out"), ((q.float(), q, q, one, q.float()), "f16 or bf16"),
                     ((q, q, q, one.long(), q), "seq_start"), ((q, q, q, one, q), "device tensors")):
        with pytest.raises(ValueError, match=msg):
            ops.PackedAttentionCall(*bad, max_rows=5)


# ---------------------------------------------------------------- copies of the header

C2R = {"int32_t": "i32", "int64_t": "i64", "float": "f32", "int": "i32", "size_t": "usize", "void*": "*mut c_void",
       "const void*": "*const c_void", "float*": "*mut f32", "const int32_t*": "*const i32",
       "const gr_paged_cache*": "*const GrPagedCache", "const gr_paged_batch*": "*const GrPagedBatch",
       "const gr_paged_rows*": "*const GrPagedRows", "const gr_paged_attention_args*": "*const GrPagedAttentionArgs",
       "const gr_packed_args*": "*const GrPackedArgs"}
STRUCTS = {"gr_paged_cache": ("GrPagedCache", "PagedCacheDesc"), "gr_paged_batch": ("GrPagedBatch", "PagedBatchDesc"),
           "gr_paged_rows": ("GrPagedRows", "PagedRows"), "gr_paged_attention_args": ("GrPagedAttentionArgs", "PagedAttentionArgs"),
           "gr_packed_args": ("GrPackedArgs", "PackedArgs")}


def _header():
    return re.sub(r"/\*.*?\*/", " ", (ROOT / "include" / "gr_paged.h").read_text(), flags=re.S)


def _split(decl):
    m = re.match(r"(.*?[\s\*])(\w+)$", re.sub(r"\s+", " ", decl.strip()))
    return m.group(2), re.sub(r"\s*\*", "*", m.group(1).strip())


def _fields(name):
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), _header(), re.S).group(1)
    return [_split(d) for d in body.split(";") if d.strip()]


def test_ctypes_copies_match_the_header(pkg):
    from gguf_runner_amd import ffi
    kinds = {"int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64, "float": ctypes.c_float}
    for name, (_, cls) in STRUCTS.items():
        want = [(n, kinds.get(t, ctypes.c_void_p)) for n, t in _fields(name)]
        assert list(getattr(ffi, cls)._fields_) == want, name


def test_rust_copies_match_the_header():
    path = ROOT / "rust" / "paged.rs"
    if not path.exists():
        pytest.skip(f"{path} is not in this checkout")
    text = path.read_text()
    for name, (rust, _) in STRUCTS.items():
        body = re.search(r"#\[repr\(C\)\]\s*pub struct %s \{(.*?)\n\}" % rust, text, re.S).group(1)
        got = re.findall(r"pub (\w+): ([^,]+),", body)
        assert got == [(n, C2R[t]) for n, t in _fields(name)], name
    want = {}
    for m in re.finditer(r"^(int|size_t) (gr_\w+)\(([^)]*)\);", _header(), re.M | re.S):
        want[m.group(2)] = ([C2R[_split(p)[1]] for p in m.group(3).split(",")], C2R[m.group(1)])
    got = {m.group(1): ([p.split(":", 1)[1].strip() for p in m.group(2).split(",")], m.group(3))
           for m in re.finditer(r"pub fn (gr_\w+)\((.*?)\) -> (\w+);", text)}
    assert len(want) == 6 and got == want
