"""The paged KV cache and the attention over packed batches, as cases that can be timed and
compared: `listed()` names twelve, `draw()` gives others of the same ranges.

Five kinds of case:

  write    the new K / V rows of a batch go to their pages (f16 or bf16 pages)
  requant  the same into Q8 pages, and the rows read back: one after the other, as a prompt's
           rows are stored and later handed on
  read     rows of a batch read out of the pages (Q8 rows dequantised)
  paged    attention of each sequence's new tokens over its pages
  packed   attention over whole prompts of different lengths, one after another

Where `own` is false, `run()` computes them with elementary torch operations in 32 bits;
where it is true, through the library's entry points.  `exact()` evaluates the same inputs
in 64 bits.
"""
from __future__ import annotations

import importlib.util
import math
import pathlib
import sys

import numpy as np
import torch

own = False

ROOT = pathlib.Path(__file__).resolve().parent.parent
_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1}


def _ops():
    name = "gguf_runner_amd"
    if name not in sys.modules:
        d = ROOT / "gguf-runner_amd"
        spec = importlib.util.spec_from_file_location(name, d / "__init__.py", submodule_search_locations=[str(d)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from gguf_runner_amd import ops
    return ops


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # One decode step of a batch of 48: a row of each sequence is stored.
        {"name": "write_bf16_step_48", "kind": "write", "rows_dtype": "bf16", "kv": "bf16", "n_seq": 48, "min_rows": 1,
         "max_rows": 1, "min_past": 0, "max_past": 1001, "kv_heads": 8, "head_dim": 128, "page": 16},
        # Chunks of seven prompts of a small model, whose projections come in f32.
        {"name": "write_f32_f16_7_chunks", "kind": "write", "rows_dtype": "f32", "kv": "f16", "n_seq": 7, "min_rows": 33,
         "max_rows": 511, "min_past": 0, "max_past": 1001, "kv_heads": 2, "head_dim": 64, "page": 32},
        # Four prompts stored in Q8 as they are computed, and read back.
        {"name": "requant_q8_4_prompts", "kind": "requant", "rows_dtype": "f16", "kv": "q8", "n_seq": 4, "min_rows": 700,
         "max_rows": 4001, "min_past": 0, "max_past": 0, "kv_heads": 8, "head_dim": 128, "page": 64},
        # Three long conversations moved out of a Q8 cache.
        {"name": "read_q8_bf16_3x32k", "kind": "read", "rows_dtype": "bf16", "kv": "q8", "n_seq": 3, "min_rows": 20011,
         "max_rows": 32768, "min_past": 0, "max_past": 0, "kv_heads": 4, "head_dim": 128, "page": 128},
        # The last rows of twenty short sequences, in f32.
        {"name": "read_f16_f32_20_short", "kind": "read", "rows_dtype": "f32", "kv": "f16", "n_seq": 20, "min_rows": 1,
         "max_rows": 300, "min_past": 0, "max_past": 700, "kv_heads": 4, "head_dim": 256, "page": 16},
        # The smallest decode: one sequence with 1024 keys.
        {"name": "paged_bf16_token_1024", "kind": "paged", "dtype": "bf16", "kv": "bf16", "n_seq": 1, "min_rows": 1,
         "max_rows": 1, "min_past": 1023, "max_past": 1023, "heads": 16, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page": 16},
        # Batched decoding: sixteen sequences of ragged lengths up to 32k.
        {"name": "paged_f16_tokens_16_32k", "kind": "paged", "dtype": "f16", "kv": "f16", "n_seq": 16, "min_rows": 1,
         "max_rows": 1, "min_past": 1023, "max_past": 32767, "heads": 32, "kv_heads": 4, "head_dim": 128, "window": 0,
         "page": 64},
        # Batched decoding over Q8 pages, drafted tokens of some sequences checked in the same step.
        {"name": "paged_q8_tokens_24_12k", "kind": "paged", "dtype": "f16", "kv": "q8", "n_seq": 24, "min_rows": 1,
         "max_rows": 5, "min_past": 300, "max_past": 12001, "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0,
         "page": 16},
        # A long question in the middle of a conversation.
        {"name": "paged_f16_chunk_501_after_7690", "kind": "paged", "dtype": "f16", "kv": "f16", "n_seq": 1,
         "min_rows": 501, "max_rows": 501, "min_past": 7690, "max_past": 7690, "heads": 32, "kv_heads": 8,
         "head_dim": 128, "window": 0, "page": 32},
        # A mixed step of a sliding-window layer: chunks and single tokens, head_dim 256.
        {"name": "paged_bf16_d256_window_mixed", "kind": "paged", "dtype": "bf16", "kv": "bf16", "n_seq": 9,
         "min_rows": 1, "max_rows": 700, "min_past": 0, "max_past": 6000, "heads": 8, "kv_heads": 4, "head_dim": 256,
         "window": 1024, "page": 64},
        # Forty short prompts of a small model in one launch.
        {"name": "packed_bf16_d64_40_short", "kind": "packed", "dtype": "bf16", "n_seq": 40, "min_rows": 9,
         "max_rows": 777, "heads": 14, "kv_heads": 2, "head_dim": 64, "window": 0},
        # Three long prompts, the longest of 8192 tokens: the largest case.
        {"name": "packed_f16_3_long", "kind": "packed", "dtype": "f16", "n_seq": 3, "min_rows": 1001, "max_rows": 8192,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "window": 0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# (query heads, KV heads, head_dim) of the attention layers.
_HEADS = [(16, 8, 128), (32, 8, 128), (32, 4, 128), (14, 2, 64), (8, 4, 256)]


def draw(rng):
    kind = rng.choice(["write", "requant", "read", "paged", "paged", "paged", "packed", "packed"])
    h, g, d = rng.choice(_HEADS)
    page = rng.choice([16, 32, 64, 128, 256])
    if kind in ("write", "requant", "read"):
        n_seq = _log_int(rng, 1, 64)
        top = 1 if kind == "write" and rng.random() < 0.3 else _log_int(rng, 1, 32768 if kind == "read" else 8192)
        # At most the bytes that the largest listed read of 4 heads of 128 moves.
        top = max(1, min(top, int((70000 if kind == "read" else 26000) * 512 / (g * d) / n_seq)))
        past = 0 if kind == "requant" or rng.random() < 0.4 else _log_int(rng, 1, 8192)
        past = min(past, int(1.6e8 / (g * d) / n_seq))
        return {"kind": kind, "rows_dtype": rng.choice(["f32", "f16", "bf16"]),
                "kv": "q8" if kind == "requant" else rng.choice(["f16", "bf16"] + ["q8"] * (kind == "read")),
                "n_seq": n_seq, "min_rows": rng.randint(max(1, top // 16), top), "max_rows": top, "min_past": 0,
                "max_past": past, "kv_heads": g, "head_dim": d, "page": page}
    c = {"kind": kind, "dtype": rng.choice(["f16", "bf16"])}
    if kind == "paged":
        form = rng.choice(["tokens", "chunk", "mixed"])
        n_seq = _log_int(rng, 1, 4) if form == "chunk" else _log_int(rng, 1, 48)
        rows = 1 if form == "tokens" else _log_int(rng, 2, 2048 if form == "chunk" else 512)
        past = _log_int(rng, 16, 32768)
        past = max(1, min(past, int(275000 * 512 / (g * d) / n_seq)))
        c["kv"] = rng.choice([c["dtype"], c["dtype"], "q8"])
        c |= {"n_seq": n_seq, "min_rows": rows if form != "mixed" else 1, "max_rows": rows,
              "min_past": rng.randint(0, past), "max_past": past, "page": page}
    else:
        n_seq = _log_int(rng, 1, 64)
        top = _log_int(rng, 1, 8192)
        c |= {"n_seq": n_seq, "min_rows": rng.randint(max(1, top // 16), top), "max_rows": top}
    c |= {"heads": h, "kv_heads": g, "head_dim": d, "window": 1024 if d == 256 and rng.random() < 0.6 else 0}
    # No more than the largest listed case, nor more scores than the plain form holds at once.
    while work(c)["flops"] > 6.9e11 or n_seq * h * c["max_rows"] * (c["max_rows"] + c.get("max_past", 0)) > 4.4e9:
        c["max_rows"] = max(1, int(c["max_rows"] * 0.7))
        c["min_rows"] = min(c["min_rows"], c["max_rows"])
    return c


# ---------------------------------------------------------------- sizes

def _sizes(case):
    """(rows, cached rows before them) of each sequence, the largest of each among them."""
    n = case["n_seq"]
    rng = np.random.default_rng(7 + n + case["max_rows"] + case.get("max_past", 0))
    rows = rng.integers(case["min_rows"], case["max_rows"] + 1, n)
    rows[int(rng.integers(0, n))] = case["max_rows"]
    past = rng.integers(case.get("min_past", 0), case.get("max_past", 0) + 1, n)
    past[int(rng.integers(0, n))] = case.get("max_past", 0)
    return rows.astype(np.int64), past.astype(np.int64)


def _visible(case):
    """Keys that some row of each sequence sees, and (row, key) pairs of all of them."""
    keys, pairs = 0, 0
    w = case["window"]
    for n, b in zip(*_sizes(case)):
        seen = np.arange(b + 1, b + n + 1)
        if w:
            seen = np.minimum(seen, w)
        keys += int(min(b + n, w + n - 1) if w else b + n)
        pairs += int(seen.sum())
    return keys, pairs


def work(case):
    g, d = case["kv_heads"], case["head_dim"]
    rows = int(_sizes(case)[0].sum())
    kind = case["kind"]
    if kind == "packed":
        _, pairs = _visible(case)
        return {"bytes": 2 * rows * d * 2 * (case["heads"] + g), "flops": 4 * case["heads"] * d * pairs}
    cached = g * (d * _SIZE[case["kv"]] + (4 if case["kv"] == "q8" else 0))
    if kind == "paged":
        keys, pairs = _visible(case)
        return {"bytes": 2 * keys * cached + 2 * rows * case["heads"] * d * 2, "flops": 4 * case["heads"] * d * pairs}
    plain = g * d * _SIZE[case["rows_dtype"]]
    per_row = plain + cached if kind != "requant" else 2 * (plain + cached)
    return {"bytes": 2 * rows * per_row, "flops": 0}


# ---------------------------------------------------------------- inputs

def _rows(gen, n, heads, d, dtype):
    """K or V rows as projections give them: unit variance, a few channels of every head larger."""
    x = torch.randn((n, heads, d), generator=gen, device="cuda", dtype=torch.float32)
    x[..., 3::37] *= 4.0
    return x.to(dtype)


def _quantise(x):
    """Q8 of f32 rows [..][d]: codes (int8) and one scale per row."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = torch.where(amax == 0, torch.ones_like(amax), amax / 127.0)
    y = x * torch.where(amax == 0, torch.zeros_like(amax), 127.0 / amax)
    whole = torch.trunc(y)
    y = whole + torch.where((y - whole).abs() >= 0.5, torch.sign(y), torch.zeros_like(y))  # halves away from zero
    return y.clamp(-127, 127).to(torch.int8), scale.squeeze(-1)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    host = np.random.default_rng(int(seed))
    g, d, n_seq = case["kv_heads"], case["head_dim"], case["n_seq"]
    rows, past = _sizes(case)
    total, lens = int(rows.sum()), rows + past
    start = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    s = {"case": case, "n_rows": total, "max_rows": int(rows.max()), "max_len": int(lens.max()),
         "row_start": torch.from_numpy(start).cuda()}
    if "heads" in case:
        dt = _DT[case["dtype"]]
        s["q"] = torch.randn((total, case["heads"], d), generator=gen, device="cuda", dtype=torch.float32).to(dt)
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "packed":
        s["k"], s["v"] = (_rows(gen, total, g, d, dt) for _ in "kv")
        return s

    # The pool: every sequence's pages at random places, some pages free; table entries past a
    # sequence's last page name none.
    page = case["page"]
    per_seq = -(-lens // page)
    n_pages = int(per_seq.sum()) + 3 + int(per_seq.sum()) // 8
    order = host.permutation(n_pages)
    table = np.full((n_seq, int(per_seq.max())), -1, np.int32)
    at = 0
    for i, n in enumerate(per_seq):
        table[i, :n] = order[at:at + n]
        at += n
    s["page_table"] = torch.from_numpy(table).cuda()
    s["kv_len"] = torch.from_numpy(lens.astype(np.int32)).cuda()
    for x in "kv":
        pool = _rows(gen, n_pages * page, g, d, torch.float32 if case["kv"] == "q8" else _DT[case["kv"]])
        pool = pool.view(n_pages, page, g, d)
        if case["kv"] == "q8":
            s[x + "_pages"], s[x + "_scale"] = _quantise(pool)
        else:
            s[x + "_pages"] = pool
        if case["kind"] in ("write", "requant"):
            s[x] = _rows(gen, total, g, d, _DT[case["rows_dtype"]])
        if case["kind"] in ("read", "requant"):
            s[x + "_out"] = torch.empty((total, g, d), dtype=_DT[case["rows_dtype"]], device="cuda")
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        ops = _ops()
        if case["kind"] == "packed":
            s["call"] = ops.PackedAttentionCall(s["q"], s["k"], s["v"], s["row_start"], s["out"],
                                                max_rows=s["max_rows"], window=case["window"])
            return s
        cache = ops.PagedCache(s["k_pages"], s["v_pages"], s.get("k_scale"), s.get("v_scale"))
        batch = ops.PagedBatch(s["row_start"], s["kv_len"], s["page_table"], n_rows=s["n_rows"],
                               max_rows=s["max_rows"], max_len=s["max_len"])
        if case["kind"] in ("write", "requant"):
            s["write"] = ops.PagedWriteCall(cache, batch, s["k"], s["v"])
        if case["kind"] in ("read", "requant"):
            s["read"] = ops.PagedReadCall(cache, batch, s["k_out"], s["v_out"])
        if case["kind"] == "paged":
            s["call"] = ops.PagedAttentionCall(cache, batch, s["q"], s["out"], window=case["window"])
    return s


# ---------------------------------------------------------------- one pass

def _places(s):
    """The (page, row in it) of every row of the batch."""
    start, page = s["row_start"].long(), s["case"]["page"]
    row = torch.arange(s["n_rows"], device="cuda")
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = s["kv_len"].long()[seq] - start[seq + 1] + row
    return s["page_table"].long()[seq, pos // page], pos % page


def _plain_write(s):
    at = _places(s)
    for x in "kv":
        if s["case"]["kv"] == "q8":
            s[x + "_pages"][at], s[x + "_scale"][at] = _quantise(s[x].float())
        else:
            s[x + "_pages"][at] = s[x].float().to(s[x + "_pages"].dtype)


def _plain_read(s):
    at = _places(s)
    for x in "kv":
        r = s[x + "_pages"][at].float()
        if s["case"]["kv"] == "q8":
            r = r * s[x + "_scale"][at].unsqueeze(-1)
        s[x + "_out"].copy_(r)


def _plain_attention(s):
    case = s["case"]
    h, g, d, w = case["heads"], case["kv_heads"], case["head_dim"], case["window"]
    start = s["row_start"].long()
    rows = start[1:] - start[:-1]
    n_seq, m = rows.numel(), s["max_rows"]
    i = torch.arange(m, device="cuda")
    there = i < rows.unsqueeze(1)                                              # [n_seq][m]
    at = (start[:-1].unsqueeze(1) + i).clamp(max=s["n_rows"] - 1)
    q = s["q"][at].float().view(n_seq, m, g, h // g, d).permute(0, 2, 1, 3, 4).reshape(n_seq, g, m * (h // g), d)
    if case["kind"] == "packed":
        k, v = (s[x][at].float().permute(0, 2, 1, 3).contiguous() for x in "kv")  # [n_seq][g][m][d]
        lens = rows
    else:
        table = s["page_table"].long().clamp(min=0)
        k, v = (s[x][table].float() for x in ("k_pages", "v_pages"))           # [n_seq][pages][page][g][d]
        if case["kv"] == "q8":
            k, v = k * s["k_scale"][table].unsqueeze(-1), v * s["v_scale"][table].unsqueeze(-1)
        k, v = (x.flatten(1, 2).permute(0, 2, 1, 3).contiguous() for x in (k, v))
        lens = s["kv_len"].long()
    score = torch.matmul(q, k.transpose(2, 3).contiguous())
    score = score.mul_(1.0 / math.sqrt(d)).view(n_seq, g, m, h // g, -1)
    key = torch.arange(score.shape[-1], device="cuda")
    pos = (lens - rows).unsqueeze(1) + i                                       # [n_seq][m]
    hidden = key > pos.unsqueeze(-1)
    if w:
        hidden |= key <= pos.unsqueeze(-1) - w
    score.masked_fill_(hidden.view(n_seq, 1, m, 1, -1), float("-inf"))
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(n_seq, g, m * (h // g), -1), v).view(n_seq, g, m, h // g, d)
    o = (o / total).permute(0, 2, 1, 3, 4).reshape(n_seq, m, h, d)
    s["out"][at[there]] = o[there].to(s["out"].dtype)


def run(state):
    s, kind = state, state["case"]["kind"]
    if kind in ("paged", "packed"):
        if own:
            s["call"]()
        else:
            _plain_attention(s)
        return s["out"]
    if kind in ("write", "requant"):
        if own:
            s["write"]()
        else:
            _plain_write(s)
        if kind == "write":
            return s["k_pages"], s["v_pages"]
    if own:
        s["read"]()
    else:
        _plain_read(s)
    return s["k_out"], s["v_out"]


# ---------------------------------------------------------------- the same in 64 bits

def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    rows, past = _sizes(case)
    table = s["page_table"].cpu().numpy() if kind != "packed" else None

    def stored(x, i):
        """The cached rows of sequence i, in 64 bits."""
        at = torch.from_numpy(table[i][table[i] >= 0].astype(np.int64)).cuda()
        r = s[x + "_pages"][at].double()
        if case["kv"] == "q8":
            r = r * s[x + "_scale"][at].double().unsqueeze(-1)
        return r.flatten(0, 1)[:int(rows[i] + past[i])]

    if kind in ("write", "requant"):
        at = 0
        back = {"k": [], "v": []}
        for i, n in enumerate(rows):
            pos = np.arange(past[i], past[i] + n)
            pg = torch.from_numpy(table[i, pos // case["page"]].astype(np.int64)).cuda()
            ro = torch.from_numpy(pos % case["page"]).cuda()
            for x in "kv":
                r = s[x][at:at + int(n)].double()
                if kind == "write":
                    if i == 0:
                        back[x] = s[x + "_pages"].double()
                    back[x][pg, ro] = r
                else:
                    a = r.abs().amax(-1, keepdim=True)
                    step = torch.where(a == 0, 1.0, a / 127)
                    c = torch.floor((r / step).abs() + 0.5) * r.sign()
                    back[x].append(c * step)
            at += int(n)
        return tuple(back[x] if kind == "write" else torch.cat(back[x]) for x in "kv")
    if kind == "read":
        return tuple(torch.cat([stored(x, i)[int(past[i]):] for i in range(len(rows))]) for x in "kv")

    group, d, w = case["heads"] // case["kv_heads"], case["head_dim"], case["window"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, n in enumerate(rows):
        n, b = int(n), int(past[i]) if kind == "paged" else 0
        q = s["q"][at:at + n].double()
        k, v = (s[x][at:at + n].double() if kind == "packed" else stored(x, i) for x in "kv")
        pos = torch.arange(b, b + n, device="cuda").unsqueeze(1)
        key = torch.arange(b + n, device="cuda").unsqueeze(0)
        seen = (key <= pos) & (key > pos - w) if w else key <= pos
        for h in range(case["heads"]):
            t = (q[:, h] @ k[:, h // group].T) / math.sqrt(d)
            out[at:at + n, h] = torch.softmax(t.masked_fill(~seen, float("-inf")), -1) @ v[:, h // group]
        at += n
    return out
