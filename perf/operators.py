"""Cases, plain forms and entry points of the cached-decoding operators.

Three operators that one decoding step of a decoder block uses in a row:

* ``rope`` / ``append``: rotary positions on queries and keys (half or
  interleaved pairs, the whole head or its first part, any table), the inverse
  rotation for gradients, and the form that writes rotated keys and values
  into the pages of a paged key-value cache;
* ``attend``: attention of one new token per sequence over that cache;
* ``copy``: copies of pages (compaction), and of the first slots of pages
  (forks).

``run`` computes them with elementary torch operations in 32 bits, or, where
``own`` is true, with this package's kernels.  ``exact`` states each operator
in 64 bits, sequence by sequence.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _lib():
    root = str(Path.cwd() / "torch-helion_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from torch_helion.b200 import lib

    return lib


# ------------------------------------------------------------------- the cases
def listed():
    return [
        # the fp32 block of 8 heads of 64 at its own sequence length: one short sequence, pure latency
        {"name": "attend_f32_one", "op": "attend", "dtype": "f32", "batch": 1, "len_min": 128, "len_max": 128, "hq": 8,
         "hkv": 8, "d": 64, "page": 16, "softcap": 0.0, "window": 0},
        # one user's stream in the 32/8-head block after its full prompt of 4096: few rows, so split over the length
        {"name": "attend_stream", "op": "attend", "dtype": "bf16", "batch": 1, "len_min": 4097, "len_max": 4097, "hq": 32,
         "hkv": 8, "d": 128, "page": 16, "softcap": 0.0, "window": 0},
        # a served batch: ragged lengths from a new prompt to twice the block's sequence length
        {"name": "attend_batch", "op": "attend", "dtype": "bf16", "batch": 64, "len_min": 17, "len_max": 8191, "hq": 32,
         "hkv": 8, "d": 128, "page": 16, "softcap": 0.0, "window": 0},
        # long documents: the largest caches
        {"name": "attend_long", "op": "attend", "dtype": "bf16", "batch": 4, "len_min": 90001, "len_max": 131071, "hq": 32,
         "hkv": 8, "d": 128, "page": 64, "softcap": 0.0, "window": 0},
        # one shared key-value head, capped scores, a sliding window, a head and pages of odd sizes
        {"name": "attend_shared_capped", "op": "attend", "dtype": "f16", "batch": 24, "len_min": 1, "len_max": 20011,
         "hq": 20, "hkv": 1, "d": 80, "page": 24, "softcap": 30.0, "window": 4096},
        # a prompt batch of the 32/8-head block (8 x 4096 tokens), queries and keys inside one fused projection
        {"name": "rope_prompt", "op": "rope", "dtype": "bf16", "tokens": 32768, "hq": 32, "hkv": 8, "d": 128,
         "rotary": 128, "interleaved": False, "inverse": False, "positions": 4096, "theta": 500000.0},
        # the gradient of interleaved rotary positions on part of the head, an odd number of tokens, fp32
        {"name": "rope_gradient", "op": "rope", "dtype": "f32", "tokens": 4097, "hq": 8, "hkv": 8, "d": 64, "rotary": 48,
         "interleaved": True, "inverse": True, "positions": 8192, "theta": 10000.0},
        # one decoding step of 64 sequences: every new token goes to its own page
        {"name": "append_step", "op": "append", "dtype": "bf16", "batch": 64, "new": 1, "before": 1023, "hq": 32, "hkv": 8,
         "d": 128, "rotary": 128, "page": 16, "interleaved": False, "theta": 500000.0},
        # prompts that enter the cache, 8 x 2047 tokens, half of each head rotated
        {"name": "append_prompt", "op": "append", "dtype": "f16", "batch": 8, "new": 2047, "before": 0, "hq": 32, "hkv": 8,
         "d": 128, "rotary": 64, "page": 16, "interleaved": False, "theta": 500000.0},
        # one fork of a sequence of the fp32 block: its last, partly filled page, keys and values of 8 heads
        {"name": "fork_one", "op": "copy", "dtype": "f32", "pool": 64, "pairs": 1, "planes": 16, "page": 16, "width": 64,
         "partial": True},
        # 64 sequences forked at once in a 32-layer cache of 8 heads: their partly filled pages
        {"name": "fork_batch", "op": "copy", "dtype": "bf16", "pool": 256, "pairs": 64, "planes": 512, "page": 16,
         "width": 128, "partial": True},
        # compaction of a 32-layer cache: whole pages to the front of the pool
        {"name": "compact", "op": "copy", "dtype": "bf16", "pool": 1024, "pairs": 509, "planes": 512, "page": 16,
         "width": 128, "partial": False},
    ]


def _log(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "rope", "append", "copy"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8, 20])
    d = rng.choice([32, 64, 80, 96, 128, 128, 256])
    heads = {"hq": hkv * group, "hkv": hkv, "d": d}
    page = rng.choice([8, 16, 16, 24, 32, 64])
    if op == "attend":
        top = _log(rng, 1, 131071)
        room = 200_000_000 // (top * hkv * d)  # under half the elements of the longest listed case
        batch = max(1, min(_log(rng, 1, 256), room))
        return {"op": op, "dtype": dtype, "batch": batch, "len_min": rng.choice([top, max(1, top // 50)]), "len_max": top,
                **heads, "page": page, "softcap": rng.choice([0.0, 0.0, 30.0]), "window": rng.choice([0, 0, _log(rng, 16, 8192)])}
    rotary = rng.choice([d, d, d // 2])
    if op == "rope":
        tokens = _log(rng, 1, max(1, min(32768, (1 << 26) // (heads["hq"] * d))))
        return {"op": op, "dtype": dtype, "tokens": tokens, **heads, "rotary": rotary, "interleaved": rng.random() < 0.4,
                "inverse": rng.random() < 0.4, "positions": _log(rng, 16, 65536), "theta": rng.choice([10000.0, 500000.0])}
    if op == "append":
        new = rng.choice([1, 1, _log(rng, 1, 4096)])
        batch = max(1, min(_log(rng, 1, 256), (1 << 26) // (new * heads["hq"] * d)))
        return {"op": op, "dtype": dtype, "batch": batch, "new": new, "before": _log(rng, 1, 1024) - 1, **heads,
                "rotary": rotary, "page": page, "interleaved": rng.random() < 0.4, "theta": rng.choice([10000.0, 500000.0])}
    planes = 2 * rng.choice([1, 4, 24, 32]) * hkv
    per_page = planes * page * d * (4 if dtype == "f32" else 2)
    pool = max(4, min(1024, (1 << 30) // per_page))
    return {"op": op, "dtype": dtype, "pool": pool, "pairs": _log(rng, 1, pool // 2 - 1), "planes": planes, "page": page,
            "width": d, "partial": rng.random() < 0.5}


# -------------------------------------------------------------------- the data
def _lengths(case):
    """Sequence lengths of a case, from the case alone: spread over the logarithm, the longest one among them."""
    r = random.Random(1000003 * case["batch"] + 8191 * case["len_max"] + case["len_min"])
    return [case["len_max"]] + [_log(r, case["len_min"], case["len_max"]) for _ in range(case["batch"] - 1)]


def _counts(case):
    """Filled slots of each copied page."""
    r = random.Random(7919 * case["pairs"] + case["page"])
    return [r.randint(1, case["page"]) if case["partial"] else case["page"] for _ in range(case["pairs"])]


def _tables(rows, rotary, theta, dev):
    """cos / sin of position x frequency, [rows, rotary / 2], as a model keeps them."""
    freq = theta ** (-torch.arange(0, rotary, 2, device=dev, dtype=torch.float64) / rotary)
    angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _pages(gen, dtype, lens, page, hkv, d, dev):
    """A pool of filled pages and a table that hands them to the sequences in random order (-1: no page)."""
    need = [-(-n // page) for n in lens]
    pool = sum(need) + max(2, sum(need) // 16)
    kv = torch.randn(2, pool, hkv, page, d, generator=gen, device=dev, dtype=dtype)
    order = torch.randperm(pool, generator=gen, device=dev)[: sum(need)].to(torch.int32)
    width = max(need)
    have = torch.arange(width, device=dev)[None] < torch.tensor(need, device=dev)[:, None]
    table = torch.full((len(lens), width), -1, device=dev, dtype=torch.int32)
    table[have] = order
    return kv[0], kv[1], table


def _fused(gen, dtype, tokens, hq, hkv, d, dev):
    """q, k and v as views of one projection's output [tokens, (hq + 2 hkv) d]."""
    qkv = torch.randn(tokens, hq + 2 * hkv, d, generator=gen, device=dev, dtype=dtype)
    return qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, op = _DTYPES[case["dtype"]], case["op"]
    if op == "attend":
        lens = _lengths(case)
        k, v, table = _pages(gen, dtype, lens, case["page"], case["hkv"], case["d"], dev)
        q = (1.5 * torch.randn(case["batch"], case["hq"], case["d"], generator=gen, device=dev)).to(dtype)
        return {"op": op, "q": q, "k_pages": k, "v_pages": v, "table": table, "longest": max(lens),
                "lens": torch.tensor(lens, device=dev, dtype=torch.int32), "scale": case["d"] ** -0.5,
                "softcap": case["softcap"], "window": case["window"]}
    if op == "rope":
        q, k, _ = _fused(gen, dtype, case["tokens"], case["hq"], case["hkv"], case["d"], dev)
        cos, sin = _tables(case["positions"], case["rotary"], case["theta"], dev)
        at = torch.randint(case["positions"], (1,), generator=gen, device=dev)
        pos = ((torch.arange(case["tokens"], device=dev) + at) % case["positions"]).to(torch.int32)
        return {"op": op, "q": q, "k": k, "positions": pos, "cos": cos, "sin": sin, "interleaved": case["interleaved"],
                "inverse": case["inverse"]}
    if op == "append":
        b, n = case["batch"], case["new"]
        before = torch.randint(case["before"] // 2, case["before"] + 1, (b,), generator=gen, device=dev)
        q, k, v = _fused(gen, dtype, b * n, case["hq"], case["hkv"], case["d"], dev)
        kp, vp, table = _pages(gen, dtype, [case["before"] + n] * b, case["page"], case["hkv"], case["d"], dev)
        cos, sin = _tables(case["before"] + n, case["rotary"], case["theta"], dev)
        return {"op": op, "q": q, "k": k, "v": v, "k_pages": kp, "v_pages": vp, "table": table, "cos": cos, "sin": sin,
                "seqs": torch.arange(b, device=dev, dtype=torch.int32).repeat_interleave(n),
                "positions": (before[:, None] + torch.arange(n, device=dev)).reshape(-1).to(torch.int32),
                "interleaved": case["interleaved"]}
    pages = torch.randn(case["pool"], case["planes"], case["page"], case["width"], generator=gen, device=dev, dtype=dtype)
    order = torch.randperm(case["pool"], generator=gen, device=dev).to(torch.int32)
    counts = torch.tensor(_counts(case), device=dev, dtype=torch.int32) if case["partial"] else None
    return {"op": op, "pages": pages, "src": order[: case["pairs"]].clone(),
            "dst": order[case["pairs"] : 2 * case["pairs"]].clone(), "counts": counts}


# ------------------------------------------------------- the package's kernels
def _run_own(s):
    lib = _lib()
    if s["op"] == "attend":
        if "workspace" not in s:  # once per cache, as a serving loop keeps it
            s["workspace"] = lib.paged_attention_workspace(s["q"], s["k_pages"])
        return lib.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], scale=s["scale"],
                                   softcap=s["softcap"], window=s["window"], workspace=s["workspace"])
    if s["op"] == "rope":
        return lib.rope(s["q"], s["k"], s["positions"], s["cos"], s["sin"], interleaved=s["interleaved"],
                        inverse=s["inverse"])
    if s["op"] == "append":
        q = lib.rope_append(s["q"], s["k"], s["v"], s["positions"], s["cos"], s["sin"], s["k_pages"], s["v_pages"],
                            s["table"], seqs=s["seqs"], interleaved=s["interleaved"])
        return q, s["k_pages"], s["v_pages"]
    lib.page_copy(s["pages"], s["src"], s["dst"], s["counts"])
    return s["pages"]


# ------------------------------------------------------------- the plain forms
def _rotate(x, positions, cos, sin, interleaved, inverse):
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    s = -s if inverse else s
    half = c.shape[-1]
    x32 = x.float()
    if interleaved:
        a, b = x32[..., 0 : 2 * half : 2], x32[..., 1 : 2 * half : 2]
        turned = torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2)
    else:
        a, b = x32[..., :half], x32[..., half : 2 * half]
        turned = torch.cat((a * c - b * s, a * s + b * c), dim=-1)
    return torch.cat((turned, x32[..., 2 * half :]), dim=-1).to(x.dtype)


def _attend(s):
    q, page = s["q"], s["k_pages"].shape[2]
    b, hq, d = q.shape
    hkv = s["k_pages"].shape[1]
    j = torch.arange(s["longest"], device=q.device)
    ids = s["table"][:, j // page].long().clamp(min=0)
    k = s["k_pages"][ids, :, j % page].float()  # [batch, longest, hkv, d]
    v = s["v_pages"][ids, :, j % page].float()
    lens = s["lens"].long()[:, None]
    seen = j < lens
    if s["window"]:
        seen = seen & (j >= lens - s["window"])
    scores = torch.matmul(q.float().view(b, hkv, hq // hkv, d), k.permute(0, 2, 3, 1)) * s["scale"]
    if s["softcap"]:
        scores = s["softcap"] * torch.tanh(scores / s["softcap"])
    scores = scores.masked_fill(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - top)
    out = torch.matmul(p, v.transpose(1, 2)) / p.sum(-1, keepdim=True)
    return out.reshape(b, hq, d).to(q.dtype)


def _run_plain(s):
    if s["op"] == "attend":
        return _attend(s)
    how = (s["positions"], s["cos"], s["sin"], s["interleaved"], s.get("inverse", False)) if "positions" in s else ()
    if s["op"] == "rope":
        return _rotate(s["q"], *how), _rotate(s["k"], *how)
    if s["op"] == "append":
        page = s["k_pages"].shape[2]
        pos = s["positions"].long()
        ids = s["table"][s["seqs"].long(), pos // page].long()
        s["k_pages"][ids, :, pos % page] = _rotate(s["k"], *how)
        s["v_pages"][ids, :, pos % page] = s["v"]
        return _rotate(s["q"], *how), s["k_pages"], s["v_pages"]
    pages, src, dst = s["pages"], s["src"].long(), s["dst"].long()
    if s["counts"] is None:
        pages[dst] = pages[src]
    else:
        filled = torch.arange(pages.shape[2], device=pages.device) < s["counts"][:, None]
        pages[dst] = torch.where(filled[:, None, :, None], pages[src], pages[dst])
    return pages


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------ in 64 bits
def _turned_64(x, cos, sin, interleaved, inverse):
    """Each pair as a complex number times exp(+-i angle)."""
    x = x.double()
    half = cos.shape[-1]
    part = x[..., : 2 * half]
    pair = part.unflatten(-1, (half, 2)) if interleaved else part.unflatten(-1, (2, half)).transpose(-1, -2)
    turn = torch.complex(cos.double(), sin.double())
    z = torch.view_as_complex(pair.contiguous()) * (turn.conj() if inverse else turn)[:, None]
    z = torch.view_as_real(z)
    x[..., : 2 * half] = (z if interleaved else z.transpose(-1, -2)).flatten(-2)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "attend":
        page, group = case["page"], case["hq"] // case["hkv"]
        out = torch.empty(s["q"].shape, device=s["q"].device, dtype=torch.float64)
        for b, n in enumerate(_lengths(case)):
            first = max(0, n - case["window"]) if case["window"] else 0
            rows = s["table"][b, : -(-n // page)].long()
            for h in range(case["hkv"]):
                k = s["k_pages"][rows, h].reshape(-1, case["d"])[first:n].double()
                v = s["v_pages"][rows, h].reshape(-1, case["d"])[first:n].double()
                x = (s["q"][b, h * group : (h + 1) * group].double() @ k.t()) * s["scale"]
                if case["softcap"]:
                    x = (x / case["softcap"]).tanh() * case["softcap"]
                out[b, h * group : (h + 1) * group] = torch.softmax(x, dim=-1) @ v
        return out
    if s["op"] == "rope":
        at = s["positions"].long()
        how = (s["cos"][at], s["sin"][at], case["interleaved"], case["inverse"])
        return _turned_64(s["q"], *how), _turned_64(s["k"], *how)
    if s["op"] == "append":
        at, seq = s["positions"].long(), s["seqs"].long()
        how = (s["cos"][at], s["sin"][at], case["interleaved"], False)
        pages = []
        for held, new in ((s["k_pages"], _turned_64(s["k"], *how)), (s["v_pages"], s["v"].double())):
            flat = held.double().transpose(1, 2).flatten(0, 1)  # a row for each slot of the pool
            flat[s["table"][seq, at // case["page"]].long() * case["page"] + at % case["page"]] = new
            pages.append(flat.unflatten(0, (-1, case["page"])).transpose(1, 2))
        return _turned_64(s["q"], *how), pages[0], pages[1]
    after = s["pages"].clone()
    for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), _counts(case)):
        after[b, :, :n] = s["pages"][a, :, :n]
    return after


# ---------------------------------------------------------------------- the work
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    op = case["op"]
    if op == "attend":
        lens = [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]
        row = case["d"] * size
        pages = sum(-(-n // case["page"]) for n in lens)
        return {"bytes": 2 * sum(lens) * case["hkv"] * row + 2 * case["batch"] * case["hq"] * row + 4 * pages + 4 * case["batch"],
                "flops": 4 * sum(lens) * case["hq"] * case["d"]}
    if op == "copy":
        return {"bytes": 2 * sum(_counts(case)) * case["planes"] * case["width"] * size + 8 * case["pairs"], "flops": 0}
    tokens = case["tokens"] if op == "rope" else case["batch"] * case["new"]
    rotated = case["hq"] + case["hkv"]
    moved = rotated + (case["hkv"] if op == "append" else 0)
    seen = min(tokens, case["positions"]) if op == "rope" else min(tokens, case["before"] + case["new"])
    return {"bytes": 2 * tokens * moved * case["d"] * size + 4 * seen * case["rotary"] + 4 * tokens * (1 if op == "rope" else 2),
            "flops": 3 * tokens * rotated * case["rotary"]}
