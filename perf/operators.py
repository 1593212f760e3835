"""Performance cases of a serving step that takes several new tokens of each
request: their latents and rotated keys go into a paged cache, their queries
attend to all that the cache holds before them, and the drafted ones among
them are accepted or replaced.

Kinds of cases and their ranges (draw):
  append    store_rope: latents and rotary keys into the paged bf16 cache of
            576-wide rows, the queries' rotation with them; 1..65536 tokens,
            0..64 query heads, with and without the latent's norm, both pair
            orders, fp32 and bf16 tables
  attend    mla_chunk_attention_paged: dense causal latent attention of a
            ragged chunk of new tokens over a paged cache, bf16 rows with
            rotary keys or the INT8 rows without; 1..64 requests of 1..2048
            new tokens each, 8..64 heads, contexts of 1..131072 tokens
  verify    verify_drafts: drafted tokens against the target's probabilities,
            1..64 requests of 0..7 drafts, 512..131072 tokens in the
            vocabulary, with the drafts' probabilities and without
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

LATENT = 512
ROPE = 64
WIDTH = LATENT + ROPE
ROW = 528            # an INT8 cache row: codes, fp32 scale, padding
EPS = 1e-6
SM_SCALE = WIDTH ** -0.5
ROPE_BASE = 10000.0


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # A decode step of eight requests, all on its own: latency of one launch.
        {"name": "append_b8", "kind": "append", "tokens": 8, "heads": 16, "norm": True, "interleaved": True,
         "block": 64, "table": "fp32", "max_pos": 131072, "slots64": True, "pages": 256},
        # A prefill chunk's tokens over the slots that the allocator gave them.
        {"name": "append_chunk_2048", "kind": "append", "tokens": 2048, "heads": 16, "norm": True,
         "interleaved": True, "block": 64, "table": "fp32", "max_pos": 131072, "slots64": True, "pages": 512},
        # A restored context: normed latents of 65536 tokens and no queries, an odd page size.
        {"name": "append_fill_65536", "kind": "append", "tokens": 65536, "heads": 0, "norm": False,
         "interleaved": False, "block": 48, "table": "bf16", "max_pos": 65536, "slots64": False, "pages": 1400},
        # One user's decode step at a short context: the smallest attention.
        {"name": "decode_b1_2k", "kind": "attend", "cache": "int8", "requests": 1, "new": 1, "heads": 16,
         "context": 2000, "block": 64, "ragged": False, "lse": False},
        # One user's decode step at the longest context: one row group over a long axis.
        {"name": "decode_b1_128k", "kind": "attend", "cache": "bf16", "requests": 1, "new": 1, "heads": 16,
         "context": 131072, "block": 64, "ragged": False, "lse": False},
        # Continuous batching: 64 requests of very different lengths.
        {"name": "decode_b64_ragged", "kind": "attend", "cache": "int8", "requests": 64, "new": 1, "heads": 16,
         "context": 16384, "block": 256, "ragged": True, "lse": False},
        # A speculative step: three drafts and the token before them for each of 24 requests.
        {"name": "verify_step_b24", "kind": "attend", "cache": "bf16", "requests": 24, "new": 4, "heads": 16,
         "context": 12000, "block": 64, "ragged": True, "lse": True},
        # Five prompts of odd lengths in one chunk, small pages, 20 heads.
        {"name": "prompts_b5", "kind": "attend", "cache": "int8", "requests": 5, "new": 301, "heads": 20,
         "context": 3001, "block": 16, "ragged": True, "lse": False},
        # The last 2048 tokens of a 16384-token prompt: the largest attention.
        {"name": "chunk_2048_16k", "kind": "attend", "cache": "bf16", "requests": 1, "new": 2048, "heads": 16,
         "context": 16384, "block": 64, "ragged": False, "lse": False},
        # A single user's drafts from a small draft model.
        {"name": "drafts_b1", "kind": "verify", "requests": 1, "drafts": 3, "vocab": 32000, "ragged": False,
         "draft_probs": True, "ids64": False},
        # Drafts by lookup (no probabilities) in a batch, an odd vocabulary.
        {"name": "drafts_b24_lookup", "kind": "verify", "requests": 24, "drafts": 5, "vocab": 50257, "ragged": True,
         "draft_probs": False, "ids64": True},
        # A full batch over a large vocabulary.
        {"name": "drafts_b64", "kind": "verify", "requests": 64, "drafts": 7, "vocab": 131072, "ragged": True,
         "draft_probs": True, "ids64": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "attend", "verify"))
    if kind == "append":
        tokens = _log_int(rng, 1, 65536)
        block = rng.choice((16, 48, 64, 256))
        return {"kind": kind, "tokens": tokens, "heads": rng.choice((0, 8, 16, 16, 20, 64)) if tokens <= 4096 else 0,
                "norm": rng.random() < 0.5, "interleaved": rng.random() < 0.5, "block": block,
                "table": rng.choice(("fp32", "bf16")), "max_pos": _log_int(rng, 1024, 262144),
                "slots64": rng.random() < 0.5, "pages": (tokens + rng.randint(0, tokens) + block) // block}
    if kind == "verify":
        return {"kind": kind, "requests": _log_int(rng, 1, 64), "drafts": rng.randint(1, 7),
                "vocab": _log_int(rng, 512, 131072), "ragged": rng.random() < 0.5,
                "draft_probs": rng.random() < 0.6, "ids64": rng.random() < 0.5}
    shape = rng.choice(("decode", "decode", "verify", "chunk"))
    case = {"kind": kind, "cache": rng.choice(("bf16", "int8")), "heads": rng.choice((16, 16, 16, 8, 20, 32, 64)),
            "block": rng.choice((16, 48, 64, 256)), "ragged": rng.random() < 0.6, "lse": rng.random() < 0.3}
    if shape == "chunk":
        case["requests"] = _log_int(rng, 1, 8)
        case["new"] = _log_int(rng, 9, 2048 // case["requests"])
        most = 2048 * 16384 * 16 // (case["requests"] * case["new"] * case["heads"])
        case["context"] = _log_int(rng, case["new"], max(case["new"], min(32768, most)))
    else:
        case["requests"] = _log_int(rng, 1, 64)
        case["new"] = 1 if shape == "decode" else rng.randint(2, 8)
        case["context"] = _log_int(rng, case["new"], min(131072, 1048576 // case["requests"]))
    return case


def _lengths(case):
    """Each request's new tokens and its length with them, from the case alone."""
    n, new, context = case["requests"], case["new"], case["context"]
    if not case["ragged"]:
        return [new] * n, [context] * n
    r = random.Random(n * 1000003 + new * 1009 + context)
    news = [new] + [max(1, new - r.randrange(0, new // 2 + 1)) for _ in range(n - 1)]
    return news, [context] + [max(k, int(context * r.random())) for k in news[1:]]


def _drafts(case):
    """Each request's number of drafts, from the case alone."""
    if not case["ragged"]:
        return [case["drafts"]] * case["requests"]
    r = random.Random(case["requests"] * 31 + case["drafts"])
    return [case["drafts"]] + [r.randint(0, case["drafts"]) for _ in range(case["requests"] - 1)]


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _bf16_rows(g, rows, width):
    out = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    for s in range(0, rows, 65536):
        out[s:s + 65536] = _normal(g, min(65536, rows - s), width)
    return out


def _int8_rows(g, rows):
    """Rows as the INT8 writer leaves unit-normal latents."""
    out = torch.zeros(rows, ROW, dtype=torch.int8, device="cuda")
    for s in range(0, rows, 131072):
        e = min(rows, s + 131072)
        out[s:e, :LATENT] = (_normal(g, e - s, LATENT) * 40).round().clamp(-127, 127).to(torch.int8)
        scale = (torch.rand((e - s, 1), generator=g, device="cuda") * 0.012 + 0.020).contiguous()
        out[s:e, LATENT:LATENT + 4] = scale.view(torch.int8)
    return out


def _table(max_pos, dtype):
    """cos and sin of every position's angles (taken in 64 bits), side by side."""
    inv = ROPE_BASE ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device="cuda") / ROPE)
    angle = torch.arange(max_pos, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat((angle.cos(), angle.sin()), dim=1).to(dtype)


def prepare(case, seed):
    pkg = str(Path(__file__).resolve().parent.parent / "glm-5.3-kernels_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    g = _gen(seed)
    if case["kind"] == "append":
        return _prepare_append(case, g)
    return _prepare_attend(case, g) if case["kind"] == "attend" else _prepare_verify(case, g)


def _prepare_append(case, g):
    n, block, heads = case["tokens"], case["block"], case["heads"]
    capacity = case["pages"] * block
    slots = torch.randperm(capacity, generator=g, device="cuda")[:n]
    d = {"case": case, "x": _bf16_rows(g, n, LATENT), "k_pe": _bf16_rows(g, n, ROPE),
         "positions": torch.randint(0, case["max_pos"], (n,), generator=g, device="cuda"),
         "cos_sin": _table(case["max_pos"], torch.float32 if case["table"] == "fp32" else torch.bfloat16),
         "cache": torch.zeros(case["pages"], block, WIDTH, dtype=torch.bfloat16, device="cuda"),
         "slots": slots if case["slots64"] else slots.to(torch.int32),
         "norm": (1 + 0.1 * _normal(g, LATENT)).to(torch.bfloat16) if case["norm"] else None,
         "q": _normal(g, n, heads, WIDTH).to(torch.bfloat16) if heads else None}
    # the rotary part of the query projection's output, a strided view
    d["q_pe"] = _normal(g, n, heads, 3 * ROPE).to(torch.bfloat16)[:, :, 2 * ROPE:] if heads else None
    return d


def _prepare_attend(case, g):
    news, lens = _lengths(case)
    block, requests = case["block"], case["requests"]
    used = [(n + block - 1) // block for n in lens]
    pages = sum(used)
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((requests, max(used)), -1, dtype=torch.int32, device="cuda")
    for i, at in enumerate(torch.tensor([0] + used).cumsum(0)[:-1].tolist()):
        table[i, :used[i]] = order[at:at + used[i]]
    int8 = case["cache"] == "int8"
    rows = _int8_rows(g, pages * block) if int8 else _bf16_rows(g, pages * block, WIDTH)
    total = sum(news)
    # queries that make a token's logits spread by about two
    q = (_normal(g, total, case["heads"], LATENT if int8 else WIDTH) * 2).to(torch.bfloat16)
    return {"case": case, "q": q, "cache": rows.view(pages, block, -1), "table": table,
            "cu": torch.tensor([0] + news, device="cuda").cumsum(0).to(torch.int32),
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "most_new": max(news), "longest": max(lens)}


def _prepare_verify(case, g):
    counts, vocab = _drafts(case), case["vocab"]
    drafts, rows = sum(counts), sum(counts) + len(counts)
    cu = torch.tensor([0] + [n + 1 for n in counts], device="cuda").cumsum(0)
    request = torch.repeat_interleave(torch.arange(len(counts), device="cuda"),
                                      torch.tensor(counts, device="cuda"), output_size=drafts)
    logits = _normal(g, rows, vocab) * 3
    at = torch.arange(drafts, device="cuda") + request    # the target's row of each draft
    near = logits[at] + 0.7 * _normal(g, drafts, vocab)
    target = torch.softmax(logits, dim=1)
    draft = torch.softmax(near, dim=1)
    ids = ((near - torch.empty_like(near).exponential_(generator=g).log()).argmax(dim=1) if drafts
           else torch.zeros(0, dtype=torch.int64, device="cuda"))
    return {"case": case, "target": target, "draft": draft.contiguous() if case["draft_probs"] else None,
            "ids": ids if case["ids64"] else ids.to(torch.int32), "cu": cu.to(torch.int32),
            "accept_u": torch.rand(drafts, generator=g, device="cuda"),
            "sample_u": torch.rand(len(counts), generator=g, device="cuda", dtype=torch.float64)}


# ------------------------------------------------------------------ the calls

def run(s):
    kind = s["case"]["kind"]
    if kind == "append":
        return _own_append(s) if own else _plain_append(s)
    if kind == "attend":
        return _own_attend(s) if own else _plain_attend(s)
    return _own_verify(s) if own else _plain_verify(s)


def _own_append(s):
    from titan_kv import store_rope
    q = s["q"]
    store_rope(s["x"], s["k_pe"], s["positions"], s["cos_sin"], s["cache"], s["slots"], q_pe=s["q_pe"],
               q_out=None if q is None else q[:, :, LATENT:], norm_weight=s["norm"], eps=EPS,
               interleaved=s["case"]["interleaved"])
    return {"cache": s["cache"], "q": q}


def _own_attend(s):
    from titan_mla import mla_chunk_attention_paged
    return mla_chunk_attention_paged(s["q"], s["cache"], s["cu"], s["lens"], s["table"], SM_SCALE,
                                     return_lse=s["case"]["lse"])


def _own_verify(s):
    from titan_spec import verify_drafts
    return verify_drafts(s["target"], s["ids"], s["draft"], s["cu"], s["accept_u"], s["sample_u"],
                         s["case"]["drafts"])


# ------------------------------------------------------------------ the plain forms

def _rotated(p, cos, sin, interleaved):
    a, b = (p[..., 0::2], p[..., 1::2]) if interleaved else (p[..., :ROPE // 2], p[..., ROPE // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)


def _plain_append(s):
    x, block, interleaved = s["x"].float(), s["cache"].shape[1], s["case"]["interleaved"]
    if s["norm"] is not None:
        x = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * s["norm"].float()
    angle = s["cos_sin"][s["positions"]].float()
    cos, sin = angle[:, :ROPE // 2], angle[:, ROPE // 2:]
    row = torch.cat((x, _rotated(s["k_pe"].float(), cos, sin, interleaved)), dim=1).to(torch.bfloat16)
    slots = s["slots"].long()
    s["cache"][slots // block, slots % block] = row
    if s["q"] is not None:
        s["q"][:, :, LATENT:] = _rotated(s["q_pe"].float(), cos[:, None], sin[:, None], interleaved).to(torch.bfloat16)
    return {"cache": s["cache"], "q": s["q"]}


def _keys(rows, int8):
    """Cache rows in 32 bits, as the keys they stand for."""
    if not int8:
        return rows.float()
    return rows[..., :LATENT].float() * rows[..., LATENT:LATENT + 4].contiguous().view(torch.float32)


def _plain_attend(s):
    q, cache, table, cu, lens = s["q"], s["cache"], s["table"].long(), s["cu"].long(), s["lens"].long()
    (total, heads, _), block, most, longest = q.shape, cache.shape[1], s["most_new"], s["longest"]
    pos = torch.arange(longest, device=q.device)
    page = table[:, pos // block].clamp_min(0)
    keys = _keys(cache[page, pos % block], cache.dtype == torch.int8)             # [requests, longest, width]
    i = torch.arange(most, device=q.device)
    n = cu[1:] - cu[:-1]
    token = (cu[:-1, None] + i).clamp_max(total - 1)
    last = lens[:, None] - n[:, None] + i                                          # the last position each sees
    qs = q[token].float().flatten(1, 2) * SM_SCALE                                 # [requests, most * heads, width]
    score = torch.matmul(qs, keys.transpose(1, 2)).view(-1, most, heads, longest)
    score = score.masked_fill_((pos > last[..., None])[:, :, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    p = score.sub_(top).exp_()
    norm = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.flatten(1, 2), keys[..., :LATENT]).view(-1, most, heads, LATENT) / norm
    there = i < n[:, None]
    out = o[there].to(torch.bfloat16)
    return (out, (top + norm.log())[there][..., 0]) if s["case"]["lse"] else out


def _plain_verify(s):
    target, draft, cu, most = s["target"], s["draft"], s["cu"].long(), s["case"]["drafts"]
    requests = cu.numel() - 1
    first = cu[:-1]
    n = (cu[1:] - first - 1).clamp_max(most)
    i = torch.arange(most, device=target.device)
    there = i < n[:, None]
    at = (first - torch.arange(requests, device=target.device))[:, None] + i       # the drafts' places
    at = at.clamp_max(s["ids"].numel() - 1)
    ids = s["ids"].long()[at]
    pt = target[(first[:, None] + i).clamp_max(target.shape[0] - 1), ids]
    pd = draft[at, ids] if draft is not None else torch.ones_like(pt)
    taken = there & (s["accept_u"][at] * pd < pt)
    count = taken.long().cumprod(dim=1).sum(dim=1)
    base = target[first + count]
    place = at.gather(1, count.clamp_max(most - 1)[:, None])[:, 0]
    if draft is not None:
        rest = (base - draft[place]).clamp_min(0)
    else:
        rest = base.scatter(1, s["ids"].long()[place][:, None], 0.0)
    rest = torch.where((count < n)[:, None], rest, base)
    weight = (rest.double() * 2.0 ** 40).floor().long()
    whole = (base.double() * 2.0 ** 40).floor().long()
    weight = torch.where(weight.sum(dim=1, keepdim=True) > 0, weight, whole)
    run_sum = weight.cumsum(dim=1)
    all_of = run_sum[:, -1]
    drawn = torch.minimum((s["sample_u"] * all_of.double()).floor().long(), all_of - 1)
    token = (run_sum <= drawn[:, None]).sum(dim=1)
    j = torch.arange(most + 1, device=target.device)
    told = torch.cat((ids, ids[:, :1]), dim=1)
    tokens = torch.where(j < count[:, None], told, torch.where(j == count[:, None], token[:, None], -1))
    return tokens.to(torch.int32), count.to(torch.int32)


# ------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, s)
    return _exact_attend(case, s) if case["kind"] == "attend" else _exact_verify(case, s)


def _exact_append(case, s):
    def turned(p, angle):
        half = ROPE // 2
        z = torch.complex(angle[..., :half].contiguous(), angle[..., half:].contiguous())
        if case["interleaved"]:
            pairs = torch.view_as_complex(p.reshape(*p.shape[:-1], half, 2).contiguous())
            return torch.view_as_real(pairs * z).flatten(-2)
        w = torch.complex(p[..., :half].contiguous(), p[..., half:].contiguous()) * z
        return torch.cat((w.real, w.imag), dim=-1)

    x = s["x"].double()
    if s["norm"] is not None:
        x = x / (x.square().sum(dim=1, keepdim=True) / LATENT + EPS).sqrt() * s["norm"].double()
    angle = s["cos_sin"].double()[s["positions"]]
    cache = s["cache"].double().view(-1, WIDTH)
    cache[s["slots"].long(), :LATENT] = x
    cache[s["slots"].long(), LATENT:] = turned(s["k_pe"].double(), angle)
    q = None
    if s["q"] is not None:
        q = s["q"].double()
        q[:, :, LATENT:] = turned(s["q_pe"].double(), angle[:, None])
    return {"cache": cache.view(s["cache"].shape), "q": q}


def _exact_attend(case, s):
    news, lens = _lengths(case)
    heads, block, int8 = case["heads"], case["block"], case["cache"] == "int8"
    outs, lses, at = [], [], 0
    for r, (n, length) in enumerate(zip(news, lens)):
        pages = s["table"][r, :(length + block - 1) // block].long()
        rows = s["cache"][pages].flatten(0, 1)[:length]
        if int8:
            scale = rows[:, LATENT:LATENT + 4].contiguous().view(torch.float32).double()
            k = rows[:, :LATENT].double() * scale
        else:
            k = rows.double()
        v = k[:, :LATENT].contiguous()
        kt = k.t().contiguous()
        hidden = torch.arange(length, device="cuda")[None] > torch.arange(length - n, length, device="cuda")[:, None]
        out = torch.empty(n, heads, LATENT, dtype=torch.float64, device="cuda")
        lse = torch.empty(n, heads, dtype=torch.float64, device="cuda")
        for h in range(heads):
            a = (s["q"][at:at + n, h].double() @ kt * SM_SCALE).masked_fill_(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(a, dim=1)
            out[:, h] = torch.softmax(a, dim=1) @ v
        outs.append(out)
        lses.append(lse)
        at += n
    out = torch.cat(outs)
    return (out, torch.cat(lses)) if case["lse"] else out


def _exact_verify(case, s):
    cu, ids, accept = s["cu"].tolist(), s["ids"].tolist(), s["accept_u"].tolist()
    most = case["drafts"]
    tokens = torch.full((len(cu) - 1, most + 1), -1, dtype=torch.int32)
    counts = torch.zeros(len(cu) - 1, dtype=torch.int32)
    for r in range(len(cu) - 1):
        n, first = min(cu[r + 1] - cu[r] - 1, most), cu[r]
        p = s["target"][first:first + n + 1].cpu()
        d = s["draft"][first - r:first - r + n].cpu() if s["draft"] is not None else None
        k = 0
        while k < n:
            x = ids[first - r + k]
            seen = torch.tensor(accept[first - r + k], dtype=torch.float32)
            if not float(seen * d[k, x] if d is not None else seen) < float(p[k, x]):
                break
            tokens[r, k] = x
            k += 1
        left = p[k].clone()
        if k < n:
            if d is None:
                left[ids[first - r + k]] = 0
            else:
                left = (left - d[k]).clamp_min(0)
        parts = (left.double() * 2.0 ** 40).floor().to(torch.int64)
        if int(parts.sum()) == 0:
            parts = (p[k].double() * 2.0 ** 40).floor().to(torch.int64)
        below = parts.cumsum(0)
        mark = min(int(float(s["sample_u"][r]) * float(below[-1])), int(below[-1]) - 1)
        tokens[r, k] = int((below > mark).nonzero()[0])
        counts[r] = k
    return tokens.cuda(), counts.cuda()


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    if case["kind"] == "append":
        n, heads = case["tokens"], case["heads"]
        per_angle = ROPE * (4 if case["table"] == "fp32" else 2)
        per_token = 2 * (2 * WIDTH) + 8 + (8 if case["slots64"] else 4) + per_angle + 2 * heads * ROPE * 2
        return {"bytes": n * per_token, "flops": n * ((4 * LATENT if case["norm"] else 0) + 3 * ROPE * (heads + 1))}
    if case["kind"] == "attend":
        news, lens = _lengths(case)
        heads, width = case["heads"], LATENT if case["cache"] == "int8" else WIDTH
        seen = sum(n * length - n * (n - 1) // 2 for n, length in zip(news, lens))
        row = ROW if case["cache"] == "int8" else 2 * WIDTH
        moved = sum(lens) * row + sum(news) * heads * 2 * (width + LATENT)
        if case["lse"]:
            moved += sum(news) * heads * 4
        return {"bytes": moved, "flops": 2 * seen * heads * (width + LATENT)}
    # the decided row of each request, and the drafts' row beside it
    rows = case["requests"] * (2 if case["draft_probs"] else 1)
    return {"bytes": rows * case["vocab"] * 4 + case["requests"] * (case["drafts"] * 24 + 16),
            "flops": 2 * rows * case["vocab"]}
