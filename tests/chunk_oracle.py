"""Plain 64-bit forms (on the CPU) of the chunk operators: attention over a
paged cache, the rotary cache writer and draft verification."""
import math

import torch

LATENT, ROPE, WIDTH, ROW = 512, 64, 576, 528


def keys_of(cache):
    """float64 keys [pages, block, width] of a bf16 or INT8 cache (on the CPU)."""
    if cache.dtype == torch.bfloat16:
        return cache.double()
    scale = cache[..., LATENT:LATENT + 4].contiguous().view(torch.float32).double()
    return cache[..., :LATENT].double() * scale


def attend(q, cache, cu, lens, table, sm_scale):
    """(out, lse, spread) in float64 for the tokens below cu[-1], the others
    zero; spread is sum_j p_j |v_j|, what the kernel's rounding of P scales with."""
    q, cu, lens, table = q.double().cpu(), cu.tolist(), lens.tolist(), table.cpu()
    cache = cache.cpu()
    pages, block = cache.shape[:2]
    T, H, _ = q.shape
    out = torch.zeros(T, H, LATENT, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    for r, length in enumerate(lens):
        n = cu[r + 1] - cu[r]
        length = min(length, table.shape[1] * block)
        full = lens[r]
        pos = torch.arange(max(length, 0))
        page = table[r, pos // block].long() if length > 0 else pos
        there = (page >= 0) & (page < pages)
        rows = cache[page.clamp(0, pages - 1), pos % block] if length > 0 else cache[:0, 0]
        k = keys_of(rows)
        for i in range(n):
            see = there & (pos <= full - n + i)
            if not bool(see.any()):
                continue
            ki = k[see]
            s = q[cu[r] + i] @ ki.t() * sm_scale
            p = torch.softmax(s, dim=1)
            out[cu[r] + i] = p @ ki[:, :LATENT]
            spread[cu[r] + i] = p @ ki[:, :LATENT].abs()
            lse[cu[r] + i] = torch.logsumexp(s, dim=1)
    return out, lse, spread


def attention_bound(out, spread):
    """Elementwise bound of the kernel's error: the output's rounding to bf16
    (half a step, 2^-8), each weight's rounding to bf16 (2^-8 of sum p |v|),
    and the logits' fp32 sums: 576 products of at most 15 in sum (the tests'
    unit-normal data after the scale) err by at most 576 * 2^-24 * 15 < 2^-10,
    which moves weights and their sum by 2^-9 together."""
    return 2.0 ** -8 * out.abs() + (2.0 ** -8 + 2.0 ** -9) * spread


def rotate(p, cos, sin, interleaved):
    half = ROPE // 2
    a, b = (p[..., 0::2], p[..., 1::2]) if interleaved else (p[..., :half], p[..., half:])
    u, v = a * cos - b * sin, b * cos + a * sin
    return torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)


def verify(target, ids, draft, cu, accept_u, sample_u, most):
    """(tokens, accepted) in whole numbers, from the definition."""
    target, ids, cu = target.cpu(), ids.tolist(), cu.tolist()
    draft = draft.cpu() if draft is not None else None
    rows, vocab = target.shape
    R = len(cu) - 1
    tokens = torch.full((R, most + 1), -1, dtype=torch.int32)
    counts = torch.zeros(R, dtype=torch.int32)

    def weights(x):
        x = torch.nan_to_num(x.double(), nan=0.0, posinf=1.0, neginf=0.0).clamp(0, 1)
        return (x * 2.0 ** 40).floor().to(torch.int64)

    for r in range(R):
        first, n = cu[r], min(cu[r + 1] - cu[r] - 1, most)
        if first < 0 or cu[r + 1] > rows or n < 0 or first - r < 0 or first - r + n > len(ids):
            continue
        k = 0
        while k < n:
            at = first - r + k
            x = ids[at]
            if not 0 <= x < vocab:
                break
            u = accept_u[at].cpu()
            q = draft[at, x] if draft is not None else torch.tensor(1.0)
            if not bool(u * q < target[first + k, x]):
                break
            tokens[r, k] = x
            k += 1
        counts[r] = k
        p = target[first + k]
        rest = p.clone()
        if k < n:
            if draft is not None:
                rest = p - draft[first - r + k]
            elif 0 <= ids[first - r + k] < vocab:
                rest[ids[first - r + k]] = 0
        w = weights(rest)
        if int(w.sum()) == 0:
            w = weights(p)
        total = int(w.sum())
        if total:
            mark = min(int(math.floor(float(sample_u[r]) * float(total))), total - 1)
            tokens[r, k] = int((w.cumsum(0) > mark).nonzero()[0])
    return tokens, counts
