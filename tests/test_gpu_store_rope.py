"""titan_kv.store_rope against the 64-bit form."""
import math

import pytest
import torch

import chunk_oracle as O
from conftest import log_case

pytestmark = pytest.mark.gpu
EPS = 1e-6


def make(dev, seed, n, heads, block, pages, table_dtype, max_pos=1000, idx=torch.int64):
    g = torch.Generator(device="cpu").manual_seed(seed)
    angle = torch.arange(max_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, 64, 2) / 64.0)
    d = {"x": torch.randn(n, 512, generator=g).to(torch.bfloat16) * 3,
         "k_pe": torch.randn(n, 64, generator=g).to(torch.bfloat16),
         "positions": torch.randint(0, max_pos, (n,), generator=g).to(idx),
         "cos_sin": torch.cat((angle.cos(), angle.sin()), dim=1).to(table_dtype),
         "cache": torch.full((pages, block, 576), 9.0, dtype=torch.bfloat16),
         "slots": torch.randperm(pages * block, generator=g)[:n].to(idx),
         "q_pe": torch.randn(n, heads, 64, generator=g).to(torch.bfloat16) if heads else None,
         "norm_weight": (torch.rand(512, generator=g) + 0.5).to(torch.bfloat16)}
    return {k: v.to(dev) if v is not None else None for k, v in d.items()}


def reference(d, norm, interleaved):
    x = d["x"].double().cpu()
    if norm:
        x = x / (x.square().mean(dim=1, keepdim=True) + EPS).sqrt() * d["norm_weight"].double().cpu()
    t = d["cos_sin"].double().cpu()[d["positions"].long().cpu()]
    cos, sin = t[:, :32], t[:, 32:]
    k = O.rotate(d["k_pe"].double().cpu(), cos, sin, interleaved)
    q = O.rotate(d["q_pe"].double().cpu(), cos[:, None], sin[:, None], interleaved) if d["q_pe"] is not None else None
    return torch.cat((x, k), dim=1), q


def close(got, want, size):
    """One rounding to bf16 (2^-8 of the value) and fp32 arithmetic: two
    products and their sum, or the norm's chain (the sum of 512 squares in a
    tree of 8 + 6 steps, a division, a root, two products), under 16 roundings
    of 2^-24 of `size`."""
    err = (got.double().cpu() - want).abs()
    return bool((err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * size).all())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("n,heads,block,table,idx", [
    (1, 16, 64, torch.float32, torch.int64), (1, 0, 1, torch.float32, torch.int32),
    (5, 1, 48, torch.bfloat16, torch.int32), (33, 20, 16, torch.float32, torch.int64),
    (300, 8, 64, torch.bfloat16, torch.int64), (17, 130, 256, torch.float32, torch.int32)])
def test_against_64_bits(cuda, n, heads, block, table, idx, norm, interleaved):
    from titan_kv import store_rope
    d = make(cuda, n + heads, n, heads, block, (2 * n) // block + 2, table, idx=idx)
    log_case("store_rope", n, heads, block, table, idx, norm, interleaved)
    q = store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], d["cache"], d["slots"], q_pe=d["q_pe"],
                   norm_weight=d["norm_weight"] if norm else None, eps=EPS, interleaved=interleaved)
    rows, qs = reference(d, norm, interleaved)
    flat = d["cache"].view(-1, 576).cpu()
    slots = d["slots"].long().cpu()
    got = flat[slots]
    if norm:
        assert close(got[:, :512], rows[:, :512], rows[:, :512].abs())
    else:
        assert torch.equal(got[:, :512], d["x"].cpu())
    assert close(got[:, 512:], rows[:, 512:], 2 * d["k_pe"].abs().max().item())
    untouched = torch.ones(flat.shape[0], dtype=torch.bool)
    untouched[slots] = False
    assert bool((flat[untouched] == 9).all())
    if heads:
        assert close(q, qs, 2 * d["q_pe"].abs().max().item())
    else:
        assert q is None


def test_padding_skips_and_positions_outside(cuda):
    from titan_kv import store_rope
    d = make(cuda, 1, 9, 4, 16, 4, torch.float32)
    d["slots"] = torch.tensor([5, -1, 64, 63, 2 ** 40, 11, -2 ** 40], device=cuda)   # 64 rows; two tokens of padding
    d["positions"][5] = 1000
    d["positions"][3] = -1
    d["x"][7:] = math.nan
    q_out = torch.full((9, 4, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    log_case("store_rope skips")
    got = store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], d["cache"], d["slots"], q_pe=d["q_pe"],
                     q_out=q_out)
    assert got is q_out
    d["positions"][5] = d["positions"][3] = 0   # for the reference's look-up
    rows, qs = reference(d, False, False)
    flat = d["cache"].view(-1, 576).cpu()
    assert torch.equal(flat[5, :512], d["x"][0].cpu())
    flat[5] = 9
    assert bool((flat == 9).all())
    assert bool((q_out[7:] == 7).all()) and not q_out[5].any() and not q_out[3].any()
    for i in (0, 1, 2, 4, 6):
        assert close(q_out[i], qs[i], 2 * d["q_pe"].abs().max().item())


def test_strides_views_and_in_place(cuda):
    from titan_kv import store_rope
    n, H = 6, 5
    d = make(cuda, 2, n, H, 16, 3, torch.float32)
    plain = d["cache"].clone()
    args = lambda c: (d["x"], d["k_pe"], d["positions"], d["cos_sin"], c, d["slots"])   # noqa: E731
    want = store_rope(*args(plain), q_pe=d["q_pe"], norm_weight=d["norm_weight"])
    # padded pages and rows, inputs inside wider buffers (aligned and not), queries' own part written in place
    wide = torch.full((3, 20, 592), 9.0, dtype=torch.bfloat16, device=cuda)
    x = torch.zeros(n, 640, dtype=torch.bfloat16, device=cuda)
    x[:, 3:515] = d["x"]
    k = torch.zeros(n, 2, 64, dtype=torch.bfloat16, device=cuda)
    k[:, 1] = d["k_pe"]
    qf = torch.full((n, H, 192), 5.0, dtype=torch.bfloat16, device=cuda)
    qf[:, :, 128:] = d["q_pe"]
    t = torch.zeros(1000, 65, device=cuda)
    t[:, 1:] = d["cos_sin"]
    w = torch.zeros(513, dtype=torch.bfloat16, device=cuda)
    w[1:] = d["norm_weight"]
    pos2, slots2 = torch.stack((d["positions"],) * 2, 1)[:, 0], torch.stack((d["slots"],) * 2, 1)[:, 0]
    log_case("store_rope strides")
    got = store_rope(x[:, 3:515], k[:, 1], pos2, t[:, 1:], wide[:, :16, :576], slots2, q_pe=qf[:, :, 128:],
                     q_out=qf[:, :, 128:], norm_weight=w[1:])
    assert torch.equal(got, want) and torch.equal(wide[:, :16, :576], plain)
    assert bool((qf[:, :, :128] == 5).all())
    assert bool((wide[:, 16:] == 9).all()) and bool((wide[:, :, 576:] == 9).all())
    # no slots, no tokens
    before = plain.clone()
    store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], plain, d["slots"][:0])
    store_rope(d["x"][:0], d["k_pe"][:0], d["positions"][:0], d["cos_sin"], plain, d["slots"][:0])
    assert torch.equal(plain, before)


def test_cache_past_four_gibibytes(cuda):
    from titan_kv import store_rope
    d = make(cuda, 3, 3, 0, 64, 1, torch.float32)
    pages = (5 << 30) // (64 * 576 * 2)
    cache = torch.zeros(pages, 64, 576, dtype=torch.bfloat16, device=cuda)
    d["slots"] = torch.tensor([pages * 64 - 1, 7, pages * 64 // 2], device=cuda)
    log_case("store_rope 5 GiB")
    store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], cache, d["slots"])
    flat = cache.view(-1, 576)
    assert torch.equal(flat[d["slots"], :512], d["x"])
    flat[d["slots"]] = 0
    assert not cache.view(torch.int32).any()


def test_captured_and_replayed(cuda):
    from titan_kv import store_rope
    d = make(cuda, 4, 8, 16, 64, 4, torch.float32)
    q = torch.zeros(8, 16, 576, dtype=torch.bfloat16, device=cuda)
    call = lambda c, o: store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], c, d["slots"],   # noqa: E731
                                   q_pe=d["q_pe"], q_out=o[:, :, 512:], norm_weight=d["norm_weight"], interleaved=True)
    call(d["cache"], q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d["cache"], q)
    for k in range(3):
        d["x"].copy_(torch.roll(d["x"], 1, 0))
        d["positions"].add_(17).remainder_(1000)
        d["slots"].add_(8).remainder_(256)
        other, oq = d["cache"].clone(), q.clone()
        log_case("store_rope replay", k)
        graph.replay()
        torch.cuda.synchronize()
        call(other, oq)
        assert torch.equal(other, d["cache"]) and torch.equal(q, oq)
