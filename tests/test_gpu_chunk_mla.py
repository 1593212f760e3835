"""titan_mla.mla_chunk_attention_paged against the 64-bit form."""
import math

import pytest
import torch

import chunk_oracle as O
from conftest import log_case

pytestmark = pytest.mark.gpu
SCALE = O.WIDTH ** -0.5


def make(dev, seed, news, lens, heads, int8, block, spare=1, table_cols=None, q_scale=1.0):
    """Inputs with every request's pages scattered; unused rows hold NaN (bf16)
    or garbage codes with a NaN scale (INT8)."""
    g = torch.Generator(device="cpu").manual_seed(seed)
    used = [max(0, -(-n // block)) for n in lens]
    pages = sum(used) + spare
    cols = table_cols or max(1, max(used, default=1))
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(news), cols), -1, dtype=torch.int32)
    if int8:
        rows = torch.zeros(pages * block, O.ROW, dtype=torch.int8)
        rows[:, :O.LATENT] = (torch.randn(pages * block, O.LATENT, generator=g) * 40).round().clamp(-127, 127)
        rows[:, O.LATENT:O.LATENT + 4] = torch.full((pages * block, 1), math.nan).view(torch.int8)
        scale = (torch.rand(pages * block, 1, generator=g) * 0.012 + 0.02).view(torch.int8)
    else:
        rows = torch.full((pages * block, O.WIDTH), math.nan, dtype=torch.bfloat16)
        data = torch.randn(pages * block, O.WIDTH, generator=g).to(torch.bfloat16)
    at = 0
    for r, n in enumerate(lens):
        table[r, :used[r]] = order[at:at + used[r]].to(torch.int32)[:cols]
        pos = torch.arange(max(n, 0))
        row = table[r, pos // block].long() * block + pos % block
        if int8:
            rows[row, O.LATENT:O.LATENT + 4] = scale[row]
        else:
            rows[row] = data[row]
        at += used[r]
    total = sum(news)
    q = (torch.randn(total, heads, O.LATENT if int8 else O.WIDTH, generator=g) * q_scale).to(torch.bfloat16)
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32)
    return (q.to(dev), rows.view(pages, block, -1).to(dev), cu.to(dev),
            torch.tensor(lens, dtype=torch.int32, device=dev), table.to(dev))


def check(got, lse, q, cache, cu, lens, table):
    want, want_lse, spread = O.attend(q, cache, cu, lens, table, SCALE)
    end = int(cu[-1])
    err = (got.double().cpu() - want).abs()[:end]
    bound = O.attention_bound(want, spread)[:end]
    assert bool((err <= bound).all()), f"worst {float((err - bound).max())} over the bound"
    if lse is not None:
        a, b = lse.double().cpu()[:end], want_lse[:end]
        assert bool((torch.isneginf(a) == torch.isneginf(b)).all())
        fine = ~torch.isneginf(b)
        assert bool(((a - b)[fine].abs() <= 1e-3).all())   # the logits' 2^-10, and the sum's fp32


CASES = [
    # news, lens, heads, block
    ([1], [1], 16, 64),
    ([1], [64], 16, 64),
    ([1], [65], 16, 64),
    ([1], [1999], 16, 64),
    ([1], [700], 1, 1),
    ([1, 1, 1], [130, 1, 63], 16, 16),
    ([1, 1], [100, 257], 128, 256),
    ([1, 1], [300, 77], 20, 48),
    ([2, 2, 2], [65, 2, 200], 16, 64),
    ([4, 3, 1, 8], [400, 3, 1, 70], 16, 64),
    ([5, 0, 2], [5, 40, 0], 16, 16),          # a request without tokens, one whose tokens see nothing
    ([7], [3], 3, 64),                        # tokens before the sequence's start
    ([70, 33], [70, 300], 16, 48),
    ([129], [129], 8, 64),
    ([33], [450], 20, 16),
    ([0, 0, 1], [10, 0, 20], 16, 64),
]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_against_64_bits(cuda, case, int8):
    news, lens, heads, block = CASES[case]
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, case, news, lens, heads, int8, block)
    log_case("chunk_mla", "int8" if int8 else "bf16", news, lens, heads, block)
    out, lse = mla_chunk_attention_paged(*a, SCALE, return_lse=True)
    check(out, lse, *a)
    again = mla_chunk_attention_paged(*a, SCALE)
    assert torch.equal(out, again)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("shape", ["rows64", "rows32", "rows16"])
def test_many_tiles(cuda, shape, int8):
    """More tiles than the split form takes: one workgroup each."""
    from titan_mla import mla_chunk_attention_paged
    news, lens, heads = {"rows64": ([270, 3], [300, 131], 128),
                         "rows32": ([2] * 520, [2 + 3 * (i % 50) for i in range(520)], 16),
                         "rows16": ([1] * 600, [i % 150 for i in range(600)], 4)}[shape]
    a = make(cuda, 5, news, lens, heads, int8, 64)
    log_case("chunk_mla many tiles", shape, int8)
    out, lse = mla_chunk_attention_paged(*a, SCALE, return_lse=True)
    check(out, lse, *a)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_growing_maxima(cuda, int8):
    """Logits that rise along the sequence, by far more than the kernel lets a
    maximum pass its reference, and fall."""
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 9, [3, 1], [500, 400], 16, int8, 64)
    if int8:
        scale = cache[..., O.LATENT:O.LATENT + 4].contiguous().view(torch.float32)
        ramp = torch.linspace(0.05, 3, cache.shape[0] * 64, device=cuda).view(-1, 64, 1)
        cache[..., O.LATENT:O.LATENT + 4] = (scale * ramp).view(torch.int8)
    else:
        cache *= torch.linspace(0.05, 3, cache.shape[0] * 64, device=cuda).view(-1, 64, 1)
    log_case("chunk_mla growing maxima", int8)
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
    want, want_lse, spread = O.attend(q, cache, cu, lens, table, SCALE)
    # three times the data: the logits' sums may be off by three times 2^-10
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 6 * 2.0 ** -10) * spread
    assert bool(((out.double().cpu() - want).abs() <= bound).all())
    assert bool(((lse.double().cpu() - want_lse).abs() <= 3e-3).all())


def test_pages_outside_the_cache_are_masked(cuda):
    from titan_mla import mla_chunk_attention_paged
    for int8 in (False, True):
        q, cache, cu, lens, table = make(cuda, 3, [2, 1], [384, 336], 16, int8, 48)   # whole pages
        table[0, 2] = cache.shape[0]
        table[0, 4] = -7
        table[1, 0] = 2 ** 31 - 1
        log_case("chunk_mla pages outside", int8)
        out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
        check(out, lse, q, cache, cu, lens, table)
        # lengths past the table: the positions that it has
        longer = lens + 10000
        out, lse = mla_chunk_attention_paged(q, cache, cu, longer, table, SCALE, return_lse=True)
        check(out, lse, q, cache, cu, longer, table)
        # nothing but masked pages
        out, lse = mla_chunk_attention_paged(q, cache, cu, lens, torch.full_like(table, -1), SCALE, return_lse=True)
        assert not out.any() and bool(torch.isneginf(lse).all())
        empty = table[:, :0]
        out, lse = mla_chunk_attention_paged(q, cache, cu, lens, empty, SCALE, return_lse=True)
        assert not out.any() and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_later_tokens_that_are_not_finite(cuda, bad):
    """A later token of the chunk with NaN or infinities leaves the rows before
    it as they are, and makes its own NaN."""
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 4, [6], [100], 16, False, 64)
    clean = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE)
    pos = 97   # the fourth of the six
    cache[int(table[0, pos // 64]), pos % 64, 5:40] = bad
    log_case("chunk_mla not finite", bad)
    out = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE)
    assert torch.equal(out[:3], clean[:3])
    if not math.isinf(bad):
        assert bool(out[3:].isnan().all())


def test_strides_padding_and_out(cuda):
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 6, [3, 2], [90, 200], 16, False, 48)
    plain = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE)
    # pages with padding between them, rows with padding, queries inside a wider buffer, padded tokens
    wide = torch.full((cache.shape[0], 50, 592), math.nan, dtype=torch.bfloat16, device=cuda)
    wide[:, :48, :576] = cache
    qw = torch.full((9, 20, 600), math.nan, dtype=torch.bfloat16, device=cuda)
    qw[:5, 2:18, 8:584] = q
    out = torch.full((9, 16, 520), 7.0, dtype=torch.bfloat16, device=cuda)
    log_case("chunk_mla strides")
    got = mla_chunk_attention_paged(qw[:, 2:18, 8:584], wide[:, :48, :576], cu, lens, table, SCALE, out=out[:, :, 4:516])
    assert got.data_ptr() == out[:, :, 4:].data_ptr()
    assert torch.equal(out[:5, :, 4:516], plain)
    assert bool((out[5:] == 7).all()) and bool((out[:, :, :4] == 7).all()) and bool((out[:, :, 516:] == 7).all())
    # strides that only a copy mends
    odd = torch.zeros(5, 16, 577, dtype=torch.bfloat16, device=cuda)
    odd[:, :, 1:] = q
    t2 = torch.stack((table, table), dim=2)[:, :, 0]
    assert torch.equal(mla_chunk_attention_paged(odd[:, :, 1:], cache, cu, lens, t2, SCALE), plain)
    # lists of two, every other
    c2 = torch.stack((cu, cu), dim=1)[:, 0]
    assert torch.equal(mla_chunk_attention_paged(q, cache, c2, lens, table, SCALE), plain)
    # nothing to do
    none = mla_chunk_attention_paged(q[:0], cache, cu[:1], lens[:0], table[:0], SCALE)
    assert none.shape == (0, 16, 512)


def test_cache_past_four_gibibytes(cuda):
    from titan_mla import mla_chunk_attention_paged
    for int8 in (False, True):
        width, size = (528, 1) if int8 else (576, 2)
        pages = (5 << 30) // (64 * width * size)
        q, small, cu, lens, table = make(cuda, 8, [2, 1], [150, 90], 16, int8, 64)
        want = mla_chunk_attention_paged(q, small, cu, lens, table, SCALE)
        big = torch.empty((pages, 64, width), dtype=small.dtype, device=cuda)
        high = (pages - 1 - table).to(torch.int32)
        high[table < 0] = -1
        for p in table.unique().tolist():
            if p >= 0:
                big[pages - 1 - p] = small[p]
        log_case("chunk_mla 5 GiB", int8)
        assert torch.equal(mla_chunk_attention_paged(q, big, cu, lens, high, SCALE), want)
        del big


def test_captured_and_replayed(cuda):
    """A graph whose lengths and tables change between replays."""
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 10, [1] * 6, [40, 700, 333, 64, 65, 1], 16, True, 64)
    out = torch.zeros(6, 16, 512, dtype=torch.bfloat16, device=cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, out=out)
    full = lens.clone()
    for k in range(4):
        lens.copy_((full - k).clamp_min(0))
        q.copy_(torch.roll(q, 1, 0))
        log_case("chunk_mla replay", k)
        graph.replay()
        torch.cuda.synchronize()
        eager = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE)
        assert torch.equal(out, eager)
        check(out, None, q, cache, cu, lens, table)


def test_two_streams_at_once(cuda):
    """Two calls side by side, each with its own workspace."""
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, 11, [4, 4, 4], [900, 2000, 77], 16, False, 64)
    b = make(cuda, 12, [1] * 9, [300 + 111 * i for i in range(9)], 16, True, 64)
    want_a, want_b = mla_chunk_attention_paged(*a, SCALE), mla_chunk_attention_paged(*b, SCALE)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    got_a, got_b = [], []
    for _ in range(5):
        with torch.cuda.stream(s):
            got_a.append(mla_chunk_attention_paged(*a, SCALE))
        with torch.cuda.stream(t):
            got_b.append(mla_chunk_attention_paged(*b, SCALE))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want_a) for x in got_a) and all(torch.equal(x, want_b) for x in got_b)


def test_the_sparse_attention_of_all_positions(cuda):
    """Over the INT8 cache, the indexed attention with every position listed."""
    from titan_mla import mla_chunk_attention_paged, triton_mla_sparse_attention_paged
    q, cache, cu, lens, table = make(cuda, 13, [1] * 4, [500, 33, 640, 127], 16, True, 64)
    idx = torch.arange(640, dtype=torch.int32, device=cuda)[None].repeat(4, 1)
    idx[idx >= lens[:, None]] = -1
    req = torch.arange(4, dtype=torch.int32, device=cuda)
    sparse = triton_mla_sparse_attention_paged(q, cache, idx, req, table, SCALE)
    dense = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE)
    want, _, spread = O.attend(q, cache, cu, lens, table, SCALE)
    bound = 2 * O.attention_bound(want, spread)   # both are within it of the same value
    assert bool(((dense.double() - sparse.double()).abs().cpu() <= bound).all())
