"""The chunk operators at the sizes where their forms change, and one after
another as a step of drafts uses them: append, attend, verify."""
import math

import pytest
import torch

import chunk_oracle as O
from conftest import log_case
from test_gpu_chunk_mla import SCALE, check, make
import test_gpu_store_rope as rope
import test_gpu_verify_drafts as drafts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("news,lens,heads,block", [
    ([40, 3], [260, 90], 20, 12),          # pages that are no multiple of eight rows: 64-row tiles
    ([2, 2, 1], [700, 90, 333], 16, 7),    # 32-row tiles
    ([1, 1], [500, 129], 16, 3),           # 16-row tiles
    ([9], [200], 128, 20),
    ([2, 1], [260, 31], 16, 8),            # pages of eight rows
    ([3, 5], [77, 500], 16, 24),
])
def test_pages_of_any_size(cuda, news, lens, heads, block, int8):
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, block, news, lens, heads, int8, block)
    log_case("chunk_mla pages", news, lens, heads, block, int8)
    out, lse = mla_chunk_attention_paged(*a, SCALE, return_lse=True)
    check(out, lse, *a)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("block", [64, 20])
def test_long_walks_over_the_table(cuda, block, int8):
    """One workgroup walks more blocks of 32 keys than the 64 whose table
    entries it holds: a long prompt, looked at for a few of its tokens."""
    from titan_mla import mla_chunk_attention_paged
    n, length, heads = 2100, 7000, 16
    q, cache, cu, lens, table = make(cuda, 21, [n], [length], heads, int8, block)
    log_case("chunk_mla long walk", block, int8)
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
    for t in (0, 1, 3, 1023, 1500, 2099):
        one = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
        upto = torch.tensor([length - n + t + 1], dtype=torch.int32, device=cuda)
        check(out[t:t + 1], lse[t:t + 1], q[t:t + 1], cache, one, upto, table)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_many_requests_on_long_contexts(cuda, int8):
    """Runs that hold the ends of some tiles and the starts of others."""
    from titan_mla import mla_chunk_attention_paged
    news = [1, 2, 4, 1, 3, 0, 1, 2, 1, 4, 4, 1]
    lens = [5000, 2, 900, 64, 3, 77, 4097, 0, 1, 33, 2500, 6000]
    a = make(cuda, 22, news, lens, 16, int8, 64)
    log_case("chunk_mla runs", int8)
    out, lse = mla_chunk_attention_paged(*a, SCALE, return_lse=True)
    check(out, lse, *a)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("news,lens,heads", [
    ([150, 90, 0, 80, 60], [200, 170, 5, 80, 300], 64),
    ([150, 90, 0, 80, 60], [1500, 1400, 5, 1300, 1450], 64),
    ([1] * 300, [1 + 37 * (i % 40) for i in range(300)], 16),
    ([2] * 300, [2000 if i == 7 else i % 3 for i in range(300)], 16),
    ([1] * 480, [i % 90 for i in range(480)], 1),     # as many requests as the split form takes
    ([0] * 255 + [1] + [0] * 256, [5] * 255 + [70] + [5] * 256, 1),
])
def test_more_tiles_than_compute_units(cuda, news, lens, heads, int8):
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, 25, news, lens, heads, int8, 64)
    log_case("chunk_mla tiles", len(news), heads, int8)
    out, lse = mla_chunk_attention_paged(*a, SCALE, return_lse=True)
    check(out, lse, *a)


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("scale", [-0.03, 0.0, 1e-30])
def test_scales(cuda, scale, int8):
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 23, [3, 1], [200, 70], 16, int8, 64)
    log_case("chunk_mla scale", scale, int8)
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, scale, return_lse=True)
    want, want_lse, spread = O.attend(q, cache, cu, lens, table, scale)
    assert bool(((out.double().cpu() - want).abs() <= O.attention_bound(want, spread)).all())
    # the sums' and the logarithm's fp32 roundings, as in the other tests' data: under 2^-10
    assert bool(((lse.double().cpu() - want_lse).abs() <= 2.0 ** -10).all())


@pytest.mark.parametrize("heads", [16, 64])
def test_key_scales_of_any_size(cuda, heads):
    """INT8 rows whose scales are 0, negative, below any normal weight's range,
    or (behind the last position) no numbers."""
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 26, [2, 1], [130, 45], heads, True, 64)
    scale = cache[..., O.LATENT:O.LATENT + 4].contiguous().view(torch.float32)
    for i, v in enumerate((0.0, -0.03, 1e-25, 1e-12, -1e-40, -0.0)):
        scale.view(-1)[i::7] = torch.where(scale.view(-1)[i::7].isnan(), math.nan, v)
    cache[..., O.LATENT:O.LATENT + 4] = scale.view(torch.int8)
    log_case("chunk_mla key scales", heads)
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
    check(out, lse, q, cache, cu, lens, table)


@pytest.mark.parametrize("heads", [4, 16, 64])
def test_one_key_is_that_key(cuda, heads):
    """One visible key: its INT8 row times its scale, rounded once."""
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, 27, [1, 1, 1], [1, 1, 1], heads, True, 16)
    log_case("chunk_mla one key", heads)
    out = mla_chunk_attention_paged(*a, SCALE)
    want = O.attend(*a, SCALE)[0]
    # a value in [2^e, 2^(e + 1)) has bf16 neighbours 2^(e - 7) apart, so that rounding it is off by at most
    # 2^(e - 8), 2^-8 of it; the scale's logarithm, power and quotient in fp32 add less than 2^-18
    assert bool(((out.double().cpu() - want).abs() <= (2.0 ** -8 + 2.0 ** -18) * want.abs()).all())


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_a_row_that_turns_to_a_late_key(cuda, int8):
    """One row of a tile meets a key far above all before it, in a block where
    the others' references stay."""
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 24, [4], [600], 16, int8, 64)
    pos, head = 500, 5
    row = cache[int(table[0, pos // 64]), pos % 64]
    key = O.keys_of(row.cpu()[None])[0].to(cuda)
    q[2, head] = (key * (60.0 / float(key.square().sum()) / SCALE)).to(torch.bfloat16)[:q.shape[2]]
    log_case("chunk_mla late key", int8)
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
    want, want_lse, spread = O.attend(q, cache, cu, lens, table, SCALE)
    # that row's logit is four times the 15 of the bound's data: 2^-10 becomes 2^-8 there
    bound = O.attention_bound(want, spread) + 2.0 ** -7 * spread
    assert bool(((out.double().cpu() - want).abs() <= bound).all())
    assert float(lse[2, head]) > 55


@pytest.mark.parametrize("heads", [0, 9])
@pytest.mark.parametrize("n", [8192, 8195, 8191])
def test_appending_many_tokens(cuda, n, heads):
    """On both sides of the size from which a wave takes four tokens, with
    tokens that are skipped."""
    from titan_kv import store_rope
    d = rope.make(cuda, n, n, heads, 48, n // 48 + 9, torch.float32, idx=torch.int32)
    d["slots"][5::97] = -1
    d["slots"][n - 1] = n // 48 * 48 + 9 * 48      # past the cache
    d["positions"][7::501] = 1000                  # past the table
    log_case("store_rope many", n, heads)
    q = store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], d["cache"], d["slots"], q_pe=d["q_pe"],
                   norm_weight=d["norm_weight"], eps=rope.EPS, interleaved=True)
    known = d["positions"].cpu() < 1000
    d["positions"].clamp_(max=999)                 # for the reference's look-up
    rows, qs = rope.reference(d, True, True)
    flat, slots = d["cache"].view(-1, 576).cpu(), d["slots"].long().cpu()
    kept = known & (slots >= 0) & (slots < flat.shape[0])
    got = flat[slots[kept]]
    assert rope.close(got[:, :512], rows[kept, :512], rows[kept, :512].abs())
    assert rope.close(got[:, 512:], rows[kept, 512:], 2 * d["k_pe"].abs().max().item())
    untouched = torch.ones(flat.shape[0], dtype=torch.bool)
    untouched[slots[kept]] = False
    assert bool((flat[untouched] == 9).all())
    if heads:
        assert rope.close(q.cpu()[known], qs[known], 2 * d["q_pe"].abs().max().item())
        assert not q.cpu()[~known].any()


def test_caches_and_tables_without_rows(cuda):
    """No page, no position: nothing is stored or seen, queries without an
    angle are zero."""
    from titan_kv import store_rope
    from titan_mla import mla_chunk_attention_paged
    d = rope.make(cuda, 3, 4, 2, 16, 1, torch.float32)
    log_case("empty cache")
    q = store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], d["cache"][:0], d["slots"], q_pe=d["q_pe"])
    assert rope.close(q, rope.reference(d, False, False)[1], 2 * d["q_pe"].abs().max().item())
    before = d["cache"].clone()
    q = store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"][:0], d["cache"], d["slots"], q_pe=d["q_pe"])
    assert not q.any() and torch.equal(before, d["cache"])
    for int8 in (False, True):
        q, cache, cu, lens, table = make(cuda, 28, [2, 1], [90, 20], 16, int8, 64)
        out, lse = mla_chunk_attention_paged(q, cache[:0], cu, lens, table, SCALE, return_lse=True)
        assert not out.any() and bool(torch.isneginf(lse).all())


@pytest.mark.parametrize("vocab", [1023, 1024, 1025, 2049, 65537, 70001])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "lookup"])
def test_vocabularies_at_the_ends_of_chunks(cuda, vocab, probs):
    a = drafts.make(cuda, vocab, [3, 0, 2, 1], vocab, probs, True)
    log_case("verify_drafts vocabulary", vocab, probs)
    drafts.check(a, 3)
    for s in (0.0, 1.0):
        a[5].fill_(s)
        drafts.check(a, 3)


@pytest.mark.parametrize("vocab", [900, 20011, 70001])
def test_nothing_left_over_many_chunks(cuda, vocab):
    """A rejected draft where the draft model's probabilities cover the
    target's: the token comes from the target itself."""
    a = drafts.make(cuda, vocab, [1, 2, 0], vocab, True, False)
    a[0][:1] *= 0.5
    a[2][0] = 2 * a[0][0]
    a[4].fill_(0.75)
    log_case("verify_drafts nothing left", vocab)
    for s in (0.0, 0.3, 0.9, 1.0):
        a[5].fill_(s)
        tokens, accepted = drafts.check(a, 2)
        assert int(accepted[0]) == 0 and int(tokens[0, 0]) >= 0


def step_inputs(dev, seed, news, lens, heads, block, vocab):
    """A step over drafts: per request one accepted token and its drafts."""
    T, R = sum(news), len(news)
    q, cache, cu, lens_t, table = make(dev, seed, news, lens, heads, False, block)
    g = torch.Generator(device="cpu").manual_seed(seed)
    slots = [int(table[r, p // block]) * block + p % block
             for r, (n, length) in enumerate(zip(news, lens)) for p in range(length - n, length)]
    positions = [p for n, length in zip(news, lens) for p in range(length - n, length)]
    d = rope.make(dev, seed, T, heads, block, 1, torch.float32, max_pos=max(lens) + 1)
    d.update(cache=cache, slots=torch.tensor(slots, device=dev), positions=torch.tensor(positions, device=dev))
    d["q"] = q
    flat = cache.view(-1, 576)
    flat[d["slots"]] = math.nan    # not there before the append
    ids = torch.randint(0, vocab, (T - R,), generator=g, dtype=torch.int32)
    return d, cu, lens_t, table, [ids.to(dev), cu, torch.rand(T - R, generator=g).to(dev),
                                  torch.rand(R, generator=g, dtype=torch.float64).to(dev)]


def test_append_attend_verify(cuda):
    from titan_kv import store_rope
    from titan_mla import mla_chunk_attention_paged
    from titan_spec import verify_drafts
    news, lens, heads, block, vocab = [4, 1, 3, 4], [300, 65, 3, 1000], 16, 64, 5000
    d, cu, lens_t, table, (ids, cu_rows, u, s) = step_inputs(cuda, 31, news, lens, heads, block, vocab)
    log_case("append, attend, verify")
    store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], d["cache"], d["slots"], q_pe=d["q"][:, :, 512:],
               q_out=d["q"][:, :, 512:], norm_weight=d["norm_weight"], eps=rope.EPS)
    out, lse = mla_chunk_attention_paged(d["q"], d["cache"], cu, lens_t, table, SCALE, return_lse=True)
    check(out, lse, d["q"], d["cache"], cu, lens_t, table)
    g = torch.Generator(device="cpu").manual_seed(1)
    head = (torch.randn(heads * 512, vocab, generator=g) * 0.05).to(cuda)
    target = torch.softmax(out.flatten(1).float() @ head, dim=1)
    ids[::2] = target.argmax(dim=1)[:ids.numel()][::2].to(torch.int32)
    tokens, accepted = verify_drafts(target, ids, None, cu_rows, u, s, 3)
    want, count = O.verify(target, ids, None, cu_rows, u, s, 3)
    assert torch.equal(tokens.cpu(), want) and torch.equal(accepted.cpu(), count)
    # the next step's lengths: what was taken and the token drawn
    assert bool(((accepted >= 0) & (accepted.cpu() < torch.tensor(news)).to(cuda)).all())


def test_int8_append_and_attend(cuda):
    """The INT8 cache's writer and the same attention."""
    from titan_kv import store_int8
    from titan_mla import mla_chunk_attention_paged
    q, cache, cu, lens, table = make(cuda, 32, [3, 2], [100, 260], 16, True, 64)
    slots = [int(table[r, p // 64]) * 64 + p % 64 for r, (n, length) in enumerate(((3, 100), (2, 260)))
             for p in range(length - n, length)]
    x = torch.randn(5, 512, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda)
    log_case("int8 append, attend")
    store_int8(x, cache, torch.tensor(slots, dtype=torch.int64, device=cuda))
    out, lse = mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE, return_lse=True)
    check(out, lse, q, cache, cu, lens, table)


def test_a_step_in_a_graph(cuda):
    """The three of a step in one graph, replayed over new inputs."""
    from titan_kv import store_rope
    from titan_mla import mla_chunk_attention_paged
    from titan_spec import verify_drafts
    vocab = 3000
    d, cu, lens, table, (ids, cu_rows, u, s) = step_inputs(cuda, 33, [2, 4, 1], [400, 90, 2000], 16, 64, vocab)
    target = torch.softmax(torch.randn(7, vocab, generator=torch.Generator().manual_seed(2)) * 4, dim=1).to(cuda)

    def step(cache, q):
        store_rope(d["x"], d["k_pe"], d["positions"], d["cos_sin"], cache, d["slots"], q_pe=d["q_pe"],
                   q_out=q[:, :, 512:], norm_weight=d["norm_weight"])
        return (mla_chunk_attention_paged(q, cache, cu, lens, table, SCALE),
                *verify_drafts(target, ids, None, cu_rows, u, s, 3))

    step(d["cache"], d["q"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(d["cache"], d["q"])
    for k in range(4):
        d["x"].copy_(torch.roll(d["x"], 1, 0))
        d["q_pe"].copy_(torch.roll(d["q_pe"], 1, 0))
        target.copy_(torch.roll(target, 3, 1))
        u.copy_(torch.rand_like(u))
        log_case("step replay", k)
        cache, q = d["cache"].clone(), d["q"].clone()
        graph.replay()
        torch.cuda.synchronize()
        want = step(cache, q)
        # (as bits: unused rows hold NaN)
        assert torch.equal(cache.view(torch.int16), d["cache"].view(torch.int16)) and torch.equal(q, d["q"])
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_graphs_at_once(cuda):
    """Two captured calls, each with its own workspace, on two streams."""
    from titan_mla import mla_chunk_attention_paged
    a = make(cuda, 34, [4] * 5, [900, 2000, 77, 4, 1500], 16, False, 64)
    b = make(cuda, 35, [1] * 7, [300 + 411 * i for i in range(7)], 16, True, 64)
    want = [mla_chunk_attention_paged(*x, SCALE) for x in (a, b)]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(mla_chunk_attention_paged(*x, SCALE))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        log_case("two graphs", k)
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(outs, want))
