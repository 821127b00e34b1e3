"""Attention over a paged 8-bit cache against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import attention as oat
from tests.attention_helpers import Batch, f64, random_cache, sequence_values, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gw():
    import gewell_b200
    return gewell_b200


def queries(rows, heads, dim, seed, std=1.0):
    return (torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(seed)) * std).bfloat16().cuda()


def assert_rows(got, q, batch, cache, scale, window, rows_of=None, what=""):
    """Every row of `rows_of` (default: all sequences' rows) against the oracle.

    With A = sum p |v|: the output's rounding is 2^-8 |o|.  A probability in two E4M3 parts is off by 2^-4 * 2^-4 = 2^-8 of it, and
    2^-11 for the half-precision value they are cut from; below 2^-17 of the largest of 32 it is lost, 32 * 2^-17 = 2^-12 of that one.
    A query element in two parts is exact down to 2^-13 of the loudest of its 32, and off by half a step of 2^-13 of it, 2^-14 at most
    (2^-18 where its second part is scaled on its own), below; the score is then off by e = 2^-14 * |scale| * max |q| * sum |k_d| at most, which
    changes a probability by 2 e (numerator and sum).  FP32 sums of a few thousand terms stay below 2^-12 of A."""
    for s, (n, length) in enumerate(batch.sequences):
        if n == 0:
            continue
        k, v = (sequence_values(batch, c, s) for c in cache)
        low = int(batch.row_offsets[s])
        picked = range(n) if rows_of is None else sorted({i % n for i in rows_of})
        for i in picked:
            position = length - n + i
            exact, size = oat.attention(f64(q[low + i:low + i + 1]), k, v, scale, position, window)
            begin = max(0, position - window + 1) if window else 0
            seen = k[:, begin:position + 1]
            loudest = float(q[low + i].abs().max())
            e = 2.0 ** -14 * abs(scale) * loudest * (np.abs(seen).sum(axis=2).max() if position >= 0 else 0.0)
            bound = 2.0 ** -8 * np.abs(exact) + (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -12 + 2.0 ** -12 + 2 * e) * size + 1e-30
            error = np.abs(f64(got[low + i:low + i + 1]) - exact)
            assert (error <= bound).all(), f"{what} sequence {s} row {i}: {float((error / bound).max())} of the bound"


def check(gw, sequences, heads, kv_heads, dim, page, window=0, seed=0, scale=None, std=1.5, rows_of=None, extra_rows=0, spread=2.0):
    batch = Batch(sequences, page, seed, extra_rows=extra_rows)
    host = random_cache(batch, kv_heads, dim, seed + 1, spread=spread)
    q = queries(batch.rows, heads, dim, seed + 2, std)
    scale = dim ** -0.5 if scale is None else scale
    y = torch.full(q.shape, 7.0, dtype=torch.bfloat16).cuda()
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, scale, window=window, y=y)
    torch.cuda.synchronize()
    assert gw.kernel_error() == 0
    assert (got[int(batch.row_offsets[-1]):] == 7.0).all()
    assert_rows(got, q, batch, host, scale, window, rows_of, f"{heads}/{kv_heads} x {dim}, page {page}, window {window}:")


LAYOUTS = [(16, 8, 256), (16, 2, 512), (8, 2, 128), (6, 2, 128), (7, 7, 256), (16, 1, 128), (2, 2, 512)]


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("page", [16, 128])
def test_decode(gw, heads, kv_heads, dim, page):
    check(gw, [(1, 1), (1, 2), (1, 127), (1, 128), (1, 129), (0, 50), (1, 700), (1, 31)], heads, kv_heads, dim, page, seed=page)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [1, 5, 128, 200])
def test_decode_window(gw, page, window):
    check(gw, [(1, 1), (1, 300), (1, 128), (1, 133), (1, 900)], 8, 4, 256, page, window=window, seed=window)


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
def test_drafts(gw, heads, kv_heads, dim):
    check(gw, [(3, 3), (5, 700), (2, 130), (4, 128), (1, 64), (0, 0), (5, 257)], heads, kv_heads, dim, 32, seed=5, extra_rows=3)


@pytest.mark.parametrize("heads,kv_heads,dim", LAYOUTS)
@pytest.mark.parametrize("window", [0, 100])
def test_prompt(gw, heads, kv_heads, dim, window):
    check(gw, [(200, 200), (130, 517), (64, 64), (1, 90), (77, 141)], heads, kv_heads, dim, 64, window=window, seed=6,
          rows_of=[0, 1, 40, 63, 64, 100, 129, 199])


def test_many_query_heads_of_one_cache_head(gw):
    check(gw, [(1, 200), (3, 150)], 64, 1, 128, 16, seed=8)
    check(gw, [(1, 200), (40, 150)], 33, 1, 256, 16, seed=9, rows_of=[0, 17, 39])


def test_one_long_sequence(gw):
    check(gw, [(1, 20011)], 4, 2, 256, 64, seed=10)
    check(gw, [(1, 9999)], 16, 2, 512, 128, seed=11)
    check(gw, [(2, 5000), (1, 3)], 8, 8, 128, 16, seed=12)


@pytest.mark.parametrize("std,scale", [(40.0, 1.0), (1e-3, 1.0), (3.0, -0.3), (1.0, 0.0), (300.0, 0.5)])
def test_sharp_and_flat_scores(gw, std, scale):
    check(gw, [(1, 600), (3, 333), (70, 400)], 8, 2, 128, 32, seed=13, std=std, scale=scale, rows_of=[0, 1, 2, 69])


def test_pages_of_very_different_loudness(gw):
    check(gw, [(1, 700), (5, 256), (80, 300)], 4, 2, 256, 16, seed=14, spread=10.0, scale=1e-3, rows_of=[0, 4, 79])


def test_one_loud_token_among_many_quiet_ones(gw):
    """A token that takes half of the sum and thousands that share the other half: their probabilities lie 2^-13 and less below
    the largest, and their values point the other way."""
    dim, tokens, page = 128, 12000, 64
    batch = Batch([(1, tokens)], page, 15)
    (k, ks), (v, vs) = random_cache(batch, 1, dim, 16, garbage=False)
    ks[:], vs[:] = 1.0, 1.0
    values = oat.e4m3_values()
    one = int(np.flatnonzero(values == 1.0)[0])
    minus = int(np.flatnonzero(values == -1.0)[0])
    k[:], v[:] = 0, minus
    for place in (0, 5000, tokens - 1):
        kk, vv = k.copy(), v.copy()
        kk[batch.table[0, place // page], 0, place % page] = one
        vv[batch.table[0, place // page], 0, place % page] = one
        q = torch.full((1, 2, dim), 1.0, dtype=torch.bfloat16).cuda()
        scale = np.log(tokens) / dim
        got = gw.paged_attention(to_device(gw, [(kk, ks), (vv, vs)]), batch.device(gw), q, float(scale))
        assert_rows(got, q, batch, [(kk, ks), (vv, vs)], float(np.float32(scale)), 0)


def test_scores_that_rise_along_the_sequence(gw):
    """Every tile of tokens louder than all before it, by far more than one power of two, and the other way round."""
    dim, tokens, page = 256, 1500, 32
    batch = Batch([(1, tokens), (150, tokens)], page, 17)
    for sign in (1.0, -1.0):
        (k, ks), (v, vs) = random_cache(batch, 2, dim, 18, garbage=False, spread=0.0)
        ones = int(np.flatnonzero(oat.e4m3_values() == 1.0)[0])
        k[:] = ones
        for s in range(2):
            for page_at, page_number in enumerate(batch.table[s, :-(-tokens // page)]):
                ks[page_number] = np.float32(sign * (page_at + 1) * 0.02) if sign > 0 else np.float32((50 - page_at) * 0.02)
        q = queries(batch.rows, 4, dim, 19, 1.0) * 0 + 1.0
        got = gw.paged_attention(to_device(gw, [(k, ks), (v, vs)]), batch.device(gw), q, 1.0)
        assert_rows(got, q, batch, [(k, ks), (v, vs)], 1.0, 0, rows_of=[0, 149])


def test_rows_without_a_token_are_zero(gw):
    """Padding of a batch: rows of a sequence that has fewer tokens than rows."""
    batch = Batch([(3, 1), (2, 0), (1, 20), (4, -5)], 16, 20)
    host = random_cache(batch, 2, 128, 21)
    q = queries(batch.rows, 4, 128, 22)
    for std in (1.0,):
        got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 0.1, y=torch.full(q.shape, 3.0, dtype=torch.bfloat16).cuda())
        assert gw.kernel_error() == 0
        assert (got[:2] == 0).all() and (got[3:5] == 0).all() and (got[6:] == 0).all()
        rest = Batch([(3, 1), (2, 0), (1, 20), (4, -5)], 16, 20)
        rest.sequences = [(0, 0), (0, 0), (1, 20), (0, 0)]
        assert_rows(got, q, rest, host, 0.1, 0)
        k, v = (sequence_values(batch, c, 0) for c in host)
        exact, size = oat.attention(f64(q[2:3]), k, v, 0.1, 0)
        assert (np.abs(f64(got[2:3]) - exact) <= 2.0 ** -7 * (np.abs(exact) + size)).all()


def test_strided_rows_and_the_same_inputs_twice(gw):
    """Queries and outputs inside wider rows; two runs give the same bits."""
    batch = Batch([(1, 1500), (90, 300), (5, 70)], 32, 23)
    host = random_cache(batch, 2, 256, 24)
    cache, held = to_device(gw, host), batch.device(gw)
    wide = torch.randn((batch.rows, 3, 8 * 256), generator=torch.Generator().manual_seed(25)).bfloat16().cuda()
    q = wide[:, 1].unflatten(1, (8, 256))
    out = torch.full((batch.rows, 2, 8 * 256), 5.0, dtype=torch.bfloat16).cuda()
    got = gw.paged_attention(cache, held, q, 0.06, y=out[:, 1].unflatten(1, (8, 256)))
    assert (out[:, 0] == 5.0).all()
    assert_rows(got, q, batch, host, 0.06, 0, rows_of=[0, 44, 89])
    again = gw.paged_attention(cache, held, q.contiguous(), 0.06)
    assert torch.equal(again, got)


@pytest.mark.parametrize("heads,kv_heads,dim,page,rows", [(32, 4, 512, 128, 1), (32, 16, 256, 64, 1), (32, 8, 128, 16, 3), (16, 2, 512, 64, 300)])
def test_many_passes_give_the_same_bits(gw, heads, kv_heads, dim, page, rows):
    """Long sequences that wait for memory, pass behind pass: what the warps of a block hand each other must not depend on who is late."""
    count = 12 if rows < 16 else 2
    batch = Batch([(rows, 9000 + 700 * s) for s in range(count)], page, 40)
    g = torch.Generator(device="cuda").manual_seed(41)
    shape = (batch.pages, kv_heads, page, dim)
    data = [torch.randn(shape, generator=g, device="cuda").clamp_(-4, 4).mul_(64).to(torch.float8_e4m3fn) for _ in range(2)]
    cache = gw.KvCache(*data, *(torch.full(shape[:2], 1 / 64, device="cuda") for _ in range(2)))
    held, q = batch.device(gw), queries(batch.rows, heads, dim, 42)
    first = gw.paged_attention(cache, held, q, dim ** -0.5)
    for _ in range(60):
        again = gw.paged_attention(cache, held, q, dim ** -0.5)
        assert torch.equal(again, first)
    assert gw.kernel_error() == 0
    host = [(d.view(torch.uint8).cpu().numpy(), np.full(shape[:2], 1 / 64, dtype=np.float32)) for d in data]
    assert_rows(first, q, batch, host, dim ** -0.5, 0, rows_of=[0])


def test_bad_pages_are_left_out(gw):
    """A page number outside the cache, and a context that reaches behind the page table: those tokens do not count, and it is reported."""
    batch = Batch([(1, 100), (20, 90)], 16, 26)
    host = random_cache(batch, 1, 128, 27, garbage=False)
    q = queries(batch.rows, 2, 128, 28)
    for bad in (-1, batch.pages, 2 ** 30):
        broken = Batch([(1, 100), (20, 90)], 16, 26)
        broken.table[0, 2] = bad
        got = gw.paged_attention(to_device(gw, host), broken.device(gw), q, 0.1)
        assert gw.kernel_error() >> 24 == 0xa1
        k, v = (np.delete(sequence_values(batch, c, 0), np.arange(32, 48), axis=1) for c in host)
        exact, size = oat.attention(f64(q[:1]), k, v, 0.1, 83)
        assert (np.abs(f64(got[:1]) - exact) <= 2.0 ** -7 * (np.abs(exact) + size)).all()
    short = batch.device(gw)
    short = gw.SequenceBatch(short.row_offsets, short.context_lengths, short.page_table[:, :5].contiguous(), batch.rows, batch.max_rows)
    got = gw.paged_attention(to_device(gw, host), short, q, 0.1)
    assert gw.kernel_error() >> 24 == 0xa1
    k, v = (sequence_values(batch, c, 0)[:, :80] for c in host)
    exact, size = oat.attention(f64(q[:1]), k, v, 0.1, 79)
    assert (np.abs(f64(got[:1]) - exact) <= 2.0 ** -7 * (np.abs(exact) + size)).all()


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 2, 128, 16), (16, 2, 512, 64), (8, 8, 256, 128)])
@pytest.mark.parametrize("sequences,window", [([(5, 90)], 0), ([(3, 400), (6, 33), (2, 2)], 20), ([(200, 300)], 0), ([(150, 700), (64, 64)], 100),
                                              ([(4, 9000)], 0)])
def test_nan_values_reach_the_queries_that_see_them_and_no_others(gw, heads, kv_heads, dim, page, sequences, window):
    """One or several elements of a token, among the step's own tokens and before them."""
    batch = Batch(sequences, page, 40)
    host = random_cache(batch, kv_heads, dim, 41)
    rng = np.random.default_rng(42)
    codes = host[1][0]
    for s, (n, length) in enumerate(sequences):
        for token in {length - 1, length - n // 2 - 1, max(0, length - n - 3), max(0, length - 2)}:
            at = codes[int(batch.table[s, token // page]), int(rng.integers(kv_heads)), token % page]
            at[rng.choice(dim, int(rng.choice([1, 3, 10])), replace=False)] = rng.choice([0x7f, 0xff])
    q = queries(batch.rows, heads, dim, 43)
    got = f64(gw.paged_attention(to_device(gw, host), batch.device(gw), q, dim ** -0.5, window=window))
    assert gw.kernel_error() == 0
    seen_any = False
    for s, (n, length) in enumerate(sequences):
        k, v = (sequence_values(batch, c, s) for c in host)
        low = int(batch.row_offsets[s])
        for i in sorted({0, n // 2 - 1, n // 2, n - 2, n - 1, n // 3} & set(range(n))):
            exact, size = oat.attention(f64(q[low + i:low + i + 1]), k, v, dim ** -0.5, length - n + i, window)
            nan = np.isnan(exact)
            seen_any |= bool(nan.any()) and not nan.all()
            assert (np.isnan(got[low + i:low + i + 1]) == nan).all(), f"sequence {s} row {i}"
            error = np.abs(got[low + i:low + i + 1] - exact)
            assert (error[~nan] <= (2.0 ** -7 * (np.abs(exact) + size))[~nan]).all()
    assert seen_any


def test_many_nan_values(gw):
    """More places than are kept: rows in front of the first of them are as they were, rows behind the last are NaN."""
    batch = Batch([(60, 200)], 16, 44)
    host = random_cache(batch, 1, 256, 45)
    for token in range(170, 180):
        host[1][0][int(batch.table[0, token // 16]), 0, token % 16] = 0x7f
    q = queries(60, 4, 256, 46)
    got = f64(gw.paged_attention(to_device(gw, host), batch.device(gw), q, 256 ** -0.5))
    assert gw.kernel_error() == 0
    assert not np.isnan(got[:30]).any() and np.isnan(got[30:]).all()


def test_more_work_than_can_be_counted_is_left_out(gw):
    """40 sequences of 2^30 tokens by their lengths (the table has a page each): 2^31 tiles and more over 8 heads."""
    batch = Batch([(1, 100)] * 40, 128, 29)
    host = random_cache(batch, 8, 128, 30)
    q = queries(40, 8, 128, 31)
    long = batch.device(gw)
    y = torch.full_like(q, 7.0)
    long.context_lengths.fill_(2 ** 30)
    gw.paged_attention(to_device(gw, host), long, q, 0.1, y=y)
    assert gw.kernel_error() == 0xa2ffffff and (y == 7.0).all()
    long.context_lengths.fill_(2 ** 30 + 1)
    gw.paged_attention(to_device(gw, host), long, q, 0.1, y=y)
    assert gw.kernel_error() >> 24 == 0xa2 and (y == 7.0).all()


def test_refusals_of_the_wrapper(gw):
    batch = Batch([(2, 40)], 16, 50)
    cache = to_device(gw, random_cache(batch, 2, 128, 51))
    held, q = batch.device(gw), queries(2, 4, 128, 52)
    strided = torch.zeros((2, 8, 128), dtype=torch.bfloat16).cuda()[:, ::2]
    for bad in (dict(window=-1), dict(window=(1 << 32) + 5), dict(scale=float("nan")), dict(query=q.float()), dict(query=q[:1]), dict(query=strided), dict(query=q.cpu()),
                dict(y=torch.empty((2, 4, 64), dtype=torch.bfloat16).cuda()), dict(y=q.cpu()), dict(query=queries(2, 3, 128, 1)),
                dict(query=queries(2, 4, 256, 1)), dict(scratch=torch.empty(16, dtype=torch.uint8).cuda()),
                dict(scratch=torch.empty(1 << 22, dtype=torch.int8).cuda())):
        with pytest.raises(gw.GewellInvalidArgument):
            gw.paged_attention(cache, held, **{**dict(query=q, scale=0.1), **bad})


def test_on_another_stream(gw):
    """Scratch that the call allocates is not handed out again while the other stream still uses it."""
    batch = Batch([(1, 4000)] * 4, 64, 53)
    host = random_cache(batch, 2, 256, 54)
    cache, held, q = to_device(gw, host), batch.device(gw), queries(4, 16, 256, 55)
    plain = gw.paged_attention(cache, held, q, 0.06)
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), torch.cuda.Stream().cuda_stream):
        results = []
        for _ in range(6):
            results.append(gw.paged_attention(cache, held, q, 0.06, stream=stream, y=torch.empty_like(q)))
            torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        assert all(torch.equal(r, plain) for r in results)


def test_captured_replayed_with_other_lengths_and_beside_another(gw):
    """One graph serves later steps: lengths and pages are read on the device.  Two graphs with scratch of their own run at once."""
    steps = [[(1, 40), (1, 700), (1, 3)], [(1, 41), (1, 1900), (1, 300)], [(1, 1), (1, 2), (0, 0)]]
    batches = [Batch(s, 32, 29) for s in steps]
    largest = max(b.pages for b in batches)
    entries = max(b.table.shape[1] for b in batches)
    q = queries(3, 8, 256, 30)
    hosts = []
    for b in batches:
        b.pages, wide = largest, np.full((3, entries), -1, dtype=np.int32)
        wide[:, :b.table.shape[1]] = b.table
        b.table = wide
        hosts.append(random_cache(b, 4, 256, 31))
    caches = [to_device(gw, hosts[0]) for _ in range(2)]
    held = [batches[0].device(gw) for _ in range(2)]
    outs = [torch.empty_like(q) for _ in range(2)]
    gw.paged_attention(caches[0], held[0], q, 0.1)
    torch.cuda.synchronize()
    graphs, streams = [torch.cuda.CUDAGraph() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            gw.paged_attention(caches[i], held[i], q, 0.1, y=outs[i])
    for step in (1, 2, 0, 1):
        for i in range(2):
            at = (step + i) % 3
            for name, source in (("k_data", hosts[at][0][0]), ("v_data", hosts[at][1][0]), ("k_scales", hosts[at][0][1]), ("v_scales", hosts[at][1][1])):
                getattr(caches[i], name).copy_(torch.from_numpy(np.ascontiguousarray(source)))
            held[i].row_offsets.copy_(torch.from_numpy(batches[at].row_offsets))
            held[i].context_lengths.copy_(torch.from_numpy(batches[at].lengths))
            held[i].page_table.copy_(torch.from_numpy(batches[at].table))
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert gw.kernel_error() == 0
        for i in range(2):
            at = (step + i) % 3
            assert_rows(outs[i], q, batches[at], hosts[at], 0.1, 0, what=f"step {step}")


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 4, 256), (8, 2, 512)])
def test_a_layer_from_its_projections_to_its_output(gw, heads, kv_heads, dim):
    """Q | K | V projection, append with norms and rotation, attention, output projection: three steps of two sequences, against
    the same in 64 bits over what the cache holds."""
    from gewell_b200 import _lib
    hidden, page = 512, 16
    g = torch.Generator().manual_seed(32)
    w = (torch.randn(((heads + 2 * kv_heads) * dim, hidden), generator=g) * 0.05).bfloat16().cuda()
    wo = (torch.randn((hidden, heads * dim), generator=g) * 0.02).bfloat16().cuda()
    qw, kw = ((1 + 0.25 * torch.randn(dim, generator=g)).bfloat16().cuda() for _ in range(2))
    f = torch.tensor([1e4 ** (-i / (dim // 2)) for i in range(dim // 2)], dtype=torch.float32).cuda()
    parts = w.split([heads * dim, kv_heads * dim, kv_heads * dim])
    query, key, value = (gw.make_projection(p, hidden, p.shape[0]) for p in parts)
    projector = gw.QkvProjector(hidden, heads * dim, kv_heads * dim, 256, _lib.POLICY_ALWAYS)
    table = torch.randperm(12, generator=g)[:10].reshape(2, 5).int().cuda()
    cache = gw.KvCache(*(torch.full((12, kv_heads, page, dim), 127, dtype=torch.uint8).cuda() for _ in range(2)),
                       *(torch.full((12, kv_heads), float("nan")).cuda() for _ in range(2)))
    lengths = [0, 0]
    for news in ([37, 20], [1, 1], [3, 0]):
        lengths = [a + b for a, b in zip(lengths, news)]
        rows = sum(news)
        offsets = torch.tensor([0, news[0], rows], dtype=torch.int32).cuda()
        batch = gw.SequenceBatch(offsets, torch.tensor(lengths, dtype=torch.int32).cuda(), table, rows, max(news))
        x = torch.randn((rows, hidden), generator=g).bfloat16().cuda()
        projector.prepare(rows)
        q, k, v, joined_one = projector.run(query, key, value, x, _lib.PHASE_PREFILL)
        assert joined_one
        q, k, v = q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))
        turned = gw.kv_cache_append(cache, batch, k, v, key_weight=kw, frequencies=f, query=q, query_weight=qw)
        seen = gw.paged_attention(cache, batch, turned, dim ** -0.5)
        plan = gw.Bf16Plan(rows, heads * dim, hidden)
        out = torch.empty((rows, hidden), dtype=torch.bfloat16).cuda()
        plan.run(seen.flatten(1), wo, out, torch.empty(max(256, plan.scratch_bytes()), dtype=torch.uint8).cuda())
        torch.cuda.synchronize()
        assert gw.kernel_error() == 0
        at = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, news)])
        exact_q = oat.head_norm_rotary(f64(q), f64(qw), True, at, f.cpu().numpy())
        assert (np.abs(f64(turned) - exact_q) <= 2.0 ** -8 * np.abs(exact_q) + 2.0 ** -19 * np.abs(exact_q).max(axis=-1, keepdims=True)).all()
        held = Batch([(m, n) for n, m in zip(lengths, news)], page, 0)
        held.table = table.cpu().numpy()
        host = [(cache.k_data.cpu().numpy(), cache.k_scales.cpu().numpy()), (cache.v_data.cpu().numpy(), cache.v_scales.cpu().numpy())]
        assert_rows(seen, turned, held, host, dim ** -0.5, 0)
        exact = f64(seen.flatten(1)) @ f64(wo).T
        assert (np.abs(f64(out) - exact) <= 2.0 ** -8 * np.abs(exact) + 2.0 ** -18 * (np.abs(f64(seen.flatten(1))) @ np.abs(f64(wo)).T)).all()


def test_pages_behind_four_gigabytes(gw):
    """The same step on the last pages of a large cache and on a small one gives the same codes, scales and results."""
    page, dim, kv_heads, rows, sequences = 128, 512, 4, 70, [(70, 70), (1, 1)]
    many = (1 << 32) // (page * dim * kv_heads) + 3
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    g = torch.Generator().manual_seed(60)
    q, k, v = (torch.randn((rows + 1, h, dim), generator=g).bfloat16().cuda() for h in (8, kv_heads, kv_heads))
    results = []
    for pages, table in ((2, [[0], [1]]), (many, [[many - 1], [many - 3]])):
        cache = gw.KvCache(*(torch.empty((pages, kv_heads, page, dim), dtype=torch.uint8, device="cuda") for _ in range(2)),
                           *(torch.empty((pages, kv_heads), device="cuda") for _ in range(2)))
        batch = gw.SequenceBatch(torch.tensor([0, rows, rows + 1], dtype=torch.int32).cuda(), torch.tensor([n for _, n in sequences], dtype=torch.int32).cuda(),
                                 torch.tensor(table, dtype=torch.int32).cuda(), rows + 1, rows)
        gw.kv_cache_append(cache, batch, k, v)
        out = gw.paged_attention(cache, batch, q, dim ** -0.5)
        at = [t[0] for t in table]
        results.append([out, cache.k_scales[at], cache.v_scales[at], cache.k_data[at[0], :, :rows].clone(), cache.v_data[at[0], :, :rows].clone(),
                        cache.k_data[at[1], :, 0].clone(), cache.v_data[at[1], :, 0].clone()])
    assert gw.kernel_error() == 0
    assert all(torch.equal(a, b) for a, b in zip(*results)) and not torch.isnan(results[0][0]).any()
