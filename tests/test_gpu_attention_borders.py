"""Attention over a paged 8-bit cache where it is easily wrong, against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import attention as oat
from tests.attention_helpers import VALUES, Batch, f64, random_cache, sequence_values, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gw():
    import gewell_b200
    return gewell_b200


def queries(rows, heads, dim, seed, std=1.0):
    return (torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(seed)) * std).bfloat16().cuda()


def bound_of(q, k, v_codes, v_scales, scale, begin, exact, size):
    """What the arithmetic of one row may be off by: q [heads, D], k [kv heads, tokens, D] and the codes [kv heads, tokens, D] and
    scales [kv heads, tokens] of the values that it sees, the first of them token `begin`; exact, size = sum p |v| [heads, D].

    A query element: x = hi + lo / 16 in blocks of 32 that are scaled to a loudest of 2^7 to 2^8.  With eight significant bits it is exact
    from 2^-6 on; below, half a step of lo is 2^-10 / 16 = 2^-14, 2^-21 of the loudest.  A score adds D / 16 products of 32 terms in
    FP32, each sum off by 2^-22 of sum |q k| at most and each of its terms by 2^-24 of the largest; its scaling (three factors, one fma)
    by 2^-22 of it.  All that together is e, and a probability over the sum of them changes by exp(2 e) - 1.
    A probability in two parts: half a step of each is 2^-4 of it, 2^-8 together; 2^-11 for the half-precision value that is cut; below
    the normal codes half a step of lo, 2^-10, with the largest p * scale of the 32 tokens of a block at 2^7 or more: 2^-17 of that.
    The sums: tokens / 16 products of 32 terms as above, tokens additions of 2^-24, 2^-21 for exp2 and the reciprocal.
    The result: half a step of BF16, 2^-8."""
    heads, group, tokens, dim = q.shape[0], q.shape[0] // k.shape[0], k.shape[1], q.shape[1]
    out = np.zeros(exact.shape)
    block = (begin + np.arange(tokens)) // 32 - begin // 32
    for h in range(heads):
        keys, codes, scales = k[h // group], np.abs(v_codes[h // group]), v_scales[h // group]
        terms = np.abs(keys * q[h])
        scores = keys @ q[h] * scale
        e = 2.0 ** -21 * abs(scale) * np.abs(q[h]).max() * np.abs(keys).sum(axis=1).max()
        e += dim / 16 * abs(scale) * (2.0 ** -22 * terms.sum(axis=1).max() + 32 * 2.0 ** -24 * terms.max())
        e += 2.0 ** -22 * np.abs(scores).max()
        p = np.exp(scores - scores.max())
        p = p / p.sum() * scales
        loudest = np.zeros(block[-1] + 1)
        np.maximum.at(loudest, block, p)
        lost = 2.0 ** -17 * (loudest[block] @ codes)
        part = 2.0 ** -8 + 2.0 ** -11 + np.expm1(2 * e) + tokens / 16 * 32 * 2.0 ** -24 + tokens * 2.0 ** -24 + 2.0 ** -21
        out[h] = (2.0 ** -8 * np.abs(exact[h]) + part * size[h] + lost) * (1 + 2.0 ** -8)
    return out


def assert_rows(got, q, batch, cache, scale, window=0, rows_of=None, share=None, what=""):
    """Rows (default: all) against the definition; `share`: what the bound may be of sum p |v|, at most, in the median."""
    got, shares = f64(got), []
    for s, (n, length) in enumerate(batch.sequences):
        if n == 0:
            continue
        k = sequence_values(batch, cache[0], s)
        pages = batch.table[s, :-(-length // batch.page_tokens)]
        codes = VALUES[cache[1][0][pages]].transpose(1, 0, 2, 3).reshape(k.shape[0], -1, k.shape[2])[:, :length]
        scales = np.repeat(cache[1][1][pages].astype(np.float64).T, batch.page_tokens, axis=1)[:, :length]
        v = codes * scales[..., None]
        for i in range(n) if rows_of is None else sorted({r % n for r in rows_of}):
            row, position = int(batch.row_offsets[s]) + i, length - n + i
            exact, size = oat.attention(f64(q[row:row + 1]), k, v, scale, position, window)
            seen = slice(max(0, position - window + 1) if window else 0, position + 1)
            bound = bound_of(f64(q[row]), k[:, seen], codes[:, seen], scales[:, seen], scale, seen.start, exact[0], size[0])
            error = np.abs(got[row] - exact[0])
            assert (error <= bound).all(), f"{what} sequence {s} row {i}: {float(np.nanmax(error / bound))} of the bound"
            shares.append(np.median(bound / size[0]))
    assert share is None or np.median(shares) <= share, np.median(shares)


@pytest.mark.parametrize("level", [80.0, 100.0, 300.0, 1000.0])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (4, 2, 256, 64), (8, 2, 512, 128)])
@pytest.mark.parametrize("sequences,window", [([(5, 130)], 0), ([(16, 400), (1, 257), (3, 129)], 0), ([(40, 300), (5, 131)], 100), ([(300, 700)], 90),
                                              ([(140, 140)], 0)])
def test_scores_far_below_zero_in_pieces_that_some_rows_do_not_see(gw, level, heads, kv_heads, dim, page, sequences, window):
    """All logits of all rows near -level.  There are fewer units of work than blocks, so every token tile of an item is a piece of its
    own, and at a causal or window border rows of the item see nothing of it."""
    batch = Batch(sequences, page, 61)
    host = random_cache(batch, kv_heads, dim, 62, spread=0.0)
    codes, scales = host[0]
    one = int(np.flatnonzero(VALUES == 1.0 / float(np.nanmax(scales)))[0])
    codes[..., :32] = one
    q = queries(batch.rows, heads, dim, 63, 0.1)
    q[..., :32] = -level / 32
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 1.0, window=window)
    assert gw.kernel_error() == 0
    assert_rows(got, q, batch, host, 1.0, window, rows_of=[0, 1, 2, 3, 4, 15, 39, 63, 64, 120, 127, 128, 139, 200, 299], share=0.05)


@pytest.mark.parametrize("std,scale", [(12.0, -1.0), (40.0, 1.0), (300.0, 0.5)])
def test_sharp_scores_within_what_the_arithmetic_allows(gw, std, scale):
    """The bound stays well below the values: any finite output would not pass."""
    batch = Batch([(1, 600), (3, 333), (70, 400)], 32, 64)
    host = random_cache(batch, 2, 128, 65, spread=0.0)
    q = queries(batch.rows, 8, 128, 66, std)
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, scale)
    assert gw.kernel_error() == 0
    assert_rows(got, q, batch, host, scale, rows_of=[0, 1, 2, 35, 69], share=0.25)


def test_a_piece_without_pages_takes_no_weight_from_scores_far_below_zero(gw):
    """A whole tile whose page is missing, as a piece of its own."""
    batch = Batch([(1, 300)], 128, 64)
    host = random_cache(batch, 1, 128, 65, garbage=False, spread=0.0)
    host[0][0][..., :32] = int(np.flatnonzero(VALUES == 1.0 / float(host[0][1].max()))[0])
    q = queries(1, 4, 128, 66, 0.1)
    q[..., :32] = -300.0 / 32
    k, v = (np.delete(sequence_values(batch, c, 0), np.arange(128, 256), axis=1) for c in host)
    batch.table[0, 1] = -1
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 1.0)
    assert gw.kernel_error() >> 24 == 0xa1
    exact, size = oat.attention(f64(q), k, v, 1.0, 171)
    # of logits near 300: 2^-21 * 9.4 * 132 + 8 * (2^-22 * 300 + 2^-19 * 9.4) + 2^-22 * 300 stays below 2^-9, twice in the exponent
    assert (np.abs(f64(got) - exact) <= 2.0 ** -8 * np.abs(exact) + (2.0 ** -8 + 2.0 ** -8 + 2.0 ** -10) * size).all()


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 256), (4, 4, 128), (2, 1, 512), (16, 2, 256)])
@pytest.mark.parametrize("window", [0, 5, 40, 64, 100])
@pytest.mark.parametrize("tokens", [(100,), (139,), (140, 141), (90, 91, 92, 150), tuple(range(135, 145)), (60, 145, 199)])
def test_tokens_of_nan_reach_the_rows_that_see_them(gw, heads, kv_heads, dim, window, tokens):
    """Whole tokens of NaN, more places than are kept for an item: at both ends of windows, and in windows shorter than a tile's rows."""
    sequences = [(60, 200)]
    batch = Batch(sequences, 16, 67)
    host = random_cache(batch, kv_heads, dim, 68)
    for token in tokens:
        host[1][0][int(batch.table[0, token // 16]), :, token % 16] = 0x7f
    q = queries(60, heads, dim, 69)
    got = f64(gw.paged_attention(to_device(gw, host), batch.device(gw), q, dim ** -0.5, window=window))
    assert gw.kernel_error() == 0
    k, v = (sequence_values(batch, c, 0) for c in host)
    for i in range(60):
        position = 140 + i
        sees = any(t <= position and (window == 0 or position - t < window) for t in tokens)
        assert np.isnan(got[i]).all() if sees else not np.isnan(got[i]).any(), f"row {i}"
        if not sees and i % 7 == 0:
            exact, size = oat.attention(f64(q[i:i + 1]), k, v, dim ** -0.5, position, window)
            assert (np.abs(got[i] - exact[0]) <= 2.0 ** -7 * (np.abs(exact[0]) + size[0])).all()


def test_a_view_of_a_wider_page_table(gw):
    """Positions behind a view's last column are behind the table, whatever the wider table holds there."""
    batch = Batch([(1, 100), (20, 90)], 16, 73)
    host = random_cache(batch, 1, 128, 74, garbage=False)
    q = queries(batch.rows, 2, 128, 75)
    columns, sequences = batch.table.shape[1], len(batch.sequences)
    wide = torch.zeros((sequences, columns + 7), dtype=torch.int32).cuda()
    whole = batch.device(gw)
    wide[:, 4:4 + columns] = whole.page_table
    offsets, lengths = whole.row_offsets, whole.context_lengths
    view = gw.SequenceBatch(offsets, lengths, wide[:, 4:4 + columns], batch.rows, batch.max_rows)
    assert torch.equal(gw.paged_attention(to_device(gw, host), view, q, 0.1), gw.paged_attention(to_device(gw, host), whole, q, 0.1))
    assert gw.kernel_error() == 0
    short = gw.SequenceBatch(offsets, lengths, whole.page_table[:, :5].contiguous(), batch.rows, batch.max_rows)
    want = gw.paged_attention(to_device(gw, host), short, q, 0.1)
    assert gw.kernel_error() >> 24 == 0xa1
    short = gw.SequenceBatch(offsets, lengths, wide[:, 4:9], batch.rows, batch.max_rows)
    assert torch.equal(gw.paged_attention(to_device(gw, host), short, q, 0.1), want)
    assert gw.kernel_error() >> 24 == 0xa1
    # and the append writes to none of the pages behind the view
    x = torch.ones((batch.rows, 1, 128), dtype=torch.bfloat16).cuda()
    cache = to_device(gw, host)
    before = cache.k_data.clone()
    gw.kv_cache_append(cache, short, x, x)
    assert gw.kernel_error() >> 24 == 0xa1
    changed = (cache.k_data != before).flatten(1).any(dim=1).cpu().numpy()
    assert not changed[batch.table[0, 5:7]].any() and not changed[batch.table[1, 5]]
    assert changed[batch.table[1, 4]]                                # tokens 70 .. 79


@pytest.mark.parametrize("kind", ["attention", "norm", "append"])
@pytest.mark.parametrize("number", [False, True])
def test_results_on_another_stream_are_not_in_memory_that_is_still_read(gw, kind, number):
    """A tensor that the current stream has yet to read, freed, is not where a call on another stream puts its results or scratch; and
    results of such a call that the current stream has yet to read are not where the next call on that stream puts its own."""
    batch = Batch([(1, 300)] * 5, 32, 76)
    cache = to_device(gw, random_cache(batch, 2, 256, 77, garbage=False))
    held, q = batch.device(gw), queries(5, 8, 256, 78)
    k = queries(5, 2, 256, 79)
    positions = torch.arange(5, dtype=torch.int32).cuda()

    def call(stream=None):
        if kind == "attention":
            return gw.paged_attention(cache, held, q, 0.06, stream=stream)
        if kind == "norm":
            return gw.qk_norm_rotary(q, None, None, None, positions, None, stream=stream)[0]
        return gw.kv_cache_append(cache, held, k, k, query=q, stream=stream)
    plain = call()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    given = other.cuda_stream if number else other
    # the caching allocator hands a block of the same size out again; several, as others may lie free
    sizes = [q.numel() * 2] * 50
    if kind == "attention":
        sizes += [gw.lib.gw_paged_attention_scratch_bytes(cache._ref, held._ref, 8)] * 4
    taken = [torch.full((n,), 9, dtype=torch.uint8, device="cuda") for n in sizes]
    read = [torch.zeros_like(t) for t in taken]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    for t, r in zip(taken, read):
        r.copy_(t)
    del taken, t
    got = call(given)
    other.synchronize()
    assert torch.equal(got, plain)
    torch.cuda.synchronize()
    assert all((r == 9).all() for r in read)
    kept = torch.zeros_like(got)
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    kept.copy_(got)
    del got                                             # the current stream has yet to read it
    with torch.cuda.stream(other):
        for _ in range(4):
            torch.full((q.numel(),), 3.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    assert torch.equal(kept, plain)


@pytest.mark.parametrize("number", [0, 1])
def test_the_default_stream_by_its_number(gw, number):
    batch = Batch([(1, 300)] * 3, 32, 83)
    cache = to_device(gw, random_cache(batch, 2, 128, 84, garbage=False))
    held, q = batch.device(gw), queries(3, 8, 128, 85)
    plain = gw.paged_attention(cache, held, q, 0.06)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        got = gw.paged_attention(cache, held, q, 0.06, stream=number)
    torch.cuda.synchronize()
    assert torch.equal(got, plain) and torch.equal(gw.paged_attention(cache, held, q, 0.06, stream=number), plain)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), -2.0 ** -7])
@pytest.mark.parametrize("window", [0, 30])
def test_value_scales_that_are_no_numbers(gw, bad, window):
    """The scale of a page that is NaN, infinite or negative makes the rows NaN that see any token of the page, and no others: it is no
    missing page.  The others need not have the bits that they have without it: a NaN asks for another reference for all rows of
    its tile, exp2(score - reference) is then another number, and its rounding to two parts falls elsewhere (2^-8 of it, in the bound)."""
    batch = Batch([(60, 200), (1, 50)], 16, 70)
    host = random_cache(batch, 2, 128, 71)
    clean = [tuple(a.copy() for a in part) for part in host]
    host[1][1][int(batch.table[0, 9]), 1] = bad                    # tokens 144 .. 159 of the first sequence, second head
    q = queries(batch.rows, 4, 128, 72)
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 0.1, window=window)
    assert gw.kernel_error() == 0
    sees = [140 + i >= 144 and (window == 0 or 140 + i - 159 < window) for i in range(60)]
    assert 0 < sum(sees) and torch.isnan(got[:60][sees][:, 2:]).all()
    rest = [i for i in range(60) if not sees[i]]
    assert_rows(got, q, batch, clean, 0.1, window, rows_of=rest)
    assert not torch.isnan(got[:, :2]).any()
    other = got.clone()
    other[:60, 2:][sees] = gw.paged_attention(to_device(gw, clean), batch.device(gw), q, 0.1, window=window)[:60, 2:][sees]
    assert_rows(other, q, batch, clean, 0.1, window, rows_of=range(0, 60, 7))


def test_reports_of_two_operators_are_both_read(gw):
    batch = Batch([(1, 20), (1, 40)], 16, 80)
    host = random_cache(batch, 1, 128, 81, garbage=False)
    broken = Batch([(1, 20), (1, 40)], 16, 80)
    broken.table[0, 1] = -1
    x = queries(2, 1, 128, 82)
    gw.kv_cache_append(to_device(gw, host), broken.device(gw), x, x)
    broken = Batch([(1, 20), (1, 40)], 16, 80)
    broken.table[1, 1] = -1
    gw.paged_attention(to_device(gw, host), broken.device(gw), x, 0.1)
    assert sorted([gw.kernel_error(), gw.kernel_error()]) == [0xa1000000, 0xa1000001] and gw.kernel_error() == 0


def test_reading_the_error_word_loads_no_kernels(tmp_path):
    """A process that has run none of these operators, perhaps with all memory taken, reads the word without their modules: what the first
    read takes is the word's own allocation, one granule of 2 MiB."""
    import subprocess
    import sys
    from pathlib import Path
    code = ("import torch, gewell_b200 as gw; torch.zeros(1).cuda(); torch.cuda.synchronize(); before = torch.cuda.mem_get_info()[0]; "
            "assert gw.kernel_error() == 0; print(before - torch.cuda.mem_get_info()[0])")
    done = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    assert int(done.stdout.split()[-1]) <= 2 << 20


def test_a_replayed_graph_reports(gw):
    batch = Batch([(1, 40)], 16, 86)
    cache, held, q = to_device(gw, random_cache(batch, 1, 128, 87, garbage=False)), batch.device(gw), queries(1, 2, 128, 88)
    gw.paged_attention(cache, held, q, 0.1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw.kv_cache_append(cache, held, q[:, :1], q[:, :1])
        gw.paged_attention(cache, held, q, 0.1)
    graph.replay()
    assert gw.kernel_error() == 0
    held.page_table.fill_(-1)
    graph.replay()
    assert gw.kernel_error() == 0xa1000000 and gw.kernel_error() == 0xa1000000 and gw.kernel_error() == 0


@pytest.mark.parametrize("window", [0, 70])
def test_more_sequences_than_threads_of_a_block(gw, window):
    """The search for a block's first unit goes over the sequences in several rounds."""
    rng = np.random.default_rng(89)
    lengths = rng.integers(1, 300, 1500)
    sequences = [(int(min(rng.integers(0, 3), n)), int(n)) for n in lengths]
    batch = Batch(sequences, 64, 90)
    host = random_cache(batch, 1, 128, 91, spread=1.0)
    q = queries(batch.rows, 4, 128, 92)
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 0.1, window=window)
    assert gw.kernel_error() == 0
    for s in range(1500):
        if s % 9 and s not in (639, 640, 641, 1279, 1280, 1281, 1499):
            batch.sequences[s] = (0, 0)                                # not looked at
    assert_rows(got, q, batch, host, 0.1, window)


@pytest.mark.parametrize("dim", [128, 256, 512])
@pytest.mark.parametrize("group,rows", [(1, 1), (16, 1), (2, 16), (32, 1), (8, 4), (64, 1), (13, 3), (64, 5), (1, 200)])
@pytest.mark.parametrize("window", [0, 60])
def test_every_width_of_a_block_with_every_head(gw, dim, group, rows, window):
    """Scales that are no powers of two, too."""
    batch = Batch([(rows, max(rows, 300)), (1, 5), (rows, max(rows, 129))], 32, 93)
    host = random_cache(batch, 2, dim, 94, spread=1.0)
    for part in host:
        part[1][:] *= np.random.default_rng(95).uniform(0.5, 2.0, part[1].shape).astype(np.float32)
    q = queries(batch.rows, 2 * group, dim, 96)
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, dim ** -0.5, window=window)
    assert gw.kernel_error() == 0
    assert_rows(got, q, batch, host, dim ** -0.5, window, rows_of=[0, 1, rows - 1, rows // 2])


@pytest.mark.parametrize("what", ["query nan", "query infinity", "key", "key scale"])
@pytest.mark.parametrize("window", [0, 30])
def test_odd_keys_and_queries_reach_the_rows_that_see_them(gw, what, window):
    batch = Batch([(60, 200), (3, 150)], 16, 97)
    host = random_cache(batch, 2, 128, 98)
    clean = [tuple(a.copy() for a in part) for part in host]
    q = queries(batch.rows, 8, 128, 99)
    odd = torch.zeros((batch.rows, 8), dtype=torch.bool)
    if what == "key":
        host[0][0][int(batch.table[0, 9]), 1, 6, 17] = 0xff           # token 150
        odd[[i for i in range(60) if 140 + i >= 150 and (window == 0 or 140 + i - 150 < window)], 4:] = True
    elif what == "key scale":
        host[0][1][int(batch.table[0, 9]), 1] = float("nan")           # tokens 144 .. 159
        odd[[i for i in range(60) if 140 + i >= 144 and (window == 0 or 140 + i - 159 < window)], 4:] = True
    else:
        q[20, 3, 50] = float("nan") if what == "query nan" else float("-inf")
        odd[20, 3] = True
    got = gw.paged_attention(to_device(gw, host), batch.device(gw), q, 0.1, window=window)
    assert gw.kernel_error() == 0
    got = got.cpu()
    assert torch.equal(torch.isnan(got).any(dim=2), odd) and torch.equal(torch.isnan(got).all(dim=2), odd)
    # the others against the definition without what is odd; in the place of the odd ones what a clean call gives
    q = torch.nan_to_num(q, 0.0, 0.0, 0.0)
    want = gw.paged_attention(to_device(gw, clean), batch.device(gw), q, 0.1, window=window).cpu()
    got[odd] = want[odd]
    assert_rows(got, q, batch, clean, 0.1, window, rows_of=[0, 3, 4, 9, 10, 19, 20, 21, 30, 45, 59])


@pytest.mark.parametrize("heads,kv_heads,dim,rows", [(8, 2, 128, 1), (16, 2, 512, 3), (4, 4, 256, 90)])
def test_results_in_the_place_of_the_queries(gw, heads, kv_heads, dim, rows):
    batch = Batch([(rows, 2000), (1, 300), (rows, 700)], 64, 100)
    cache = to_device(gw, random_cache(batch, kv_heads, dim, 101, garbage=False))
    held, q = batch.device(gw), queries(batch.rows, heads, dim, 102)
    want = gw.paged_attention(cache, held, q, dim ** -0.5)
    assert gw.paged_attention(cache, held, q, dim ** -0.5, y=q) is q and torch.equal(q, want)
