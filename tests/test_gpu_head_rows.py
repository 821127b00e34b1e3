"""Head norms with rotation, and keys and values appended to a paged 8-bit cache, against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import attention as oat
from tests.attention_helpers import VALUES, Batch, f64, joined, random_cache, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gw():
    import gewell_b200
    return gewell_b200


def frequencies(width, still=0, base=1e4):
    half = width // 2
    return torch.tensor([base ** (-i / half) for i in range(half - still)] + [0.0] * still, dtype=torch.float32)


def weight_of(dim, seed):
    return (1.0 + 0.25 * torch.randn(dim, generator=torch.Generator().manual_seed(seed))).bfloat16().cuda()


def slack(exact):
    """What FP32 and the hardware's sine leave of a head of exact values: 2^-21 of absolute error on sine and cosine, and a
    dozen roundings of 2^-24, on elements of up to the head's largest -- 2^-19 of it covers both."""
    return 2.0 ** -19 * np.abs(exact).max(axis=-1, keepdims=True)


def assert_bf16(got, exact):
    error = np.abs(f64(got) - exact)
    assert (error <= 2.0 ** -8 * np.abs(exact) + slack(exact)).all(), float(error.max())


@pytest.mark.parametrize("rows,heads,kv_heads,dim,width,still,interleaved,far", [
    (1, 16, 2, 512, 512, 192, False, 262000), (37, 32, 16, 256, 256, 0, False, 131000), (5, 24, 8, 128, 64, 0, True, 30000),
    (300, 7, 7, 128, 128, 0, False, 500000), (3, 3, 1, 96, 96, 8, False, 900), (2, 1, 1, 8, 8, 0, True, 3), (11, 5, 2, 64, 48, 0, False, 70000),
    (4, 2, 2, 320, 320, 0, False, 10), (6, 9, 4, 512, 128, 0, False, 1000000), (9, 4, 4, 256, 2, 0, False, 2000000000),
    (130, 16, 8, 256, 208, 40, True, 4000), (2, 8, 1, 200, 100, 0, False, 5000)])
def test_norm_rotary(gw, rows, heads, kv_heads, dim, width, still, interleaved, far):
    q, k, _ = joined(rows, heads, kv_heads, dim, 1, 3.0)
    positions = torch.randint(0, far, (rows,), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    positions[0] = far - 1
    f, qw, kw = frequencies(width, still), weight_of(dim, 3), weight_of(dim, 4)
    qo, ko = gw.qk_norm_rotary(q, k, qw, kw, positions.cuda(), f.cuda(), interleaved=interleaved)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        assert_bf16(got, oat.head_norm_rotary(f64(x), f64(w), True, positions.numpy(), f.numpy(), interleaved))


def test_norm_rotary_in_place_and_alone(gw):
    """Queries alone, without rotation, into their own rows; what lies between the rows stays."""
    q, k, _ = joined(9, 4, 2, 256, 5)
    before, other = f64(q), k.clone()
    got, none = gw.qk_norm_rotary(q, None, None, None, torch.zeros(9, dtype=torch.int32).cuda(), None, query_out=q)
    assert none is None and got is q
    assert_bf16(q, oat.head_norm_rotary(before, None, True, None, None))
    assert torch.equal(k, other)
    zero = torch.zeros((2, 3, 128), dtype=torch.bfloat16).cuda()
    got, _ = gw.qk_norm_rotary(zero, None, None, None, torch.zeros(2, dtype=torch.int32).cuda(), None)
    assert torch.equal(got, zero)
    assert gw.qk_norm_rotary(zero[:0], None, None, None, torch.zeros(0, dtype=torch.int32).cuda(), None)[0].shape == (0, 3, 128)


def check_append(gw, batch, kv_heads, dim, seed, width=None, still=0, interleaved=False, norm=True, weight=True, loud=1.0, query=0,
                 positions=None):
    cache_host = random_cache(batch, kv_heads, dim, seed)
    # tokens that are there already lie in pages whose scale is small, so that the call's tokens are often the louder ones
    cache = to_device(gw, cache_host)
    q, k, v = joined(batch.rows, max(1, query), kv_heads, dim, seed + 1, loud)
    w = weight_of(dim, seed + 2) if weight else None
    f = frequencies(width or dim, still)
    out = gw.kv_cache_append(cache, batch.device(gw), k, v, key_weight=w, normalize_key=norm, normalize_value=norm, frequencies=f.cuda(),
                             interleaved=interleaved, positions=None if positions is None else positions.cuda(),
                             query=q if query else None, query_weight=w if query else None)
    torch.cuda.synchronize()
    assert gw.kernel_error() == 0
    rows = int(batch.row_offsets[-1])
    at = np.concatenate([np.arange(length - n, length) for n, length in batch.sequences]) if positions is None else positions.numpy()[:rows]
    host_w = f64(w) if weight else None
    exact_k = oat.head_norm_rotary(f64(k)[:rows], host_w, norm, at, f.numpy(), interleaved)
    exact_v = oat.head_norm_rotary(f64(v)[:rows], None, norm, None, None)
    for x, (codes, scales), got, got_scales in ((exact_k, cache_host[0], cache.k_data, cache.k_scales), (exact_v, cache_host[1], cache.v_data, cache.v_scales)):
        got, got_scales = got.cpu().numpy(), f64(got_scales)
        wanted, wanted_scales, touched = oat.append(VALUES[codes], scales, x, batch.row_offsets, batch.lengths, batch.table)
        same = (got_scales == wanted_scales) | (np.isnan(got_scales) & np.isnan(wanted_scales))
        assert same.all(), np.argwhere(~same)[:4]
        assert (got[touched == 0] == codes[touched == 0]).all()
        assert (VALUES[got[touched == 1]] == wanted[touched == 1]).all()
        # a new token: half a step of E4M3 (2^-4 of the value, 2^-10 below the normal ones), and a tie may fall the other way
        new = wanted[touched == 2]
        assert (np.abs(VALUES[got[touched == 2]] - new) <= 2.0 ** -4 * np.abs(new) + 2.0 ** -10 + 2.0 * slack(new)).all()
    if query:
        exact_q = oat.head_norm_rotary(f64(q)[:rows], host_w, True, at, f.numpy(), interleaved)
        assert_bf16(out[:rows], exact_q)
    return cache


DECODE = [(1, 1), (1, 17), (1, 64), (1, 65), (1, 1000), (1, 2), (1, 16), (1, 129)]
MIXED = [(1, 40), (200, 200), (0, 77), (7, 131), (64, 64), (1, 1), (33, 96), (0, 0), (130, 515)]


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("kv_heads,dim", [(3, 128), (2, 256), (4, 512)])
@pytest.mark.parametrize("kind", ["decode", "mixed", "drafts"])
def test_append(gw, page, kv_heads, dim, kind):
    sequences = {"decode": DECODE, "mixed": MIXED, "drafts": [(3, 18), (5, 5), (1, 66), (4, 130), (2, 200)]}[kind]
    check_append(gw, Batch(sequences, page, page + dim), kv_heads, dim, page + dim + 1)


@pytest.mark.parametrize("options", [dict(interleaved=True, width=64), dict(width=96), dict(norm=False, weight=False, loud=30.0),
                                     dict(norm=False, loud=1e-3), dict(still=48), dict(query=6), dict(query=3, width=32)])
@pytest.mark.parametrize("sequences", [DECODE, MIXED])
def test_append_options(gw, options, sequences):
    check_append(gw, Batch(sequences, 32, 9), 2, 128, 10, **options)


def test_append_positions_of_the_caller(gw):
    batch = Batch([(1, 40), (5, 90)], 16, 3, extra_rows=2)
    check_append(gw, batch, 2, 256, 4, positions=torch.tensor([7, 100000, 3, 3, 250000, 1, 0, 0], dtype=torch.int32), query=2)


def test_append_rows_behind_the_last_sequence_and_long_batches(gw):
    check_append(gw, Batch([(2, 30), (1, 9)], 16, 5, extra_rows=5), 2, 128, 6, query=2)
    rng = np.random.default_rng(0)
    lengths = rng.integers(1, 90, 700)
    check_append(gw, Batch([(int(rng.integers(0, min(4, n + 1))), int(n)) for n in lengths], 32, 7), 1, 128, 8)


def test_append_step_by_step_rounds_a_page_again(gw):
    """Tokens that get louder one by one: after each the page holds every token to the rounding of the scale it has then, and the
    same tokens in one call give the page the same scale."""
    page, dim, steps = 16, 128, 16
    g = torch.Generator().manual_seed(3)
    rows = torch.stack([torch.randn((1, dim), generator=g) * 2.0 ** (i / 2 - 3) for i in range(steps)]).bfloat16().cuda()
    pool = [torch.zeros((2, 1, page, dim), dtype=torch.uint8).cuda() for _ in range(4)]
    scales = [torch.full((2, 1), float("nan")).cuda() for _ in range(4)]
    one, all_at_once = gw.KvCache(*pool[:2], *scales[:2]), gw.KvCache(*pool[2:], *scales[2:])
    table = torch.tensor([[1]], dtype=torch.int32).cuda()
    for i in range(steps):
        batch = gw.SequenceBatch(torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.tensor([i + 1], dtype=torch.int32).cuda(), table, 1, 1)
        gw.kv_cache_append(one, batch, rows[i:i + 1], rows[i:i + 1], normalize_key=False, normalize_value=False)
        scale = float(one.k_scales[1])
        held = VALUES[one.k_data[1, 0, :i + 1].cpu().numpy()] * scale
        exact = f64(rows[:i + 1, 0])
        # a value is rounded again at most when the scale doubles: normal codes keep their value then, so all but one rounding
        # fall on codes below the normal ones, half a step of 2^-9 of the scale each time; the halves of earlier, smaller scales add up to one more
        assert (np.abs(held - exact) <= 2.0 ** -4 * np.abs(exact) + 2 * 2.0 ** -10 * scale).all()
    batch = gw.SequenceBatch(torch.tensor([0, steps], dtype=torch.int32).cuda(), torch.tensor([steps], dtype=torch.int32).cuda(), table, steps, steps)
    gw.kv_cache_append(all_at_once, batch, rows, rows, normalize_key=False, normalize_value=False)
    assert torch.equal(one.k_scales[1], all_at_once.k_scales[1]) and gw.kernel_error() == 0


def test_append_odd_values(gw):
    """Zeros, infinities and NaN: the scale goes by what is finite."""
    x = torch.zeros((3, 1, 128), dtype=torch.bfloat16)
    x[1, 0, :4] = torch.tensor([3.0, float("inf"), float("-inf"), float("nan")])
    x = x.cuda()
    cache = gw.KvCache(*(torch.full((3, 1, 16, 128), 9, dtype=torch.uint8).cuda() for _ in range(2)), *(torch.ones((3, 1)).cuda() for _ in range(2)))
    batch = gw.SequenceBatch(torch.tensor([0, 1, 3], dtype=torch.int32).cuda(), torch.tensor([1, 2], dtype=torch.int32).cuda(),
                             torch.tensor([[2], [0]], dtype=torch.int32).cuda(), 3, 2)
    gw.kv_cache_append(cache, batch, x, x, normalize_key=False, normalize_value=False)
    assert float(cache.k_scales[2]) == oat.TINY and (cache.k_data[2, 0, 0] == 0).all() and (cache.k_data[2, 0, 1:] == 9).all()
    scale = float(cache.k_scales[0])
    assert scale == 2.0 ** -7 and (cache.k_data[0, 0, 1] == 0).all() and (cache.k_data[0, 0, 2:] == 9).all()
    first = VALUES[cache.k_data[0, 0, 0, :5].cpu().numpy()] * scale
    assert first[0] == 3.0 and first[1] == 448 * scale and first[2] == -448 * scale and np.isnan(first[3]) and first[4] == 0
    assert (cache.k_data[1] == 9).all() and float(cache.k_scales[1]) == 1.0


def test_append_leaves_out_what_it_cannot_follow(gw):
    """Page numbers outside the cache, positions behind the table, offsets out of range: left out and reported; the rest is done."""
    def cache():
        return gw.KvCache(*(torch.zeros((2, 1, 16, 128), dtype=torch.uint8).cuda() for _ in range(2)), *(torch.ones((2, 1)).cuda() for _ in range(2)))
    x = torch.ones((4, 1, 128), dtype=torch.bfloat16).cuda()

    def run(offsets, lengths, table, rows=4, most=4):
        c = cache()
        t = [torch.tensor(a, dtype=torch.int32).cuda() for a in (offsets, lengths, table)]
        gw.kv_cache_append(c, gw.SequenceBatch(*t, rows, most), x, x, normalize_key=False, normalize_value=False)
        return c.k_data.cpu().numpy().any(axis=(1, 3)), gw.kernel_error()
    for table in ([[5], [1]], [[-1], [1]], [[2 ** 30], [1]]):
        for offsets, most in (([0, 2, 4], 4), ([0, 1, 2], 1)):
            written, error = run(offsets, [2, 2], table, most=most)
            assert error >> 24 == 0xa1 and not written[0].any() and written[1, :2].any()
    written, error = run([0, 2, 4], [2, 40], [[0], [1]])              # the second sequence's pages lie behind the table
    assert error >> 24 == 0xa1 and written[0, :2].all() and not written[1].any()
    for offsets in ([0, 2, 9], [-3, 2, 4], [0, 4, 2]):
        written, error = run(offsets, [2, 2], [[0], [1]])
        assert error >> 24 == 0xa2
    written, error = run([0, 3, 4], [1, 0], [[0], [-1]])              # rows in front of position 0: no tokens, no error
    assert error == 0 and written[0, 0] and not written[0, 1:].any() and not written[1].any()


def test_append_captured_and_on_a_stream(gw):
    batch, dim = Batch(MIXED, 32, 11), 256
    host = random_cache(batch, 2, dim, 12)
    _, k, v = joined(batch.rows, 1, 2, dim, 13)
    plain, other = to_device(gw, host), to_device(gw, host)
    gw.kv_cache_append(plain, batch.device(gw), k, v)
    held = batch.device(gw)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        gw.kv_cache_append(other, held, k, v)
    for _ in range(2):                     # the same tokens again: nothing changes
        graph.replay()
    torch.cuda.synchronize()
    for name in ("k_data", "v_data", "k_scales", "v_scales"):
        a, b = getattr(plain, name), getattr(other, name)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name
    assert gw.kernel_error() == 0
