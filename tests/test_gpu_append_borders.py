"""Append to the paged cache and head norms where they are easily wrong."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import attention as oat
from tests.attention_helpers import VALUES, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gw():
    import gewell_b200
    return gewell_b200


def small_cache(gw, pages, dim=128, page=16, heads=1):
    return gw.KvCache(*(torch.zeros((pages, heads, page, dim), dtype=torch.uint8).cuda() for _ in range(2)),
                      *(torch.ones((pages, heads)).cuda() for _ in range(2)))


def batch_of(gw, offsets, lengths, table, rows, most):
    return gw.SequenceBatch(*(torch.tensor(np.asarray(a).tolist(), dtype=torch.int32).cuda() for a in (offsets, lengths, table)), rows, most)


@pytest.mark.parametrize("dim,page,most", [(128, 16, 1), (128, 16, 2), (256, 16, 8), (512, 64, 20), (128, 128, 100)])
@pytest.mark.parametrize("kind", ["length", "offset", "rows"])
def test_a_bad_sequence_behind_many_good_ones_is_reported(gw, dim, page, most, kind):
    """The last of 1200 sequences cannot be followed: it is left out and reported, and the others are done."""
    count = 1200
    offsets, lengths = np.arange(count + 1), np.ones(count, dtype=np.int64)
    rows = count + most + 1
    if kind == "length":
        lengths[-1] = 2 ** 30 + 1
    elif kind == "offset":
        offsets[-1] = rows + 1
    else:
        offsets[-1] = count + most                                       # one row more than max_rows
    x = torch.ones((rows, 1, dim), dtype=torch.bfloat16).cuda()
    cache = small_cache(gw, count, dim, page)
    gw.kv_cache_append(cache, batch_of(gw, offsets, lengths, np.arange(count).reshape(count, 1), rows, most), x, x, normalize_key=False, normalize_value=False)
    assert gw.kernel_error() == 0xa2000000 | (count - 1)
    written = cache.k_data[:, 0, 0].any(dim=1)
    assert written[:-1].all() and not written[-1]


@pytest.mark.parametrize("given", [False, True])
def test_query_rows_of_no_sequence_stay(gw, given):
    """Rows behind the last sequence, and of one that cannot be followed, are left as they are, wherever the positions come from."""
    heads, dim, rows = 3, 128, 9
    x = torch.randn((rows, heads, dim), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    k = x[:, :1].contiguous()
    positions = torch.tensor([5, 0, 1, 2, 9, 9, 9, 9, 9], dtype=torch.int32)
    f = torch.tensor([1e4 ** (-i / 64) for i in range(64)], dtype=torch.float32)
    for lengths, good, error in (([6, 3], [0, 1, 2, 3], 0), ([6, 2 ** 30 + 1], [0], 0xa2000001)):
        y = torch.full_like(x, 7.0)
        gw.kv_cache_append(small_cache(gw, 2, dim), batch_of(gw, [0, 1, 4], lengths, [[0], [1]], rows, 3), k, k, frequencies=f.cuda(),
                           positions=positions.cuda() if given else None, query=x, query_out=y)
        assert gw.kernel_error() == error
        rest = [r for r in range(rows) if r not in good]
        assert (y[rest] == 7.0).all()
        exact = oat.head_norm_rotary(f64(x)[good], None, True, positions.numpy()[good], f.numpy())
        assert (np.abs(f64(y)[good] - exact) <= 2.0 ** -8 * np.abs(exact) + 2.0 ** -19 * np.abs(exact).max(axis=-1, keepdims=True)).all()


def test_single_elements_of_wider_tensors(gw):
    """One row at a position, one pair and one sequence, each a view with another stride."""
    x = torch.randn((1, 2, 128), generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    position, f = torch.tensor([9, 0, 0, 0], dtype=torch.int32).cuda(), torch.tensor([0.25, 0.0, 0.0], dtype=torch.float32).cuda()
    got, _ = gw.qk_norm_rotary(x, None, None, None, position[::4], f[::3])
    want, _ = gw.qk_norm_rotary(x, None, None, None, position[:1], f[:1])
    exact = oat.head_norm_rotary(f64(x), None, True, np.array([9]), np.array([0.25]))
    assert torch.equal(got, want)
    assert (np.abs(f64(got) - exact) <= 2.0 ** -8 * np.abs(exact) + 2.0 ** -19 * np.abs(exact).max(axis=-1, keepdims=True)).all()


@pytest.mark.parametrize("dim,width", [(128, 64), (256, 20), (512, 16), (128, 2)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows", [1, 3, 30])
def test_odd_values_behind_the_rotated_width_stay_where_they_are(gw, dim, width, interleaved, rows):
    """An infinity or NaN among the elements that are not turned changes none of its neighbours."""
    x = torch.zeros((rows, 1, dim), dtype=torch.bfloat16)
    x[:, 0, width:] = 3.0
    x[:, 0, :width] = 1.0
    x[:, 0, width], x[:, 0, width + 6], x[:, 0, dim - 1] = float("inf"), float("nan"), float("-inf")
    cache = small_cache(gw, 2, dim, 32)
    f = torch.ones(width // 2, dtype=torch.float32).cuda()
    gw.kv_cache_append(cache, batch_of(gw, [0, rows], [rows], [[1]], rows, rows), x.cuda(), x.cuda(), normalize_key=False, normalize_value=False,
                       frequencies=f, interleaved=interleaved)
    assert gw.kernel_error() == 0 and float(cache.k_scales[1]) == 2.0 ** -7
    got = VALUES[cache.k_data[1, 0, :rows].cpu().numpy()] * 2.0 ** -7
    wanted = np.full((rows, dim - width), 3.0)
    wanted[:, 0], wanted[:, 6], wanted[:, -1] = 3.5, np.nan, -3.5           # infinities become the largest code
    np.testing.assert_array_equal(got[:, width:], wanted)


PI = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)


def sine_cosine(position, frequency):
    """Of position * frequency (FP32), reduced in whole numbers."""
    angle = position * Fraction(frequency)
    rest = angle - round(angle / (2 * PI)) * 2 * PI
    return math.sin(rest), math.cos(rest)


@pytest.mark.parametrize("low,high", [(0, 1 << 12), (1 << 19, 1 << 20), ((1 << 24) - 1000, 1 << 24), ((1 << 24) + 1, (1 << 24) + 1000), ((1 << 31) - 1000, (1 << 31) - 1)])
@pytest.mark.parametrize("dim,width,interleaved", [(128, 128, False), (128, 128, True), (128, 64, False), (512, 512, False)])
def test_sines_are_as_exact_as_fp32(gw, low, high, dim, width, interleaved):
    """Pairs that nearly cancel: (sin a, cos a) turned by a has a first element of 2^-9 or less, and the error of the sines is seen next to its
    rounding to BF16.

    A sine or cosine is off by a unit of 2^-24 (sincospif), the angle's rest by 2^-28 turns, 2^-25 rad, and the correction by it by half a unit:
    2 * 2^-24 in all, of both elements n of the pair; each of those is rounded once (2^-24), and so is their first product.  The norm's
    factor is common to both and cancels with them.  What the hardware's sines leave is 2^-21 of each element."""
    rng = np.random.default_rng(7)
    rows, pairs = 96, width // 2
    positions = rng.integers(low, high, rows)
    positions[0] = high - 1
    f = np.array([1e4 ** (-i / pairs) for i in range(pairs)], dtype=np.float32)
    f[::7] = 1.0
    turned = np.array([[sine_cosine(int(p), float(v)) for v in f] for p in positions])
    first = np.arange(0, width, 2) if interleaved else np.arange(pairs)
    second = first + 1 if interleaved else first + pairs
    x = np.zeros((rows, 1, dim))
    x[:, 0, first], x[:, 0, second] = turned[..., 0], turned[..., 1]
    held = torch.from_numpy(x).bfloat16().cuda()
    got, _ = gw.qk_norm_rotary(held, None, None, None, torch.from_numpy(positions).int().cuda(), torch.from_numpy(f).cuda(), interleaved=interleaved)
    n = oat.head_norm_rotary(f64(held), None, True, None, None)
    a, b = n[:, 0, first], n[:, 0, second]
    exact = a * turned[..., 1] - b * turned[..., 0]
    error = np.abs(f64(got)[:, 0, first] - exact)
    bound = 2.0 ** -8 * np.abs(exact) + 4 * 2.0 ** -24 * (np.abs(a) + np.abs(b))
    assert (np.abs(exact) < 2.0 ** -13).sum() > 50
    assert (error <= bound).all(), float((error / bound).max())
