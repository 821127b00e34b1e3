"""Append to the paged cache and head norms where they are easily wrong."""
import numpy as np
import pytest
import torch

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
