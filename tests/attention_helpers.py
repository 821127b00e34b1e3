"""Random batches and caches of the attention tests."""
from __future__ import annotations

import numpy as np
import torch

from oracle import attention as oat

VALUES = oat.e4m3_values()


class Batch:
    """Sequences [(rows, length)] over a pool with some pages to spare, their numbers shuffled, and entries that are not needed -1."""

    def __init__(self, sequences, page_tokens, seed, extra_rows=0, spare=2, extra_entries=2):
        rng = np.random.default_rng(seed)
        self.sequences, self.page_tokens = sequences, page_tokens
        needed = [-(-max(0, length) // page_tokens) for _, length in sequences]
        self.pages = sum(needed) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(sequences), max(needed) + extra_entries), -1, dtype=np.int32)
        at = 0
        for s, n in enumerate(needed):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.row_offsets = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
        self.lengths = np.array([length for _, length in sequences], dtype=np.int32)
        self.rows = int(self.row_offsets[-1]) + extra_rows
        self.max_rows = max(1, max(n for n, _ in sequences))

    def device(self, gw):
        return gw.SequenceBatch(*(torch.from_numpy(a).cuda() for a in (self.row_offsets, self.lengths, self.table)), self.rows, self.max_rows)


def random_cache(batch, kv_heads, dim, seed, spread=2.0, garbage=True):
    """Codes [pages, heads, P, D] (uint8) and scales of N(0, 1)-like rows, pages of different loudness; slots behind a sequence's last
    token, and pages of no sequence, hold any code (NaN too) and their scales NaN where garbage is wanted."""
    rng = np.random.default_rng(seed)
    shape = (batch.pages, kv_heads, batch.page_tokens, dim)
    out = []
    for _ in range(2):
        loud = 2.0 ** rng.uniform(-spread, spread, shape[:2])
        scales = 2.0 ** np.ceil(np.log2(loud * 5.0 / 448.0))
        x = torch.from_numpy((rng.standard_normal(shape) * (loud / scales)[..., None, None]).astype(np.float32)).clamp(-448, 448)
        codes = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy().copy()
        if garbage:
            used = np.zeros(shape[:1] + shape[2:3], dtype=bool)
            for s, (_, length) in enumerate(batch.sequences):
                for at in range(max(0, length)):
                    used[batch.table[s, at // batch.page_tokens], at % batch.page_tokens] = True
            rubbish = rng.integers(0, 256, shape, dtype=np.uint8)
            rubbish[..., ::3] = 127
            codes = np.where(used[:, None, :, None], codes, rubbish)
            scales = np.where(used.any(axis=1)[:, None], scales, np.nan)
        out.append((codes, scales.astype(np.float32)))
    return out


def to_device(gw, cache):
    (k, ks), (v, vs) = cache
    return gw.KvCache(*(torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in (k, v, ks, vs)))


def sequence_values(batch, cache, s):
    """Keys or values [heads, tokens, D] of a sequence in 64 bits."""
    codes, scales = cache
    length = int(batch.lengths[s])
    pages = batch.table[s, :-(-length // batch.page_tokens)]
    x = VALUES[codes[pages]] * scales[pages].astype(np.float64)[:, :, None, None]
    return x.transpose(1, 0, 2, 3).reshape(codes.shape[1], -1, codes.shape[3])[:, :length]


def joined(rows, heads, kv_heads, dim, seed, std=1.0):
    """Q, K, V slices of a joined projection output, BF16 on the device."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((rows, (heads + 2 * kv_heads) * dim), generator=g) * std).bfloat16().cuda()
    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    return q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))


def f64(t):
    return t.detach().double().cpu().numpy()
