"""A paged cache with ragged sequences, a permuted block table and poison in every place that must not be read, with
plain 64-bit forms of the serving operators on it."""
import math

import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}   # half a step relative to the value


class Cache:
    def __init__(self, rng, lens, hkv, d, dv, block, dtype, room=0, poison=np.nan, round_bf16=None, spare_pages=3):
        self.lens, self.hkv, self.d, self.dv, self.block, self.dtype = list(lens), hkv, d, dv, block, dtype
        self.batch = len(self.lens)
        self.max_blocks = max(1, max((n + room + block - 1) // block for n in self.lens))
        need = [(n + room + block - 1) // block for n in self.lens]
        self.num_blocks = sum(need) + spare_pages
        pages = rng.permutation(self.num_blocks)
        self.table = np.full((self.batch, self.max_blocks), -7, np.int32)     # never followed
        self.k_pool = np.full((self.num_blocks, hkv, block, d), poison, np.float32)
        self.v_pool = np.full((self.num_blocks, hkv, block, dv), poison, np.float32)
        self.keys, self.values = [], []
        at = 0
        for b, n in enumerate(self.lens):
            k = rng.standard_normal((hkv, n, d)).astype(np.float32)
            v = rng.standard_normal((hkv, n, dv)).astype(np.float32)
            if dtype == "bf16":
                k, v = round_bf16(k), round_bf16(v)
            self.keys.append(k.astype(np.float64))
            self.values.append(v.astype(np.float64))
            for i in range(need[b]):
                self.table[b, i] = pages[at]
                rows = max(0, min(block, n - i * block))
                self.k_pool[pages[at], :, :rows] = k[:, i * block:i * block + rows]
                self.v_pool[pages[at], :, :rows] = v[:, i * block:i * block + rows]
                at += 1

    def rows(self, pool, b, n):
        """[hkv, n, dim] of sequence b out of a (possibly changed) pool."""
        if n == 0:
            return np.zeros((self.hkv, 0, pool.shape[-1]))
        pages = self.table[b, : (n + self.block - 1) // self.block]
        return np.concatenate([pool[p] for p in pages], axis=1)[:, :n].astype(np.float64)


def softmax_rows(x):
    """Rows of logits (-inf = masked) -> weights; a row without a visible entry gives zeros."""
    top = x.max(-1, keepdims=True, initial=-np.inf)
    e = np.exp(x - np.where(np.isfinite(top), top, 0.0))
    total = e.sum(-1, keepdims=True)
    return e / np.where(total == 0.0, 1.0, total)


def attention_bound(q, keys, values, want, dtype, scale):
    """How far a correct kernel may be from the 64-bit result.  A logit is a sum of d products held in 32 bits: off by
    at most (d + 4) half steps of sum |q_i k_i| * scale; weights change by twice that relatively; each exponential is
    good to 2^-21, the sums over n keys to n half steps of 32 bits; bf16 kernels round the weights once and the output
    once, half a step of bf16 each."""
    if keys.shape[0] == 0:
        return np.zeros_like(want)
    logit = (q.shape[-1] + 4) * HALF_STEP["f32"] * (np.abs(q) @ np.abs(keys).T).max(-1, keepdims=True) * scale
    weights = 2.0 * logit + 2.0 ** -21 + keys.shape[0] * HALF_STEP["f32"]
    if dtype == "bf16":
        weights = weights + HALF_STEP["bf16"]
    return weights * np.abs(values).max() + HALF_STEP[dtype] * np.abs(want) + 1e-30


def attend(q, keys, values, dtype, scale=0.0, hidden=None):
    """q [rows, d] over keys [n, d]: (output, bound, weights) in 64 bits."""
    scale = scale if scale > 0 else 1.0 / math.sqrt(q.shape[-1])
    x = q @ keys.T * scale
    if hidden is not None:
        x = np.where(hidden, -np.inf, x)
    p = softmax_rows(x)
    want = p @ values if keys.shape[0] else np.zeros((q.shape[0], values.shape[-1]))
    return want, attention_bound(q, keys, values, want, dtype, scale), p


def ancestors(parents, count):
    """Visible matrix [count, count] of a tree."""
    see = np.zeros((count, count), bool)
    for i in range(count):
        if 0 <= parents[i] < i:
            see[i] = see[parents[i]]
        see[i, i] = True
    return see


def random_tree(rng, nodes):
    return np.array([int(rng.integers(-1, i)) if i else -1 for i in range(nodes)], np.int32)
