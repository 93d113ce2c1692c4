"""Serving operators over the paged cache through the kernel ABI: tree attention, append of an accepted path, block
bounds and sparse decode, accumulated weights and eviction, each against a plain 64-bit form."""
import ctypes as C

import numpy as np
import pytest

from cache_problem import Cache, ancestors, attend, random_tree
from schedforge_b200 import lib as L

gpu = pytest.mark.gpu
CODE = {"f32": L.F32, "bf16": L.BF16}


# ---- helpers ---------------------------------------------------------------------------------------------------


def status_word():
    word = C.c_uint32(0)
    L.check(L.load().sfb_device_status(C.byref(word)))
    return word.value


class Device:
    """The cache's arrays on the device, in its type; `keep` holds what the argument structs point to."""

    def __init__(self, dev, cache):
        self.dev, self.cache = dev, cache
        self.put = dev.bf16 if cache.dtype == "bf16" else dev.f32
        self.type = dev.torch.bfloat16 if cache.dtype == "bf16" else dev.torch.float32
        self.k_pool, self.v_pool = self.put(cache.k_pool), self.put(cache.v_pool)
        self.table, self.lens = dev.i32(cache.table), dev.i32(np.array(cache.lens))

    def fill(self, a, **more):
        c = self.cache
        a.k_pool, a.v_pool = self.k_pool.data_ptr(), self.v_pool.data_ptr()
        a.block_table, a.context_len = self.table.data_ptr(), self.lens.data_ptr()
        a.batch, a.kv_heads, a.head_dim, a.head_dim_value = c.batch, c.hkv, c.d, c.dv
        a.block_tokens, a.max_blocks, a.num_blocks = c.block, c.max_blocks, c.num_blocks
        a.dtype = CODE[c.dtype]
        for name, value in more.items():
            setattr(a, name, value.data_ptr() if hasattr(value, "data_ptr") else value)
        return a


def workspace(dev, nbytes):
    return dev.torch.full((max(16, int(nbytes)),), 0xff, dtype=dev.torch.uint8, device="cuda")  # NaN patterns: never read first


def rounder(port, dtype):
    return port.round_bf16 if dtype == "bf16" else (lambda a: a.astype(np.float32))


def close(got, want, bound):
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), f"off by {off.max():.3e}, allowed {bound.flat[np.argmax(off - bound)]:.3e}"


# ---- tree attention ------------------------------------------------------------------------------------------------


def tree_call(dev, port, cache, hq, nodes, counts, parents, q, dk, dv, token_major=0, splits=0, scale=0.0, stream=None,
              max_context=None, poison=7.0):
    d = Device(dev, cache)
    torch = dev.torch
    t = dict(q=d.put(q), draft_k=d.put(dk), draft_v=d.put(dv), parents=dev.i32(parents), node_count=dev.i32(counts))
    shape = (cache.batch, nodes, hq, cache.dv) if token_major else (cache.batch, hq, nodes, cache.dv)
    out = torch.full(shape, poison, dtype=d.type, device="cuda")
    a = d.fill(L.TreeArgs(), **t, out=out, q_heads=hq, nodes=nodes, splits=splits, scale=scale, token_major=token_major,
               max_context=max(cache.lens) if max_context is None else max_context)
    ws = workspace(dev, L.load().sfb_attention_tree_workspace(C.byref(a)))
    a.workspace = ws.data_ptr()
    torch.cuda.synchronize()
    L.check(L.load().sfb_k_attention_tree_paged(C.byref(a), C.c_void_p(stream if stream is not None else dev.stream())))
    torch.cuda.synchronize()
    got = dev.np(out)
    return got.transpose(0, 2, 1, 3) if token_major else got


def tree_inputs(rng, port, cache, hq, nodes, counts, chain=False):
    r = rounder(port, cache.dtype)
    q = r(rng.standard_normal((cache.batch, hq, nodes, cache.d)).astype(np.float32) * 1.5)
    dk = r(rng.standard_normal((cache.batch, cache.hkv, nodes, cache.d)).astype(np.float32))
    dv = r(rng.standard_normal((cache.batch, cache.hkv, nodes, cache.dv)).astype(np.float32))
    parents = np.stack([np.arange(nodes, dtype=np.int32) - 1 if chain else random_tree(rng, nodes) for _ in range(cache.batch)])
    for b, n in enumerate(counts):   # dead nodes hold anything
        dk[b, :, n:], dv[b, :, n:] = np.nan, np.inf
        parents[b, n:] = 1 << 20
    return q, dk, dv, parents


def tree_check(got, cache, hq, counts, parents, q, dk, dv, scale=0.0, poison=7.0):
    group = hq // cache.hkv
    for b in range(cache.batch):
        n = counts[b]
        assert np.all(got[b, :, n:] == poison), "rows of dead nodes were written"
        if n == 0:
            continue
        hidden = np.concatenate([np.zeros((n, cache.lens[b]), bool), ~ancestors(parents[b], n)], 1)
        for h in range(hq):
            k = np.concatenate([cache.keys[b][h // group], dk[b, h // group, :n].astype(np.float64)])
            v = np.concatenate([cache.values[b][h // group], dv[b, h // group, :n].astype(np.float64)])
            want, bound, _ = attend(q[b, h, :n].astype(np.float64), k, v, cache.dtype, scale, hidden)
            close(got[b, h, :n], want, bound)


TREE_CASES = [
    # dtype, hq, hkv, d, dv, block, nodes, lens, counts, token_major, splits
    ("f32", 4, 2, 32, 32, 16, 5, [0, 1, 33], [5, 3, 1], 0, 0),
    ("f32", 6, 2, 20, 12, 4, 7, [9, 64, 65], [7, 0, 7], 1, 0),          # dims and blocks that are no multiples of anything
    ("f32", 8, 8, 64, 64, 16, 27, [500, 130], [27, 20], 0, 3),
    ("f32", 8, 1, 256, 200, 32, 33, [70], [33], 0, 0),
    ("f32", 8, 2, 128, 128, 16, 40, [300, 0, 64, 63], [40, 40, 33, 1], 1, 0),
    ("f32", 4, 1, 72, 40, 16, 70, [129, 640], [70, 64], 0, 2),           # three tiles of 128 query rows, two of draft keys
    ("f32", 2, 2, 8, 8, 16, 3, [70], [3], 0, 0),
    ("bf16", 8, 2, 64, 64, 16, 1, [300, 0, 17], [1, 1, 1], 0, 0),       # one token
    ("bf16", 8, 2, 128, 128, 16, 9, [300, 0, 17, 128], [9, 9, 4, 2], 0, 0),
    ("bf16", 32, 8, 128, 128, 16, 64, [700, 1000], [64, 50], 1, 0),     # two row tiles of 128
    ("bf16", 8, 1, 128, 128, 32, 61, [257, 511], [61, 60], 0, 2),       # 488 query rows for one K/V head
    ("bf16", 8, 2, 64, 64, 64, 37, [640, 63], [37, 31], 1, 0),
    ("bf16", 6, 2, 80, 96, 16, 12, [100, 47], [12, 5], 0, 0),           # not for the tensor-core kernel
    ("bf16", 3, 3, 128, 128, 24, 20, [100, 191], [20, 20], 0, 0),       # block of 24 tokens
    ("bf16", 4, 4, 64, 64, 16, 256, [40], [256], 0, 0),                 # the most nodes there can be
    ("bf16", 4, 1, 128, 128, 8, 11, [300, 5], [11, 11], 0, 0),          # the smallest blocks TMA takes
    ("bf16", 4, 1, 64, 64, 256, 11, [700, 129], [11, 2], 1, 0),         # blocks longer than a key tile
    ("bf16", 4, 1, 128, 128, 1, 4, [37], [4], 0, 0),                    # blocks of one token
    ("bf16", 4, 2, 128, 128, 16, 130, [1500], [129], 0, 5),             # draft keys over more than one tile
]


@gpu
@pytest.mark.parametrize("dtype,hq,hkv,d,dv,block,nodes,lens,counts,token_major,splits", TREE_CASES)
def test_tree_attention(dev, port, dtype, hq, hkv, d, dv, block, nodes, lens, counts, token_major, splits):
    rng = np.random.default_rng(nodes * 7 + d)
    cache = Cache(rng, lens, hkv, d, dv, block, dtype, round_bf16=port.round_bf16)
    q, dk, dvv, parents = tree_inputs(rng, port, cache, hq, nodes, counts)
    got = tree_call(dev, port, cache, hq, nodes, counts, parents, q, dk, dvv, token_major, splits)
    assert status_word() == 0
    tree_check(got, cache, hq, counts, parents, q, dk, dvv)


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("f32", 64)])
def test_tree_of_one_branch_is_causal_attention(dev, port, dtype, d):
    rng = np.random.default_rng(3)
    cache = Cache(rng, [200, 77], 2, d, d, 16, dtype, round_bf16=port.round_bf16)
    nodes, hq, counts = 40, 8, [40, 40]
    q, dk, dv, parents = tree_inputs(rng, port, cache, hq, nodes, counts, chain=True)
    got = tree_call(dev, port, cache, hq, nodes, counts, parents, q, dk, dv, scale=0.05)
    for b in range(2):
        for h in range(hq):
            k = np.concatenate([cache.keys[b][h // 4], dk[b, h // 4].astype(np.float64)])
            v = np.concatenate([cache.values[b][h // 4], dv[b, h // 4].astype(np.float64)])
            hidden = np.arange(k.shape[0])[None, :] > cache.lens[b] + np.arange(nodes)[:, None]
            want, bound, _ = attend(q[b, h].astype(np.float64), k, v, dtype, 0.05, hidden)
            close(got[b, h], want, bound)


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 32)])
def test_tree_large_logits_and_every_split_count_agree(dev, port, dtype, d):
    """Logits in the hundreds: the running maximum moves; all split counts stay within the bound."""
    rng = np.random.default_rng(4)
    cache = Cache(rng, [900], 2, d, d, 16, dtype, round_bf16=port.round_bf16)
    q, dk, dv, parents = tree_inputs(rng, port, cache, 4, 6, [6])
    q = rounder(port, dtype)(q * 20.0)
    for splits in (1, 2, 4, 128):
        got = tree_call(dev, port, cache, 4, 6, [6], parents, q, dk, dv, splits=splits)
        tree_check(got, cache, 4, [6], parents, q, dk, dv)


@gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 32)])
def test_tree_bad_parents_counts_lengths_and_blocks_are_cut_and_reported(dev, port, dtype, d):
    rng = np.random.default_rng(5)
    lens = [64, 64, 64, 64]
    cache = Cache(rng, lens, 1, d, d, 16, dtype, round_bf16=port.round_bf16)
    nodes, hq, counts = 6, 2, [6, 6, 6, 6]
    q, dk, dv, parents = tree_inputs(rng, port, cache, hq, nodes, counts)
    status_word()
    bad = parents.copy()
    bad[0, 3], bad[0, 4] = 3, -9                        # its own parent; below -1: both count as roots
    good = parents.copy()
    good[0, 3] = good[0, 4] = -1
    got = tree_call(dev, port, cache, hq, nodes, counts, bad, q, dk, dv)
    assert status_word() & 0x200
    tree_check(got, cache, hq, counts, good, q, dk, dv)
    tree_call(dev, port, cache, hq, nodes, [6, 6, 6, -1], parents, q, dk, dv)
    assert status_word() & 0x200
    got = tree_call(dev, port, cache, hq, nodes, [6, 99, 6, -3], parents, q, dk, dv)   # cut to 6 and to 0
    assert status_word() & 0x200
    tree_check(got, cache, hq, [6, 6, 6, 0], parents, q, dk, dv)
    cache.lens = [64, 1000, 64, -5]                                                     # cut to 64 and to 0
    got = tree_call(dev, port, cache, hq, nodes, counts, parents, q, dk, dv, max_context=64)
    assert status_word() & 0x200
    cache.lens = [64, 64, 64, 0]
    keys, values = list(cache.keys), list(cache.values)
    cache.keys[3], cache.values[3] = keys[3][:, :0], values[3][:, :0]
    tree_check(got, cache, hq, counts, parents, q, dk, dv)
    cache.lens, cache.keys, cache.values = lens, keys, values
    cache.table[2, 1] = cache.num_blocks + 11                                           # positions 16..31 are masked
    got = tree_call(dev, port, cache, hq, nodes, counts, parents, q, dk, dv)
    assert status_word() & 0x200
    keep = np.r_[0:16, 32:64]
    cache.keys[2], cache.values[2] = cache.keys[2][:, keep], cache.values[2][:, keep]
    cache.lens = [64, 64, 48, 64]
    tree_check(got, cache, hq, counts, parents, q, dk, dv)


# ---- accepted path ---------------------------------------------------------------------------------------------------


def accept_call(dev, d, cache, nodes, path, path_len, dk, dv, new_len=True):
    t = dict(draft_k=d.put(dk), draft_v=d.put(dv), path=dev.i32(path), path_len=dev.i32(path_len))
    out = dev.i32(np.full(cache.batch, -99))
    a = L.AcceptArgs()
    c = cache
    a.k_pool, a.v_pool, a.block_table, a.start_len = (x.data_ptr() for x in (d.k_pool, d.v_pool, d.table, d.lens))
    for name, x in t.items():
        setattr(a, name, x.data_ptr())
    if new_len:
        a.new_len = out.data_ptr()
    a.batch, a.kv_heads, a.nodes, a.max_path, a.head_dim, a.head_dim_value = c.batch, c.hkv, nodes, path.shape[1], c.d, c.dv
    a.block_tokens, a.max_blocks, a.num_blocks, a.dtype = c.block, c.max_blocks, c.num_blocks, CODE[c.dtype]
    L.check(L.load().sfb_k_paged_kv_accept(C.byref(a), C.c_void_p(dev.stream())))
    return dev.np(out)


@gpu
@pytest.mark.parametrize("dtype,d,dv,block,lens,nodes,plen", [
    ("bf16", 128, 128, 16, [0, 15, 31], 8, [3, 4, 0]),
    ("bf16", 64, 72, 5, [4, 9], 64, [13, 1]),
    ("f32", 20, 3, 16, [16, 2], 9, [9, 2]),
])
def test_accept_appends_the_path(dev, port, dtype, d, dv, block, lens, nodes, plen):
    rng = np.random.default_rng(1)
    cache = Cache(rng, lens, 2, d, dv, block, dtype, room=max(plen), poison=0.25, round_bf16=port.round_bf16)
    r = rounder(port, dtype)
    dk = r(rng.standard_normal((cache.batch, 2, nodes, d)).astype(np.float32))
    dvv = r(rng.standard_normal((cache.batch, 2, nodes, dv)).astype(np.float32))
    path = np.full((cache.batch, max(plen)), -5, np.int32)
    for b, n in enumerate(plen):
        path[b, :n] = np.sort(rng.permutation(nodes)[:n])
    dd = Device(dev, cache)
    status_word()
    new_len = accept_call(dev, dd, cache, nodes, path, np.array(plen), dk, dvv)
    assert status_word() == 0
    assert list(new_len) == [a + n for a, n in zip(lens, plen)]
    k_pool, v_pool = cache.k_pool.copy(), cache.v_pool.copy()
    for b, n in enumerate(plen):
        for t in range(n):
            page, slot = cache.table[b, (lens[b] + t) // block], (lens[b] + t) % block
            k_pool[page, :, slot], v_pool[page, :, slot] = dk[b, :, path[b, t]], dvv[b, :, path[b, t]]
    assert np.array_equal(dev.np(dd.k_pool), k_pool) and np.array_equal(dev.np(dd.v_pool), v_pool)


@gpu
def test_accept_skips_bad_nodes_and_positions(dev, port):
    rng = np.random.default_rng(2)
    cache = Cache(rng, [31, 20], 1, 8, 8, 16, "f32", poison=0.25)          # two blocks each: positions 0..31
    dk = rng.standard_normal((2, 1, 4, 8)).astype(np.float32)
    dd = Device(dev, cache)
    status_word()
    new_len = accept_call(dev, dd, cache, 4, np.array([[0, 1, 2], [9, 3, -1]]), np.array([7, 2]), dk, dk)
    assert status_word() & 0x200
    assert list(new_len) == [34, 22]                                          # path_len cut to 3
    k_pool = cache.k_pool.copy()
    k_pool[cache.table[0, 1], :, 15] = dk[0, :, 0]                             # position 31; 32 and 33 lie past the table
    k_pool[cache.table[1, 1], :, 5] = dk[1, :, 3]                              # node 9 skipped, node 3 at position 21
    assert np.array_equal(dev.np(dd.k_pool), k_pool)


# ---- bounds and sparse decode ----------------------------------------------------------------------------------------


def bounds_call(dev, d, bounds, start, end, max_tokens):
    c = d.cache
    s, e = dev.i32(start), dev.i32(end)
    a = L.BoundsArgs()
    a.k_pool, a.bounds, a.block_table, a.start_len, a.end_len = (x.data_ptr() for x in (d.k_pool, bounds, d.table, s, e))
    a.batch, a.kv_heads, a.head_dim, a.max_tokens = c.batch, c.hkv, c.d, max_tokens
    a.block_tokens, a.max_blocks, a.num_blocks, a.dtype = c.block, c.max_blocks, c.num_blocks, CODE[c.dtype]
    L.check(L.load().sfb_k_paged_kv_bounds(C.byref(a), C.c_void_p(dev.stream())))
    dev.torch.cuda.synchronize()


def plain_bounds(cache, lens, start):
    """{(b, block): (low, high)} of the touched blocks."""
    out = {}
    for b, n in enumerate(lens):
        for i in range(start[b] // cache.block, (n + cache.block - 1) // cache.block if n > start[b] else 0):
            k = cache.keys[b][:, i * cache.block:min(n, (i + 1) * cache.block)]
            out[b, i] = (k.min(1), k.max(1))
    return out


@gpu
@pytest.mark.parametrize("dtype,d,block,hint", [("bf16", 128, 16, 1), ("bf16", 64, 32, 400), ("f32", 33, 7, 20), ("f32", 256, 16, 3)])
def test_block_bounds(dev, port, dtype, d, block, hint):
    rng = np.random.default_rng(6)
    lens, start = [100, 0, 1, 64, 333], [0, 0, 0, 63, 40]
    cache = Cache(rng, lens, 2, d, d, block, dtype, round_bf16=port.round_bf16)
    dd = Device(dev, cache)
    bounds = dd.put(np.full((cache.num_blocks, 2, 2, d), 9.0, np.float32))
    status_word()
    bounds_call(dev, dd, bounds, start, lens, hint)
    assert status_word() == 0
    want = np.full((cache.num_blocks, 2, 2, d), 9.0)
    for (b, i), (low, high) in plain_bounds(cache, lens, start).items():
        want[cache.table[b, i], :, 0], want[cache.table[b, i], :, 1] = low, high
    assert np.array_equal(dev.np(bounds), want)


def sparse_call(dev, d, q, bounds, hq, budget, sink, recent, splits=0, scale=0.0, max_context=None, stream=None):
    c, torch = d.cache, dev.torch
    qd = d.put(q)
    out = torch.full((c.batch, hq, c.dv), 7.0, dtype=d.type, device="cuda")
    selected = torch.full((c.batch, c.hkv, budget), -77, dtype=torch.int32, device="cuda")
    a = d.fill(L.SparseArgs(), q=qd, bounds=bounds, out=out, selected=selected, q_heads=hq, budget_blocks=budget,
               sink_blocks=sink, recent_blocks=recent, splits=splits, scale=scale,
               max_context=max(1, max(c.lens)) if max_context is None else max_context)
    ws = workspace(dev, L.load().sfb_attention_sparse_workspace(C.byref(a)))
    a.workspace = ws.data_ptr()
    L.check(L.load().sfb_k_attention_decode_sparse(C.byref(a), C.c_void_p(stream if stream is not None else dev.stream())))
    return dev.np(out), dev.np(selected)


def plain_select(cache, b, h, q, budget, sink, recent):
    n = (cache.lens[b] + cache.block - 1) // cache.block
    score = []
    for i in range(n):
        k = cache.keys[b][h, i * cache.block:min(cache.lens[b], (i + 1) * cache.block)]
        score.append(np.maximum(q * k.min(0), q * k.max(0)).sum(-1).max())
    forced = set(range(min(sink, n))) | set(range(max(0, n - recent), n))
    rest = sorted((i for i in range(n) if i not in forced), key=lambda i: (-score[i], i))
    return sorted(list(forced) + rest[:max(0, min(budget, n) - len(forced))])


SPARSE_CASES = [
    # dtype, hq, hkv, d, dv, block, lens, budget, sink, recent, splits
    ("f32", 4, 2, 32, 32, 16, [0, 1, 300, 1000], 5, 1, 2, 0),
    ("f32", 6, 2, 20, 12, 4, [90, 7], 3, 0, 0, 0),
    ("f32", 9, 1, 64, 64, 16, [2000], 33, 2, 3, 4),             # nine heads share a K/V head
    ("bf16", 32, 8, 128, 128, 16, [1500, 16, 700], 20, 1, 2, 0),
    ("bf16", 8, 8, 128, 128, 16, [5000], 1, 0, 1, 0),
    ("bf16", 8, 2, 64, 64, 32, [4000, 2111], 40, 1, 4, 3),
    ("bf16", 16, 2, 128, 128, 48, [4000, 2111], 17, 0, 1, 0),
    ("bf16", 6, 2, 80, 96, 16, [500], 9, 1, 1, 0),
    ("bf16", 22, 2, 72, 72, 16, [900, 33], 9, 1, 1, 0),         # eleven heads, head_dim no multiple of 16
    ("bf16", 22, 2, 256, 64, 16, [1900], 19, 1, 1, 0),
    ("f32", 20, 2, 128, 128, 16, [3000, 100], 30, 0, 2, 0),
    ("f32", 2, 1, 256, 256, 16, [3000], 30, 0, 2, 0),
    ("f32", 8, 2, 96, 96, 8, [3000], 30, 0, 2, 0),
    ("bf16", 16, 1, 64, 64, 16, [40000], 300, 1, 4, 0),
    ("bf16", 2, 1, 16, 16, 1, [43000], 300, 1, 4, 0),             # blocks of one token, more of them than the bit mask holds
]


@gpu
@pytest.mark.parametrize("dtype,hq,hkv,d,dv,block,lens,budget,sink,recent,splits", SPARSE_CASES)
def test_sparse_decode(dev, port, dtype, hq, hkv, d, dv, block, lens, budget, sink, recent, splits):
    rng = np.random.default_rng(budget + d)
    cache = Cache(rng, lens, hkv, d, dv, block, dtype, round_bf16=port.round_bf16)
    dd = Device(dev, cache)
    bounds = dd.put(np.full((cache.num_blocks, hkv, 2, d), np.nan, np.float32))
    status_word()
    bounds_call(dev, dd, bounds, [0] * cache.batch, lens, max(lens))
    q = rounder(port, dtype)(rng.standard_normal((cache.batch, hq, d)).astype(np.float32) * 2.0)
    got, selected = sparse_call(dev, dd, q, bounds, hq, budget, sink, recent, splits)
    assert status_word() == 0
    group = hq // hkv
    for b in range(cache.batch):
        for h in range(hkv):
            qh = q[b, h * group:(h + 1) * group].astype(np.float64)
            kept = plain_select(cache, b, h, qh, budget, sink, recent)
            assert list(selected[b, h]) == kept + [-1] * (budget - len(kept)), (b, h)
            at = [t for i in kept for t in range(i * block, min(lens[b], (i + 1) * block))]
            want, bound, _ = attend(qh, cache.keys[b][h][at], cache.values[b][h][at], dtype)
            close(got[b, h * group:(h + 1) * group], want, bound)


@gpu
def test_sparse_ties_go_to_the_lower_block_and_nan_scores_rank_last(dev):
    rng = np.random.default_rng(8)
    cache = Cache(rng, [16 * 3000], 1, 8, 8, 16, "f32")
    row = rng.standard_normal((1, 1, 16, 8)).astype(np.float32)
    cache.k_pool[:] = row                                      # every block scores the same
    cache.keys[0] = np.tile(row[0], (1, 3000, 1)).astype(np.float64)
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 1, 2, 8), np.float32))
    bounds_call(dev, dd, bounds, [0], cache.lens, 48000)
    q = np.ones((1, 2, 8), np.float32)
    _, selected = sparse_call(dev, dd, q, bounds, 2, 700, 0, 1)
    assert list(selected[0, 0]) == list(range(699)) + [2999]
    nan = bounds.clone()
    nan[cache.table[0, :5].tolist()] = float("nan")
    _, selected = sparse_call(dev, dd, q, nan, 2, 700, 0, 0)
    assert list(selected[0, 0]) == list(range(5, 705))
    inf = bounds.clone()
    inf[cache.table[0, 77].item()] = float("inf")
    inf[cache.table[0, 78].item()] = float("-inf")
    _, selected = sparse_call(dev, dd, q, inf, 2, 2, 0, 0)
    assert list(selected[0, 0]) == [0, 77]
    _, selected = sparse_call(dev, dd, q, inf, 2, 2999, 0, 0)
    assert list(selected[0, 0]) == [i for i in range(3000) if i != 78]
    _, selected = sparse_call(dev, dd, 0.0 * q, bounds, 2, 5, 1, 1)     # a query of zeros: every score is zero
    assert list(selected[0, 0]) == [0, 1, 2, 3, 2999]


@gpu
@pytest.mark.parametrize("dtype,d", [("f32", 32), ("f32", 20), ("bf16", 64)])
@pytest.mark.parametrize("q_size,k_size", [(2.0 ** -70, 2.0 ** -70), (2.0 ** 80, 2.0 ** 50), (2.0 ** -75, 1.0), (1.0, 2.0 ** 100)])
def test_sparse_ranks_scores_outside_the_range_of_float32_by_their_64_bit_sums(dev, port, dtype, d, q_size, k_size):
    """Products that vanish or overflow in 32 bits (keys are equal within a block, so sums cancel)."""
    rng = np.random.default_rng(d)
    cache = Cache(rng, [16 * 60], 1, d, d, 16, dtype, round_bf16=port.round_bf16)
    for i in range(60):
        row = cache.keys[0][:, 16 * i:16 * i + 1] * k_size
        cache.keys[0][:, 16 * i:16 * i + 16] = row
        cache.k_pool[cache.table[0, i]] = row
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 1, 2, d), np.float32))
    bounds_call(dev, dd, bounds, [0], cache.lens, 960)
    q = rounder(port, dtype)(rng.standard_normal((1, 3, d)).astype(np.float32)) * np.float32(q_size)
    for budget, sink, recent in ((7, 1, 1), (1, 0, 0), (59, 0, 3)):
        _, selected = sparse_call(dev, dd, q, bounds, 3, budget, sink, recent)
        assert list(selected[0, 0]) == plain_select(cache, 0, 0, q[0].astype(np.float64), budget, sink, recent)


@gpu
@pytest.mark.parametrize("dtype,d", [("f32", 32), ("f32", 20), ("bf16", 64)])
def test_sparse_ignores_an_element_whose_query_is_zero(dev, port, dtype, d):
    """A block whose keys are all NaN in one element has low = inf and high = -inf there."""
    rng = np.random.default_rng(d)
    cache = Cache(rng, [16 * 60], 1, d, d, 16, dtype, round_bf16=port.round_bf16)
    q = rounder(port, dtype)(rng.standard_normal((1, 3, d)).astype(np.float32))
    q[:, :, 5] = 0.0
    want = plain_select(cache, 0, 0, q[0].astype(np.float64), 9, 0, 0)
    for i in range(0, 60, 3):
        cache.k_pool[cache.table[0, i], :, :, 5] = np.nan
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 1, 2, d), np.float32))
    bounds_call(dev, dd, bounds, [0], cache.lens, 960)
    _, selected = sparse_call(dev, dd, q, bounds, 3, 9, 0, 0)
    assert list(selected[0, 0]) == want
    q[:, 1, 5] = 1.0                                          # now such a block's second head has no upper bound but -inf
    q[:, 0], q[:, 2] = q[:, 1], q[:, 1]
    _, selected = sparse_call(dev, dd, q, bounds, 3, 40, 0, 0)
    assert list(selected[0, 0]) == [i for i in range(60) if i % 3]


@gpu
@pytest.mark.parametrize("blocks,block", [(3000, 16), (300, 16), (43000, 1)])
def test_sparse_bf16_ties_go_to_the_lower_block_and_infinite_scores_count(dev, blocks, block):
    rng = np.random.default_rng(blocks)
    cache = Cache(rng, [block * blocks], 1, 16, 16, block, "f32")
    cache.dtype = "bf16"
    row = np.exp2(rng.integers(-3, 4, (1, 1, 1, 16))).astype(np.float32)
    cache.k_pool[:] = row                                      # every block scores the same
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 1, 2, 16), np.float32))
    bounds_call(dev, dd, bounds, [0], cache.lens, block * blocks)
    q = np.ones((1, 2, 16), np.float32)
    _, selected = sparse_call(dev, dd, q, bounds, 2, 250, 0, 1)
    assert list(selected[0, 0]) == list(range(249)) + [blocks - 1]
    inf = bounds.clone()
    inf[cache.table[0, 77].item()] = float("inf")
    inf[cache.table[0, 78].item()] = float("-inf")
    _, selected = sparse_call(dev, dd, q, inf, 2, 2, 0, 0)
    assert list(selected[0, 0]) == [0, 77]
    _, selected = sparse_call(dev, dd, q, inf, 2, blocks - 1, 0, 0)
    assert list(selected[0, 0]) == [i for i in range(blocks) if i != 78]
    _, selected = sparse_call(dev, dd, 0.0 * q, bounds, 2, 5, 1, 1)
    assert list(selected[0, 0]) == [0, 1, 2, 3, blocks - 1]


@gpu
def test_sparse_bad_lengths_and_blocks(dev, port):
    rng = np.random.default_rng(9)
    cache = Cache(rng, [320, 320, 320], 2, 64, 64, 16, "bf16", round_bf16=port.round_bf16)
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 2, 2, 64), np.float32))
    bounds_call(dev, dd, bounds, [0] * 3, cache.lens, 320)
    q = port.round_bf16(rng.standard_normal((3, 4, 64)).astype(np.float32))
    good, chosen = sparse_call(dev, dd, q, bounds, 4, 6, 1, 1)
    status_word()
    dd.lens = dev.i32(np.array([320, 9999, -1]))
    got, selected = sparse_call(dev, dd, q, bounds, 4, 6, 1, 1, max_context=320)
    assert status_word() & 0x200
    assert np.array_equal(got[:2], good[:2]) and np.array_equal(selected[:2], chosen[:2])
    assert np.all(got[2] == 0.0) and np.all(selected[2] == -1)
    dd.lens = dev.i32(np.array(cache.lens))
    cache.table[0, 3] = -1                                    # ranks last, and its positions are masked if kept
    dd.table = dev.i32(cache.table)
    got, selected = sparse_call(dev, dd, q, bounds, 4, 20, 0, 0)
    assert status_word() & 0x200
    at = np.r_[0:48, 64:320]
    for h in range(4):
        want, bound, _ = attend(q[0, h:h + 1].astype(np.float64), cache.keys[0][h // 2][at], cache.values[0][h // 2][at], "bf16")
        close(got[0, h:h + 1], want, bound)


# ---- accumulated weights -----------------------------------------------------------------------------------------------


def weights_call(dev, d, q, hq, weights, weights_out, stride, positions=None, query_position=None, splits=0, max_context=None,
                 stream=None):
    c, torch = d.cache, dev.torch
    qd = d.put(q)
    out = torch.full((c.batch, hq, c.dv), 7.0, dtype=d.type, device="cuda")
    a = d.fill(L.WeightsArgs(), q=qd, out=out, weights_out=weights_out, q_heads=hq, weight_stride=stride, splits=splits,
               max_context=max(1, max(c.lens)) if max_context is None else max_context)
    if weights is not None:
        a.weights = weights.data_ptr()
    if positions is not None:
        a.positions, a.query_position = positions.data_ptr(), query_position.data_ptr()
    ws = workspace(dev, L.load().sfb_attention_weights_workspace(C.byref(a)))
    a.workspace = ws.data_ptr()
    L.check(L.load().sfb_k_attention_decode_weights(C.byref(a), C.c_void_p(stream if stream is not None else dev.stream())))
    return dev.np(out)


@gpu
@pytest.mark.parametrize("dtype,hq,hkv,d,dv,block,lens,splits", [
    ("f32", 4, 2, 32, 32, 16, [0, 1, 300, 77], 0),
    ("f32", 6, 2, 20, 12, 4, [90, 7], 3),
    ("f32", 12, 1, 64, 64, 16, [1300], 1),
    ("bf16", 32, 8, 128, 128, 16, [1500, 16, 0, 700], 0),
    ("bf16", 8, 8, 128, 128, 32, [2050], 5),
    ("bf16", 14, 2, 64, 64, 16, [1100, 63], 2),
    ("bf16", 32, 1, 128, 128, 16, [500], 0),
    ("bf16", 4, 2, 80, 96, 16, [100, 2], 0),
])
def test_decode_with_weights(dev, port, dtype, hq, hkv, d, dv, block, lens, splits):
    rng = np.random.default_rng(d + hq)
    cache = Cache(rng, lens, hkv, d, dv, block, dtype, round_bf16=port.round_bf16)
    dd = Device(dev, cache)
    q = rounder(port, dtype)(rng.standard_normal((cache.batch, hq, d)).astype(np.float32) * 1.5)
    stride = max(lens) + 5
    before = rng.random((cache.batch, hkv, stride)).astype(np.float32)
    torch = dev.torch
    separate = dev.f32(np.full_like(before, 3.5))
    same = dev.f32(before)
    fresh = dev.f32(np.full_like(before, 3.5))
    positions = dev.i32(np.full(before.shape, -4))
    query_position = dev.i32(np.arange(cache.batch) + 1000)
    status_word()
    source = dev.f32(before)
    got = weights_call(dev, dd, q, hq, source, separate, stride, positions, query_position, splits)
    again = weights_call(dev, dd, q, hq, same, same, stride, splits=splits)
    third = weights_call(dev, dd, q, hq, None, fresh, stride, splits=splits)
    assert status_word() == 0
    assert np.array_equal(got, again) and np.array_equal(got, third)
    w_sep, w_same, w_fresh, pos = dev.np(separate), dev.np(same), dev.np(fresh), dev.np(positions)
    group = hq // hkv
    for b, n in enumerate(lens):
        assert np.all(w_sep[b, :, n:] == 3.5) and np.array_equal(w_same[b, :, n:], before[b, :, n:])
        want_pos = np.full((hkv, stride), -4)
        if n:
            want_pos[:, n - 1] = 1000 + b
        assert np.array_equal(pos[b], want_pos)
        for h in range(hkv):
            qh = q[b, h * group:(h + 1) * group].astype(np.float64)
            want, bound, p = attend(qh, cache.keys[b][h], cache.values[b][h], dtype)
            close(got[b, h * group:(h + 1) * group], want, bound)
            if n == 0:
                continue
            # a weight: twice the logit's error, the exponential and the row sum, then `group` + 1 additions in 32 bits
            logit = (d + 4) * 2.0 ** -24 * (np.abs(qh) @ np.abs(cache.keys[b][h]).T).max() / np.sqrt(d)
            rel = 2.0 * logit + 2.0 ** -20 + n * 2.0 ** -24
            total = p.sum(0)
            close(w_fresh[b, h, :n], total, total * rel + (group + 2) * 2.0 ** -24 * total + 1e-30)
            added = before[b, h, :n].astype(np.float64) + total
            close(w_sep[b, h, :n], added, total * rel + (group + 3) * 2.0 ** -24 * added)
            assert np.array_equal(w_sep[b, h, :n], w_same[b, h, :n])


# ---- eviction ------------------------------------------------------------------------------------------------------------


def evict_call(dev, d, weights, weights_out, positions, positions_out, new_len, stride, budget, sink, recent, max_context=None):
    c = d.cache
    a = d.fill(L.EvictArgs(), weights=weights, weights_out=weights_out, positions=positions, positions_out=positions_out,
               new_len=new_len, weight_stride=stride, budget=budget, sink_tokens=sink, recent_tokens=recent,
               max_context=max(1, max(c.lens)) if max_context is None else max_context)
    ws = workspace(dev, L.load().sfb_paged_kv_evict_workspace(C.byref(a)))
    a.workspace = ws.data_ptr()
    L.check(L.load().sfb_k_paged_kv_evict(C.byref(a), C.c_void_p(dev.stream())))
    dev.torch.cuda.synchronize()


def plain_evict(weights, positions, n, budget, sink, recent):
    """(kept slot of every new slot) of one row."""
    k = min(n, budget)
    if k == 0:
        return []
    newest = positions[:n].max()
    rank = []
    for i in range(n):
        safe = positions[i] < sink or positions[i] > newest - recent
        w = weights[i]
        rank.append((0 if safe else 1, 0.0 if safe else (np.inf if np.isnan(w) else -float(w)), 1 if not safe and np.isnan(w) else 0, i))
    kept = set(i for *_, i in sorted(rank)[:k])
    source = list(range(k))
    for to, since in zip([i for i in range(k) if i not in kept], [i for i in range(k, n) if i in kept]):
        source[to] = since
    return source


@gpu
@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("dtype,hkv,d,dv,block,lens,budget,sink,recent", [
    ("f32", 2, 32, 32, 16, [0, 1, 300, 77, 64], 64, 4, 8),
    ("f32", 1, 20, 3, 4, [90, 7, 10], 9, 0, 0),
    ("bf16", 8, 128, 128, 16, [513, 2049, 512], 512, 4, 64),
    ("bf16", 2, 64, 64, 32, [5000, 4097], 4096, 0, 4096),       # everything kept is recent
    ("bf16", 1, 80, 7, 16, [100], 1000, 1, 1),                   # nothing leaves
    ("f32", 3, 8, 8, 16, [3000], 1, 1, 0),                       # all but one leave
    ("f32", 1, 8, 8, 64, [50000, 41000], 20000, 3, 100),         # rows too long for the bit mask
])
def test_evict(dev, port, alias, dtype, hkv, d, dv, block, lens, budget, sink, recent):
    rng = np.random.default_rng(budget)
    cache = Cache(rng, lens, hkv, d, dv, block, dtype, poison=0.25, round_bf16=port.round_bf16)
    stride = max(lens) + 3
    weights = np.exp(2.0 * rng.standard_normal((cache.batch, hkv, stride))).astype(np.float32)
    weights[:, :, ::3] = 0.5                                      # many ties
    weights[:, :, 1::7] = 0.0
    weights[:, :, 5::11] = -0.0
    weights[:, :, 2::13] = np.nan
    weights[:, :, 6::17] = np.inf
    positions = np.full((cache.batch, hkv, stride), 1 << 20, np.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            positions[b, h, :n] = rng.permutation(2 * n)[:n]       # out of order, with gaps
    dd = Device(dev, cache)
    w, p = dev.f32(weights), dev.i32(positions)
    w_out, p_out = (w, p) if alias else (dev.f32(np.full_like(weights, 3.5)), dev.i32(np.full_like(positions, 33)))
    new_len = dd.lens if alias else dev.i32(np.full(cache.batch, -9))
    status_word()
    evict_call(dev, dd, w, w_out, p, p_out, new_len, stride, budget, sink, recent)
    assert status_word() == 0
    assert list(dev.np(new_len)) == [min(n, budget) for n in lens]
    got_w, got_p, k_pool, v_pool = dev.np(w_out), dev.np(p_out), dev.np(dd.k_pool), dev.np(dd.v_pool)
    for b, n in enumerate(lens):
        k = min(n, budget)
        new_k, new_v = cache.rows(k_pool, b, n), cache.rows(v_pool, b, n)
        for h in range(hkv):
            source = plain_evict(weights[b, h], positions[b, h], n, budget, sink, recent)
            assert np.array_equal(got_w[b, h, :k], weights[b, h][source], equal_nan=True)
            assert np.array_equal(got_p[b, h, :k], positions[b, h][source])
            assert np.all(got_w[b, h, k:n] == 0.0) and np.all(got_p[b, h, k:n] == -1)
            behind_w, behind_p = (weights, positions) if alias else (np.full_like(weights, 3.5), np.full_like(positions, 33))
            assert np.array_equal(got_w[b, h, n:], behind_w[b, h, n:], equal_nan=True)
            assert np.array_equal(got_p[b, h, n:], behind_p[b, h, n:])
            assert np.array_equal(new_k[h, :k], cache.keys[b][h][source]) and np.array_equal(new_v[h, :k], cache.values[b][h][source])
            assert np.array_equal(new_k[h, k:], cache.keys[b][h][k:]) and np.array_equal(new_v[h, k:], cache.values[b][h][k:])
    used = set(int(t) for b, n in enumerate(lens) for t in cache.table[b, : (n + block - 1) // block])
    for page in set(range(cache.num_blocks)) - used:
        assert np.all(k_pool[page] == 0.25)


@gpu
@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("kind", ["distinct", "few values", "equal"])
@pytest.mark.parametrize("hkv,lens,budget,sink,recent", [
    (2, [16384, 0, 5, 12001, 4097], 2048, 4, 256),
    (1, [40960, 33], 20000, 3, 100),                             # the longest row that a bit mask holds
    (3, [5000], 1, 1, 0),
    (1, [8191, 4100], 8190, 0, 8190),                            # everything kept is recent, or one leaves
    (8, [4200, 4133, 9000, 300], 4100, 64, 0),
    (1, [16385, 16384], 16383, 2, 16000),                        # where a cluster takes over
    (2, [65543, 90, 40961], 30000, 4, 30),
    (1, [163840, 163839], 2048, 4, 256),                         # the longest rows of a cluster
    (1, [163841, 20], 100000, 4, 256),                           # and longer ones
])
def test_evict_long_rows(dev, alias, kind, hkv, lens, budget, sink, recent):
    rng = np.random.default_rng(budget + hkv)
    cache = Cache(rng, lens, hkv, 4, 4, 16, "f32", poison=0.25)
    stride = max(lens) + 5
    shape = (cache.batch, hkv, stride)
    weights = {"distinct": rng.permutation(np.prod(shape)).reshape(shape), "few values": rng.integers(0, 40, shape),
               "equal": np.full(shape, 3)}[kind].astype(np.float32)
    positions = np.full(shape, 1 << 20, np.int32)
    for b, n in enumerate(lens):
        for h in range(hkv):
            positions[b, h, :n] = np.arange(n)
    positions[-1, 0, :min(lens[-1], 7)] = 0                       # positions that repeat
    dd = Device(dev, cache)
    w, p = dev.f32(weights), dev.i32(positions)
    w_out, p_out = (w, p) if alias else (dev.f32(np.full_like(weights, 3.5)), dev.i32(np.full_like(positions, 33)))
    new_len = dev.i32(np.full(cache.batch, -9))
    status_word()
    evict_call(dev, dd, w, w_out, p, p_out, new_len, stride, budget, sink, recent)
    assert status_word() == 0
    assert list(dev.np(new_len)) == [min(n, budget) for n in lens]
    got_w, got_p, k_pool = dev.np(w_out), dev.np(p_out), dev.np(dd.k_pool)
    for b, n in enumerate(lens):
        k = min(n, budget)
        new_k = cache.rows(k_pool, b, n)
        for h in range(hkv):
            source = plain_evict(weights[b, h], positions[b, h], n, budget, sink, recent)
            assert np.array_equal(got_w[b, h, :k], weights[b, h][source])
            assert np.array_equal(got_p[b, h, :k], positions[b, h][source])
            assert np.all(got_w[b, h, k:n] == 0.0) and np.all(got_p[b, h, k:n] == -1)
            assert np.array_equal(new_k[h, :k], cache.keys[b][h][source])


# ---- refusals (no device needed) -------------------------------------------------------------------------------------------


def valid_args(kind):
    """Arguments that pass every check, with host addresses that nothing follows."""
    a = {"tree": L.TreeArgs, "accept": L.AcceptArgs, "bounds": L.BoundsArgs, "sparse": L.SparseArgs, "weights": L.WeightsArgs,
         "evict": L.EvictArgs}[kind]()
    at = 1 << 20
    for name, kind_of in a._fields_:
        if kind_of is L.vp:
            setattr(a, name, at)
            at += 1 << 20
        elif kind_of is C.c_int:
            setattr(a, name, 2)
    a.dtype = L.BF16
    a.kv_heads, a.head_dim = 1, 64
    if hasattr(a, "splits"):
        a.splits = 0
    if kind != "bounds":
        a.head_dim_value = 64
    if hasattr(a, "max_context"):
        a.max_context = 20
    a.block_tokens, a.max_blocks, a.num_blocks = 16, 4, 9
    if hasattr(a, "weight_stride"):
        a.weight_stride = 64
    if kind == "sparse":
        a.budget_blocks, a.sink_blocks, a.recent_blocks = 4, 1, 1
    if kind == "evict":
        a.budget, a.sink_tokens, a.recent_tokens = 16, 4, 4
    return a


CALLS = {"tree": "sfb_k_attention_tree_paged", "accept": "sfb_k_paged_kv_accept", "bounds": "sfb_k_paged_kv_bounds",
         "sparse": "sfb_k_attention_decode_sparse", "weights": "sfb_k_attention_decode_weights", "evict": "sfb_k_paged_kv_evict"}
SHAPES = [("batch", 0), ("batch", -1), ("kv_heads", 0), ("head_dim", 0), ("block_tokens", 0), ("max_blocks", -3),
          ("num_blocks", 0), ("dtype", 2)]
REFUSED = [(kind, *change, L.SFB_INVALID_ARGUMENT) for kind in CALLS for change in SHAPES] + \
          [(kind, "head_dim", 257, L.SFB_UNSUPPORTED) for kind in CALLS] + \
          [(kind, "block_tokens", 1 << 29, L.SFB_UNSUPPORTED) for kind in CALLS] + \
          [(kind, "batch", 65536, L.SFB_UNSUPPORTED) for kind in CALLS] + \
          [(kind, "block_table", 0, L.SFB_INVALID_ARGUMENT) for kind in CALLS] + \
          [(kind, "workspace", 8 + (1 << 22), L.SFB_INVALID_ARGUMENT) for kind in ("sparse", "weights", "evict")] + \
          [(kind, "workspace", 0, L.SFB_INVALID_ARGUMENT) for kind in ("sparse", "weights", "evict")] + \
          [(kind, "kv_heads", 3, L.SFB_INVALID_ARGUMENT) for kind in ("tree", "sparse", "weights")] + [
    ("tree", "nodes", 0, L.SFB_INVALID_ARGUMENT), ("tree", "nodes", 257, L.SFB_UNSUPPORTED),
    ("tree", "max_context", -1, L.SFB_INVALID_ARGUMENT), ("tree", "parents", 0, L.SFB_INVALID_ARGUMENT),
    ("tree", "out", 0, L.SFB_INVALID_ARGUMENT), ("tree", "head_dim_value", 300, L.SFB_UNSUPPORTED),
    ("accept", "nodes", 0, L.SFB_INVALID_ARGUMENT), ("accept", "max_path", 0, L.SFB_INVALID_ARGUMENT),
    ("accept", "path_len", 0, L.SFB_INVALID_ARGUMENT),
    ("bounds", "max_tokens", 0, L.SFB_INVALID_ARGUMENT), ("bounds", "bounds", 0, L.SFB_INVALID_ARGUMENT),
    ("sparse", "budget_blocks", 0, L.SFB_INVALID_ARGUMENT), ("sparse", "sink_blocks", -1, L.SFB_INVALID_ARGUMENT),
    ("sparse", "recent_blocks", 4, L.SFB_INVALID_ARGUMENT), ("sparse", "max_context", 0, L.SFB_INVALID_ARGUMENT),
    ("sparse", "selected", 0, L.SFB_INVALID_ARGUMENT),
    ("weights", "max_context", 0, L.SFB_INVALID_ARGUMENT), ("weights", "weight_stride", 19, L.SFB_INVALID_ARGUMENT),
    ("weights", "query_position", 0, L.SFB_INVALID_ARGUMENT), ("weights", "weights_out", 0, L.SFB_INVALID_ARGUMENT),
    ("evict", "budget", 0, L.SFB_INVALID_ARGUMENT), ("evict", "sink_tokens", 13, L.SFB_INVALID_ARGUMENT),
    ("evict", "recent_tokens", -1, L.SFB_INVALID_ARGUMENT), ("evict", "weight_stride", 3, L.SFB_INVALID_ARGUMENT),
    ("evict", "positions", 0, L.SFB_INVALID_ARGUMENT),
]


@pytest.mark.parametrize("kind,field,value,status", REFUSED)
def test_refusals(sfb, kind, field, value, status):
    a = valid_args(kind)
    setattr(a, field, value or None if field in ("block_table", "workspace", "parents", "out", "path_len", "bounds", "selected",
                                                 "query_position", "weights_out", "positions") else value)
    assert getattr(sfb.load(), CALLS[kind])(C.byref(a), None) == status
    assert len(sfb.load().sfb_last_error()) > 0


@pytest.mark.parametrize("kind", list(CALLS))
def test_null_arguments_are_refused(sfb, kind):
    assert getattr(sfb.load(), CALLS[kind])(None, None) == L.SFB_INVALID_ARGUMENT


def test_accept_refuses_new_len_over_start_len(sfb):
    a = valid_args("accept")
    a.new_len = a.start_len
    assert sfb.load().sfb_k_paged_kv_accept(C.byref(a), None) == L.SFB_INVALID_ARGUMENT


def test_workspace_sizes_need_no_device(sfb):
    lib = sfb.load()
    a = valid_args("evict")
    a.max_context = 20
    assert lib.sfb_paged_kv_evict_workspace(C.byref(a)) == 80 + 2 * 20     # 20 - 16 rows may move: 9 words a head; one byte a position
    a.budget = 1000
    assert lib.sfb_paged_kv_evict_workspace(C.byref(a)) == 16 + 2 * 20
    w = valid_args("weights")
    w.splits, w.dtype = 1, L.F32
    assert lib.sfb_attention_weights_workspace(C.byref(w)) == 2 * 2 * 66 * 4 + 2 * 2 * 20 * 4
    s = valid_args("sparse")
    s.splits, s.dtype = 1, L.F32
    assert lib.sfb_attention_sparse_workspace(C.byref(s)) == 2 * 2 * 8 + 16 + 16 + 2 * 2 * 66 * 4   # exact, 32-bit, sizes, partials
    s.q_heads = 3
    s.kv_heads = 2
    assert lib.sfb_attention_sparse_workspace(C.byref(s)) == 0                          # refused arguments
    t = valid_args("tree")
    t.splits, t.dtype = 1, L.F32
    assert lib.sfb_attention_tree_workspace(C.byref(t)) == 0                            # no partial results to keep


def test_struct_sizes(sfb):
    assert C.sizeof(sfb.TreeArgs) == 11 * 8 + 14 * 4
    assert C.sizeof(sfb.AcceptArgs) == 9 * 8 + 10 * 4
    assert C.sizeof(sfb.BoundsArgs) == 5 * 8 + 8 * 4
    assert C.sizeof(sfb.SparseArgs) == 9 * 8 + 16 * 4      # 15 members of 4 bytes, padded
    assert C.sizeof(sfb.WeightsArgs) == 11 * 8 + 14 * 4    # 13, padded
    assert C.sizeof(sfb.EvictArgs) == 10 * 8 + 14 * 4      # 13, padded
