"""The serving operators as a program uses them: PagedKVCache's host calls in a row (draft, verify, accept, sparse and
tracked decode, eviction), captured graphs, several streams, pools beyond 2^31 elements."""
import ctypes as C
from types import SimpleNamespace

import numpy as np
import pytest

from cache_problem import Cache, ancestors, attend
from schedforge_b200 import api, lib as L
from test_cache_ops import (CODE, Device, accept_call, bounds_call, close, evict_call, rounder, sparse_call, status_word, tree_call,
                            tree_check, tree_inputs, weights_call, workspace)

pytestmark = pytest.mark.gpu


def check_rows(got, q, keys, values, dtype, hidden=None):
    """got, q [B, Hq, n, D]; keys, values [B, Hkv, m, D]."""
    group = q.shape[1] // keys.shape[1]
    for b in range(q.shape[0]):
        for h in range(q.shape[1]):
            want, bound, _ = attend(q[b, h].astype(np.float64), keys[b, h // group].astype(np.float64),
                                    values[b, h // group].astype(np.float64), dtype, 0.0, None if hidden is None else hidden[b])
            close(got[b, h], want, bound)


@pytest.mark.parametrize("dtype,d,page", [("bf16", 128, 16), ("bf16", 64, 32), ("f32", 64, 16), ("f32", 24, 5)])
def test_host_cache_from_draft_to_eviction(port, dtype, d, page):
    rng = np.random.default_rng(d)
    r = rounder(port, dtype)
    batch, hq, hkv, capacity = 2, 8, 2, 700
    cache = api.PagedKVCache(batch, hkv, d, d, page, capacity, dtype=CODE[dtype])
    keys, values = (r(rng.standard_normal((batch, hkv, 0, d)).astype(np.float32)) for _ in range(2))

    def fresh(n):
        return (r(rng.standard_normal((batch, hkv, n, d)).astype(np.float32)) for _ in range(2))

    # a first tree over the empty cache, then over a prompt
    for prompt in (0, 400):
        if prompt:
            k, v = fresh(prompt)
            cache.append(k, v, prompt)
            keys, values = np.concatenate([keys, k], 2), np.concatenate([values, v], 2)
        n = keys.shape[2]
        nodes = 7
        q = r(rng.standard_normal((batch, hq, nodes, d)).astype(np.float32))
        dk, dv = fresh(nodes)
        parents = np.array([[-1, 0, 0, 1, 3, -1, 5], [-1, -1, 1, 2, 3, 4, 5]], np.int32)
        config = api.attention_config(batch, hq, hkv, nodes, max(n, 1), d)
        out, ms = cache.decode_tree(config, q, dk, dv, parents)
        assert ms >= 0.0
        hidden = [np.concatenate([np.zeros((nodes, n), bool), ~ancestors(p, nodes)], 1) for p in parents]
        check_rows(out, q, np.concatenate([keys, dk], 2), np.concatenate([values, dv], 2), dtype, hidden)
        # one branch of each tree is accepted
        path = np.array([[0, 1, 3, 4], [1, 2, 3, 4]], np.int32)
        cache.accept(dk, dv, path)
        pick = path[:, None, :, None]
        keys = np.concatenate([keys, np.take_along_axis(dk, np.broadcast_to(pick, (batch, hkv, 4, d)), 2)], 2)
        values = np.concatenate([values, np.take_along_axis(dv, np.broadcast_to(pick, (batch, hkv, 4, d)), 2)], 2)
        gk, gv = cache.gather()
        assert np.array_equal(gk, keys) and np.array_equal(gv, values)
    n = keys.shape[2]
    one = api.attention_config(batch, hq, hkv, 1, capacity, d)
    pages = (n + page - 1) // page
    # sparse decode over all pages is decode; over some, it is attention over those
    q = r(rng.standard_normal((batch, hq, 1, d)).astype(np.float32) * 1.5)
    out, selected, _ = cache.decode_sparse(one, q, pages + 3, 1, 1)
    assert np.array_equal(selected, np.broadcast_to(np.r_[0:pages, [-1] * 3], selected.shape))
    check_rows(out, q, keys, values, dtype)
    for grow in (0, 1):      # the bounds of the page a new token falls into follow
        if grow:
            k, v = fresh(1)
            cache.append(k * 3, v, 1)
            keys, values = np.concatenate([keys, r(k * 3)], 2), np.concatenate([values, v], 2)
            n += 1
        out, selected, _ = cache.decode_sparse(one, q, 6, 1, 2)
        live = (n + page - 1) // page
        for b in range(batch):
            for h in range(hkv):
                qh = q[b, h * 4:h * 4 + 4, 0].astype(np.float64)
                blocks = [keys[b, h, i * page:min(n, (i + 1) * page)].astype(np.float64) for i in range(live)]
                score = [np.maximum(qh * x.min(0), qh * x.max(0)).sum(-1).max() for x in blocks]
                rest = sorted(range(1, live - 2), key=lambda i: (-score[i], i))[:3]
                kept = sorted([0, live - 2, live - 1] + rest)
                assert list(selected[b, h]) == kept
                at = [t for i in kept for t in range(i * page, min(n, (i + 1) * page))]
                want, bound, _ = attend(qh, keys[b, h][at].astype(np.float64), values[b, h][at].astype(np.float64), dtype)
                close(out[b, h * 4:h * 4 + 4, 0], want, bound)
    with pytest.raises(L.InvalidArgument, match="no accumulated attention weights"):
        cache.evict(100)
    # tracked decode: the same output, and weights that add up to one per query head and step
    for step in range(3):
        if step:
            k, v = fresh(1)
            cache.append(k, v, 1)
            keys, values = np.concatenate([keys, k], 2), np.concatenate([values, v], 2)
        out, _ = cache.decode_tracked(one, q)
        check_rows(out, q, keys, values, dtype)
    n = keys.shape[2]
    weights, positions = cache.weights()
    assert np.allclose(weights.sum(-1), 3 * hq // hkv, rtol=1e-5)
    assert np.array_equal(positions, np.broadcast_to(np.arange(n), positions.shape))
    # eviction down to a budget: pages come back, rows and weights stay together, decode sees the kept ones
    budget = 128
    before = cache.info()
    cache.evict(budget, 4, 16)
    info = cache.info()
    assert info["length"] == budget and len(info["page_table"]) == (budget + page - 1) // page
    assert len(info["page_table"]) + len(info["free_pages"]) == len(before["page_table"]) + len(before["free_pages"])
    kept_w, kept_p = cache.weights()
    gk, gv = cache.gather()
    for b in range(batch):
        for h in range(hkv):
            p = kept_p[b, h]
            assert len(set(p)) == budget and set(range(4)) <= set(p) and set(range(n - 16, n)) <= set(p)
            assert np.array_equal(kept_w[b, h], weights[b, h][p])
            assert np.array_equal(gk[b, h], keys[b, h][p]) and np.array_equal(gv[b, h], values[b, h][p])
            middle = [i for i in p if 4 <= i < n - 16]
            left = np.setdiff1d(np.arange(4, n - 16), middle)
            assert weights[b, h][middle].min() >= weights[b, h][left].max()
    out, _ = cache.decode(one, q)
    check_rows(out, q, gk, gv, dtype)
    # the next tokens continue the text positions; a cache within the budget stays as it is
    k, v = fresh(2)
    cache.append(k, v, 2)
    _, positions = cache.weights()
    assert np.all(positions[:, :, budget:] == np.array([n, n + 1]))
    cache.evict(budget + 2, 0, 0)
    assert cache.info()["length"] == budget + 2
    out, selected, _ = cache.decode_sparse(one, q, 1000, 0, 0)
    check_rows(out, q, np.concatenate([gk, k], 2), np.concatenate([gv, v], 2), dtype)
    cache.evict(1, 0, 1)
    assert np.array_equal(cache.weights()[1], np.full((batch, hkv, 1), n + 1))
    cache.close()


def test_host_cache_refusals():
    cache = api.PagedKVCache(1, 2, 16, 16, 4, 12, dtype=L.F32)
    z = np.zeros((1, 2, 3, 16), np.float32)
    q = np.zeros((1, 4, 3, 16), np.float32)
    tree = api.attention_config(1, 4, 2, 3, 12, 16)
    with pytest.raises(L.InvalidArgument, match="parent has to come before"):
        cache.decode_tree(tree, q, z, z, np.array([[-1, 1, 0]]))
    with pytest.raises(ValueError):
        cache.decode_tree(tree, q, z, z, np.array([[-1, 0]]))
    with pytest.raises(L.InvalidArgument, match="paged KV shape violates compiled guard"):
        cache.decode_tree(api.attention_config(1, 4, 1, 3, 12, 16), q, z, z, np.array([[-1, 0, 0]]))
    with pytest.raises(L.InvalidArgument, match="not in the tree"):
        cache.accept(z, z, np.array([[0, 3]]))
    with pytest.raises(L.InvalidArgument, match="paged KV capacity exceeded"):
        cache.accept(z, z, np.zeros((1, 13), np.int32))
    one = api.attention_config(1, 4, 2, 1, 12, 16)
    with pytest.raises(L.InvalidArgument, match="paged KV length violates compiled guard"):
        cache.decode_sparse(one, q[:, :, :1], 4)          # empty cache
    cache.append(z, z, 3)
    with pytest.raises(L.InvalidArgument, match="have to fit into the budget"):
        cache.decode_sparse(one, q[:, :, :1], 1, 1, 1)
    with pytest.raises(L.InvalidArgument, match="one query token"):
        cache.decode_tracked(tree, q)
    with pytest.raises(L.InvalidArgument, match="no accumulated"):
        cache.weights()
    cache.decode_tracked(one, q[:, :, :1])
    with pytest.raises(L.InvalidArgument, match="have to fit into the budget"):
        cache.evict(2, 2, 1)


# ---- graphs and streams --------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64)])
def test_a_step_captured_in_a_graph_follows_its_inputs(dev, port, dtype, d):
    """Tree, accept, bounds, sparse decode, weights and eviction captured once; replayed after the lengths, the queries
    and the tree have changed in place, the graph gives what direct calls give."""
    torch = dev.torch
    rng = np.random.default_rng(11)
    lens, nodes, hq, hkv, budget = [400, 123], 9, 8, 2, 100
    cache = Cache(rng, lens, hkv, d, d, 16, dtype, room=32, poison=0.5, round_bf16=port.round_bf16)
    r = rounder(port, dtype)
    stride, max_context = 448, 432
    lib = L.load()

    def inputs(seed):
        g = np.random.default_rng(seed)
        q, dk, dv, parents = tree_inputs(g, port, cache, hq, nodes, [nodes] * 2)
        return dict(q=q, dk=dk, dv=dv, parents=parents, path=np.sort(np.stack([g.permutation(nodes)[:4] for _ in range(2)])),
                    path_len=g.integers(0, 5, 2), q1=r(g.standard_normal((2, hq, d)).astype(np.float32)),
                    len=np.array(lens) if seed == 0 else np.array([333, 41]))

    class Step:
        def __init__(self):
            self.d = Device(dev, cache)
            x = inputs(0)
            self.t = {k: (self.d.put(v) if v.dtype == np.float32 else dev.i32(v)) for k, v in x.items()}
            z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")
            i32 = torch.int32
            self.out, self.out1, self.out2 = (torch.zeros(s, dtype=self.d.type, device="cuda") for s in ((2, hq, nodes, d), (2, hq, d), (2, hq, d)))
            self.new_len, self.cut_len = z(2, t=i32), z(2, t=i32)
            self.bounds = self.d.put(np.zeros((cache.num_blocks, hkv, 2, d), np.float32))
            self.selected = z(2, hkv, 6, t=i32)
            self.weights, self.positions = z(2, hkv, stride), torch.arange(stride, dtype=i32, device="cuda").repeat(2, hkv, 1)
            self.zero = z(2, t=i32)
            d_, t, fill = self.d, self.t, self.d.fill
            self.d.lens = t["len"]
            self.a = [
                ("sfb_k_attention_tree_paged", fill(L.TreeArgs(), q=t["q"], draft_k=t["dk"], draft_v=t["dv"], parents=t["parents"], out=self.out,
                                                    q_heads=hq, nodes=nodes, max_context=max_context)),
                ("sfb_k_paged_kv_accept", self.accept()),
                ("sfb_k_paged_kv_bounds", self.block_bounds()),
                ("sfb_k_attention_decode_sparse", fill(L.SparseArgs(), q=t["q1"], bounds=self.bounds, out=self.out1, selected=self.selected,
                                                       q_heads=hq, budget_blocks=6, sink_blocks=1, recent_blocks=1, max_context=max_context)),
                ("sfb_k_attention_decode_weights", fill(L.WeightsArgs(), q=t["q1"], out=self.out2, weights=self.weights, weights_out=self.weights,
                                                        q_heads=hq, weight_stride=stride, max_context=max_context)),
                ("sfb_k_paged_kv_evict", fill(L.EvictArgs(), weights=self.weights, weights_out=self.weights, positions=self.positions,
                                              positions_out=self.positions, new_len=self.cut_len, weight_stride=stride, budget=budget,
                                              sink_tokens=2, recent_tokens=8, max_context=max_context)),
            ]
            sizes = {0: "sfb_attention_tree_workspace", 3: "sfb_attention_sparse_workspace", 4: "sfb_attention_weights_workspace",
                     5: "sfb_paged_kv_evict_workspace"}
            self.keep = []
            for i, (name, a) in enumerate(self.a):
                if i >= 3:      # these see the accepted tokens
                    a.context_len = self.new_len.data_ptr()
                if i in sizes:
                    ws = workspace(dev, getattr(lib, sizes[i])(C.byref(a)))
                    a.workspace = ws.data_ptr()
                    self.keep.append(ws)

        def accept(self):
            a, t, c = L.AcceptArgs(), self.t, cache
            a.draft_k, a.draft_v, a.k_pool, a.v_pool = (x.data_ptr() for x in (t["dk"], t["dv"], self.d.k_pool, self.d.v_pool))
            a.block_table, a.start_len, a.path, a.path_len = (x.data_ptr() for x in (self.d.table, t["len"], t["path"], t["path_len"]))
            a.new_len = self.new_len.data_ptr()
            a.batch, a.kv_heads, a.nodes, a.max_path, a.head_dim, a.head_dim_value = 2, hkv, nodes, 4, d, d
            a.block_tokens, a.max_blocks, a.num_blocks, a.dtype = 16, c.max_blocks, c.num_blocks, CODE[dtype]
            return a

        def block_bounds(self):
            a = L.BoundsArgs()
            a.k_pool, a.bounds, a.block_table = self.d.k_pool.data_ptr(), self.bounds.data_ptr(), self.d.table.data_ptr()
            a.start_len, a.end_len = self.zero.data_ptr(), self.new_len.data_ptr()
            a.batch, a.kv_heads, a.head_dim, a.max_tokens = 2, hkv, d, max_context
            a.block_tokens, a.max_blocks, a.num_blocks, a.dtype = 16, cache.max_blocks, cache.num_blocks, CODE[dtype]
            return a

        def run(self, stream):
            for name, a in self.a:
                L.check(getattr(lib, name)(C.byref(a), C.c_void_p(stream)))

        def load(self, seed):
            for k, v in inputs(seed).items():
                self.t[k].copy_(torch.from_numpy(np.ascontiguousarray(v)))
            self.d.k_pool.copy_(self.d.put(cache.k_pool))
            self.d.v_pool.copy_(self.d.put(cache.v_pool))
            self.weights.zero_()
            self.positions.copy_(torch.arange(stride, device="cuda", dtype=torch.int32).repeat(2, hkv, 1))
            torch.cuda.synchronize()

        def results(self):
            torch.cuda.synchronize()
            n = self.new_len.tolist()
            kept = [self.weights[b, :, :n[b]].clone() for b in range(2)]
            return [x.clone() for x in (self.out, self.out1, self.out2, self.new_len, self.cut_len, self.selected, self.positions,
                                        self.d.k_pool, self.d.v_pool)] + kept

    status_word()
    direct, captured = Step(), Step()
    side = torch.cuda.Stream()
    captured.load(0)
    with torch.cuda.stream(side):
        captured.run(side.cuda_stream)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.run(torch.cuda.current_stream().cuda_stream)
    for seed in (0, 5, 6):
        direct.load(seed)
        direct.run(dev.stream())
        want = direct.results()
        captured.load(seed)
        graph.replay()
        for x, y in zip(captured.results(), want):
            assert torch.equal(x, y)
    assert status_word() == 0


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("f32", 64)])
def test_calls_on_several_streams_and_again_give_the_same_bits(dev, port, dtype, d):
    torch = dev.torch
    rng = np.random.default_rng(12)
    cache = Cache(rng, [700, 90, 333], 2, d, d, 16, dtype, round_bf16=port.round_bf16)
    q, dk, dv, parents = tree_inputs(rng, port, cache, 8, 20, [20, 20, 11])
    first = tree_call(dev, port, cache, 8, 20, [20, 20, 11], parents, q, dk, dv)
    dd = Device(dev, cache)
    bounds = dd.put(np.zeros((cache.num_blocks, 2, 2, d), np.float32))
    bounds_call(dev, dd, bounds, [0] * 3, cache.lens, 700)
    q1 = np.ascontiguousarray(q[:, :, 0])
    sparse = sparse_call(dev, dd, q1, bounds, 8, 9, 1, 1)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for s in streams:
        assert np.array_equal(tree_call(dev, port, cache, 8, 20, [20, 20, 11], parents, q, dk, dv, stream=s.cuda_stream), first)
    jobs = []
    for s in streams:      # in flight together, each with its own outputs and scratch
        out = torch.zeros((3, 8, d), dtype=dd.type, device="cuda")
        selected = torch.zeros((3, 2, 9), dtype=torch.int32, device="cuda")
        qd = dd.put(q1)
        a = dd.fill(L.SparseArgs(), q=qd, bounds=bounds, out=out, selected=selected, q_heads=8, budget_blocks=9, sink_blocks=1,
                    recent_blocks=1, max_context=700)
        ws = workspace(dev, L.load().sfb_attention_sparse_workspace(C.byref(a)))
        a.workspace = ws.data_ptr()
        jobs.append((a, out, selected, qd, ws))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (a, *_rest) in zip(streams, jobs):
            L.check(L.load().sfb_k_attention_decode_sparse(C.byref(a), C.c_void_p(s.cuda_stream)))
    torch.cuda.synchronize()
    for _, out, selected, *_rest in jobs:
        assert np.array_equal(dev.np(out), sparse[0]) and np.array_equal(dev.np(selected), sparse[1])


# ---- large pools, odd addresses ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64), ("f32", 24)])
def test_pools_beyond_2_to_the_31_elements(dev, port, dtype, d):
    """The same pages at the end of a pool of more than 2^31 elements give the same bits as in a small one."""
    torch = dev.torch
    rng = np.random.default_rng(13)
    hkv, block, hq, nodes = 2, 16, 8, 6
    lens = [130, 47]
    cache = Cache(rng, lens, hkv, d, d, block, dtype, room=8, poison=0.5, round_bf16=port.round_bf16)
    q, dk, dv, parents = tree_inputs(rng, port, cache, hq, nodes, [6, 6])
    q1 = np.ascontiguousarray(q[:, :, 0])
    path, path_len = np.array([[0, 2, 4], [1, 3, 5]], np.int32), np.array([3, 2])
    stride = 160
    weights = rng.random((2, hkv, stride)).astype(np.float32)
    positions = np.broadcast_to(np.arange(stride), (2, hkv, stride)).astype(np.int32)
    big_blocks = (1 << 31) // (hkv * block * d) + cache.num_blocks + 1
    results = []
    for large in (False, True):
        dd = Device(dev, cache)
        if large:
            shift = big_blocks - cache.num_blocks
            for name in ("k_pool", "v_pool"):
                pool = torch.empty((big_blocks, hkv, block, d), dtype=dd.type, device="cuda")
                pool[shift:] = getattr(dd, name)
                setattr(dd, name, pool)
            dd.table = torch.where(dd.table >= 0, dd.table + shift, dd.table)
            dd.cache = SimpleNamespace(**{**vars(cache), "num_blocks": big_blocks})
        else:
            shift = 0
        c = dd.cache
        t = dict(q=dd.put(q), draft_k=dd.put(dk), draft_v=dd.put(dv), parents=dev.i32(parents))
        out = torch.zeros((2, hq, nodes, d), dtype=dd.type, device="cuda")
        a = dd.fill(L.TreeArgs(), **t, out=out, q_heads=hq, nodes=nodes, max_context=130)
        ws = workspace(dev, L.load().sfb_attention_tree_workspace(C.byref(a)))
        a.workspace = ws.data_ptr()
        L.check(L.load().sfb_k_attention_tree_paged(C.byref(a), C.c_void_p(dev.stream())))
        got = [dev.np(out)]
        new_len = accept_call(dev, dd, c, nodes, path, path_len, dk, dv)
        dd.lens = dev.i32(new_len)
        dd.cache = SimpleNamespace(**{**vars(c), "lens": list(new_len)})
        bounds = torch.zeros((c.num_blocks, hkv, 2, d), dtype=dd.type, device="cuda")
        bounds_call(dev, dd, bounds, [0, 0], new_len, 140)
        got += list(sparse_call(dev, dd, q1, bounds, hq, 4, 1, 1))
        w, p = dev.f32(weights), dev.i32(positions)
        got.append(weights_call(dev, dd, q1, hq, w, w, stride))
        cut = dev.i32(np.zeros(2))
        evict_call(dev, dd, w, w, p, p, cut, stride, 60, 2, 5)
        got += [dev.np(w), dev.np(p), dev.np(cut), dev.np(dd.k_pool[shift:]), dev.np(dd.v_pool[shift:]), dev.np(bounds[shift:])]
        results.append(got)
        del bounds, dd
        torch.cuda.empty_cache()
    for x, y in zip(*results):
        assert np.array_equal(x, y, equal_nan=True)


@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("f32", 64)])
def test_addresses_that_are_only_element_aligned(dev, port, dtype, d):
    """Queries, drafts and pools that start one element behind a 16-byte boundary take the kernels for any layout."""
    torch = dev.torch
    rng = np.random.default_rng(14)
    cache = Cache(rng, [200, 33], 2, d, d, 16, dtype, round_bf16=port.round_bf16)
    nodes, hq = 5, 4
    q, dk, dv, parents = tree_inputs(rng, port, cache, hq, nodes, [5, 5])

    def odd(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
        view = flat[1:].view(x.shape)
        view.copy_(x)
        return view

    dd = Device(dev, cache)
    dd.k_pool, dd.v_pool = odd(dd.k_pool), odd(dd.v_pool)
    t = dict(q=odd(dd.put(q)), draft_k=odd(dd.put(dk)), draft_v=odd(dd.put(dv)), parents=dev.i32(parents))
    out = odd(torch.full((2, hq, nodes, d), 7.0, dtype=dd.type, device="cuda"))
    a = dd.fill(L.TreeArgs(), **t, out=out, q_heads=hq, nodes=nodes, max_context=200)
    ws = workspace(dev, L.load().sfb_attention_tree_workspace(C.byref(a)))
    a.workspace = ws.data_ptr()
    L.check(L.load().sfb_k_attention_tree_paged(C.byref(a), C.c_void_p(dev.stream())))
    tree_check(dev.np(out), cache, hq, [5, 5], parents, q, dk, dv)
    bounds = odd(torch.zeros((cache.num_blocks, 2, 2, d), dtype=dd.type, device="cuda"))
    bounds_call(dev, dd, bounds, [0, 0], cache.lens, 200)
    q1 = np.ascontiguousarray(q[:, :, 0])
    aligned = Device(dev, cache)
    aligned_bounds = torch.zeros((cache.num_blocks, 2, 2, d), dtype=dd.type, device="cuda")
    bounds_call(dev, aligned, aligned_bounds, [0, 0], cache.lens, 200)
    assert torch.equal(bounds, aligned_bounds)
    got, selected = sparse_call(dev, dd, q1, bounds, hq, 5, 1, 1)
    want, chosen = sparse_call(dev, aligned, q1, aligned_bounds, hq, 5, 1, 1)
    assert np.array_equal(selected, chosen)
    w = dev.f32(np.zeros((2, 2, 200)))
    again = weights_call(dev, dd, q1, hq, None, w, 200)
    for b in range(2):
        for h in range(hq):
            k, v = cache.keys[b][h // 2], cache.values[b][h // 2]
            at = [t for i in selected[b, h // 2] if i >= 0 for t in range(i * 16, min(cache.lens[b], i * 16 + 16))]
            for rows, result in ((at, got), (slice(None), again)):
                exact, bound, _ = attend(q1[b, h:h + 1].astype(np.float64), k[rows], v[rows], dtype)
                close(result[b, h:h + 1], exact, bound)
