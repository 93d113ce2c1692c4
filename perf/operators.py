"""Serving operators over the paged K/V cache: what they compute, at which sizes they are measured, and their plain forms.

  tree     attention of a tree of drafted tokens over the cache (sfb_k_attention_tree_paged)
  accept   append of the accepted path's K/V rows (sfb_k_paged_kv_accept)
  sparse   block bounds, block selection and attention over the selected blocks, one decode step
           (sfb_k_paged_kv_bounds, sfb_k_attention_decode_sparse)
  weights  decode attention that adds its softmax weights to a running sum (sfb_k_attention_decode_weights)
  evict    removal of the positions with the least accumulated weight (sfb_k_paged_kv_evict)

`own` chooses between the plain torch forms (False) and the calls of schedforge_b200 (True).
"""
import ctypes
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ---- cases -----------------------------------------------------------------------------------------------


def listed():
    heads8b = dict(q_heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16")   # the decoder layer of the benchmark
    small = dict(q_heads=8, kv_heads=2, head_dim=64, block=16)                     # the small layer of the tests
    return [
        # one user, a short chat, a handful of drafted tokens: latency is all that counts
        dict(name="tree_step", op="tree", batch=1, context=512, nodes=8, ragged=False, **heads8b),
        # exact-order serving of a small model: float32, every sequence of another length and tree size
        dict(name="tree_ragged", op="tree", batch=16, context=1500, nodes=27, ragged=True, dtype="fp32", **small),
        # a batch of long documents with wide trees: 256 query rows for each K/V head
        dict(name="tree_long", op="tree", batch=8, context=16384, nodes=64, ragged=True, **heads8b),
        # the token bookkeeping after a verified step: one sequence, and a full batch
        dict(name="accept_step", op="accept", batch=1, context=512, nodes=8, path=5, ragged=False, **heads8b),
        dict(name="accept_batch", op="accept", batch=64, context=200, nodes=64, path=16, ragged=True, **heads8b),
        # one user over a medium context that reads an eighth of its blocks
        dict(name="sparse_step", op="sparse", batch=1, context=8192, budget=64, sink=1, recent=2, ragged=False, **heads8b),
        # ragged batch of the small float32 model with an odd budget; short sequences keep every block
        dict(name="sparse_ragged", op="sparse", batch=24, context=8192, budget=33, sink=1, recent=4, ragged=True,
             dtype="fp32", **small),
        # long-context serving: 128 thousand tokens a sequence, about 1.6 % of the blocks read
        dict(name="sparse_long", op="sparse", batch=8, context=131072, budget=128, sink=1, recent=4, ragged=False, **heads8b),
        # decode steps that also keep the accumulated attention weights: one user, and the paged batch of the benchmark
        dict(name="weights_step", op="weights", batch=1, context=2048, ragged=False, **heads8b),
        dict(name="weights_batch", op="weights", batch=64, context=8192, ragged=True, **heads8b),
        # a cache held at its budget: every step one position leaves
        dict(name="evict_step", op="evict", batch=16, context=2049, budget=2048, sink=4, recent=64, ragged=False, **heads8b),
        # after a long prompt the cache is cut to its budget once (float32 cache of the small model)
        dict(name="evict_prompt", op="evict", batch=4, context=16384, budget=2048, sink=4, recent=256, ragged=True,
             dtype="fp32", **small),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "accept", "sparse", "sparse", "weights", "evict"])
    case = dict(op=op, kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 128]), block=rng.choice([16, 16, 32]),
                dtype=rng.choice(["bf16", "bf16", "fp32"]), ragged=rng.random() < 0.7)
    group = rng.choice([1, 2, 4, 8])
    case["q_heads"] = case["kv_heads"] * group
    if op == "tree":
        case["nodes"] = _log(rng, 1, 128)
        case["batch"] = _log(rng, 1, 32)
        case["context"] = _log(rng, 1, 16384 if case["dtype"] == "bf16" else 2048)
        case["context"] = max(1, min(case["context"], 131072 // case["batch"]))
    elif op == "accept":
        case["nodes"] = _log(rng, 1, 128)
        case["path"] = rng.randint(1, min(16, case["nodes"]))
        case["batch"] = _log(rng, 1, 64)
        case["context"] = _log(rng, 1, 1000)
    elif op == "sparse":
        case["batch"] = _log(rng, 1, 32)
        case["context"] = min(_log(rng, 1, 131072), 1048576 // case["batch"] // (1 if case["dtype"] == "bf16" else 4))
        case["budget"] = _log(rng, 8, 256)
        case["sink"] = rng.randint(0, 3)
        case["recent"] = rng.randint(0, 5)
    elif op == "weights":
        case["batch"] = _log(rng, 1, 64)
        case["context"] = min(_log(rng, 1, 32768), 524288 // case["batch"] // (1 if case["dtype"] == "bf16" else 4))
    else:
        case["batch"] = _log(rng, 1, 16)
        case["context"] = min(_log(rng, 64, 32768), 131072 // case["batch"])
        case["budget"] = max(16, int(case["context"] * rng.uniform(0.1, 1.1)))
        case["sink"] = rng.randint(0, 4)
        case["recent"] = rng.randint(0, case["budget"] // 4)
    return case


# ---- inputs ----------------------------------------------------------------------------------------------


def _lengths(case, seed):
    """Context lengths as host integers: all equal, or spread down to a sixteenth."""
    g = torch.Generator().manual_seed(seed * 7 + 1)
    n, longest = case["batch"], case["context"]
    if not case["ragged"]:
        return [longest] * n
    lens = torch.randint(max(1, longest // 16), longest + 1, (n,), generator=g).tolist()
    lens[seed % n] = longest
    return lens


def _nodes_of(case, seed):
    g = torch.Generator().manual_seed(seed * 7 + 2)
    if not case["ragged"]:
        return [case["nodes"]] * case["batch"]
    return torch.randint(max(1, case["nodes"] // 2), case["nodes"] + 1, (case["batch"],), generator=g).tolist()


def _paths_of(case, seed):
    g = torch.Generator().manual_seed(seed * 7 + 3)
    if not case["ragged"]:
        return [case["path"]] * case["batch"]
    return torch.randint(0, case["path"] + 1, (case["batch"],), generator=g).tolist()


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    b, hkv, hq, d, block = (case[k] for k in ("batch", "kv_heads", "q_heads", "head_dim", "block"))
    lens = _lengths(case, seed)
    room = case["path"] if case["op"] == "accept" else 0
    max_blocks = -(-(case["context"] + room) // block)
    num_blocks = b * max_blocks
    s = dict(case=case, lens=lens, max_blocks=max_blocks, num_blocks=num_blocks)
    # pages of all sequences are interleaved in the pool, as an allocator leaves them
    s["table"] = torch.randperm(num_blocks, generator=gen, device=device).to(torch.int32).reshape(b, max_blocks)
    s["len"] = torch.tensor(lens, dtype=torch.int32, device=device)

    def normal(*shape, scale=1.0):
        x = torch.empty(shape, dtype=dt, device=device).normal_(generator=gen)
        return x if scale == 1.0 else x.mul_(scale)

    s["k_pool"] = normal(num_blocks, hkv, block, d)
    s["v_pool"] = normal(num_blocks, hkv, block, d)
    op = case["op"]
    if op == "sparse":  # keys of one block resemble each other, so that some blocks matter more than others
        s["k_pool"] += normal(num_blocks, hkv, 1, d, scale=0.7)
        s["bounds"] = torch.stack([s["k_pool"].amin(2), s["k_pool"].amax(2)], dim=2).contiguous()
        s["start"] = s["len"] - 1
        s["selected"] = torch.empty((b, hkv, case["budget"]), dtype=torch.int32, device=device)
    if op in ("sparse", "weights"):
        s["q"] = normal(b, hq, d, scale=1.5)
        s["out"] = torch.zeros((b, hq, d), dtype=dt, device=device)
    if op in ("tree", "accept"):
        n = case["nodes"]
        s["draft_k"], s["draft_v"] = normal(b, hkv, n, d), normal(b, hkv, n, d)
    if op == "tree":
        s["q"] = normal(b, hq, n, d, scale=1.5)
        i = torch.arange(n, device=device)
        pick = torch.rand((b, n), generator=gen, device=device)
        s["parents"] = ((pick * (i + 1)).floor().long().clamp(max=i) - 1).to(torch.int32)   # -1 .. i - 1
        s["node_count"] = torch.tensor(_nodes_of(case, seed), dtype=torch.int32, device=device)
        s["out"] = torch.zeros((b, hq, n, d), dtype=dt, device=device)
    if op == "accept":
        step = torch.rand((b, n), generator=gen, device=device).argsort(1)[:, : case["path"]]
        s["path"] = step.sort(1).values.to(torch.int32).contiguous()       # ascending node ids, as along a branch
        s["path_len"] = torch.tensor(_paths_of(case, seed), dtype=torch.int32, device=device)
        s["new_len"] = torch.zeros(b, dtype=torch.int32, device=device)
    if op in ("weights", "evict"):
        stride = max_blocks * block
        s["stride"] = stride
        slot = torch.arange(stride, device=device)
        live = (slot[None, :] < s["len"][:, None])[:, None, :]
        w = torch.empty((b, hkv, stride), device=device).normal_(generator=gen).mul_(2.0).exp_().mul_(1e-3)   # a few positions take most
        s["weights"] = (w * live).contiguous()
        s["weights_out"] = torch.zeros_like(s["weights"])
    if op == "evict":
        # slots are out of order after earlier evictions: positions are shuffled within the first half
        key = torch.rand((b, hkv, stride), generator=gen, device=device) * (slot < case["context"] // 2)
        order = (key + slot * (slot >= case["context"] // 2)).argsort(dim=2, stable=True)
        s["positions"] = torch.where(live, order, torch.full_like(order, -1)).to(torch.int32).contiguous()
        s["positions_out"] = torch.full_like(s["positions"], -1)
        s["new_len"] = torch.zeros(b, dtype=torch.int32, device=device)
    return s


# ---- one pass ----------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"tree": _own_tree, "accept": _own_accept, "sparse": _own_sparse, "weights": _own_weights,
                "evict": _own_evict}[op](state)
    return {"tree": _plain_tree, "accept": _plain_accept, "sparse": _plain_sparse, "weights": _plain_weights,
            "evict": _plain_evict}[op](state)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _workspace(state, nbytes):
    """The scratch a program keeps beside its cache: made on the first pass, zero bytes are never required."""
    if "workspace" not in state:
        state["workspace"] = torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device="cuda")
    return state["workspace"].data_ptr()


def _dtype(case, lib):
    return lib.BF16 if case["dtype"] == "bf16" else lib.F32


def _own_tree(s):
    from schedforge_b200 import lib as L
    c, lib = s["case"], L.load()
    a = L.TreeArgs()
    a.q, a.k_pool, a.v_pool = s["q"].data_ptr(), s["k_pool"].data_ptr(), s["v_pool"].data_ptr()
    a.block_table, a.context_len = s["table"].data_ptr(), s["len"].data_ptr()
    a.draft_k, a.draft_v = s["draft_k"].data_ptr(), s["draft_v"].data_ptr()
    a.parents, a.node_count, a.out = s["parents"].data_ptr(), s["node_count"].data_ptr(), s["out"].data_ptr()
    a.batch, a.q_heads, a.kv_heads, a.nodes = c["batch"], c["q_heads"], c["kv_heads"], c["nodes"]
    a.head_dim = a.head_dim_value = c["head_dim"]
    a.block_tokens, a.max_blocks, a.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    a.max_context, a.dtype = c["context"], _dtype(c, L)
    if "workspace" not in s:
        _workspace(s, lib.sfb_attention_tree_workspace(ctypes.byref(a)))
    a.workspace = s["workspace"].data_ptr()
    L.check(lib.sfb_k_attention_tree_paged(ctypes.byref(a), _stream()))
    return s["out"]


def _own_accept(s):
    from schedforge_b200 import lib as L
    c = s["case"]
    a = L.AcceptArgs()
    a.draft_k, a.draft_v = s["draft_k"].data_ptr(), s["draft_v"].data_ptr()
    a.k_pool, a.v_pool, a.block_table = s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["table"].data_ptr()
    a.start_len, a.path, a.path_len = s["len"].data_ptr(), s["path"].data_ptr(), s["path_len"].data_ptr()
    a.new_len = s["new_len"].data_ptr()
    a.batch, a.kv_heads, a.nodes, a.max_path = c["batch"], c["kv_heads"], c["nodes"], c["path"]
    a.head_dim = a.head_dim_value = c["head_dim"]
    a.block_tokens, a.max_blocks, a.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    a.dtype = _dtype(c, L)
    L.check(L.load().sfb_k_paged_kv_accept(ctypes.byref(a), _stream()))
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], "new_len": s["new_len"]}


def _own_sparse(s):
    from schedforge_b200 import lib as L
    c, lib, stream = s["case"], L.load(), _stream()
    u = L.BoundsArgs()
    u.k_pool, u.bounds, u.block_table = s["k_pool"].data_ptr(), s["bounds"].data_ptr(), s["table"].data_ptr()
    u.start_len, u.end_len = s["start"].data_ptr(), s["len"].data_ptr()
    u.batch, u.kv_heads, u.head_dim, u.max_tokens = c["batch"], c["kv_heads"], c["head_dim"], 1
    u.block_tokens, u.max_blocks, u.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    u.dtype = _dtype(c, L)
    L.check(lib.sfb_k_paged_kv_bounds(ctypes.byref(u), stream))
    a = L.SparseArgs()
    a.q, a.k_pool, a.v_pool, a.bounds = (s[k].data_ptr() for k in ("q", "k_pool", "v_pool", "bounds"))
    a.block_table, a.context_len = s["table"].data_ptr(), s["len"].data_ptr()
    a.out, a.selected = s["out"].data_ptr(), s["selected"].data_ptr()
    a.batch, a.q_heads, a.kv_heads = c["batch"], c["q_heads"], c["kv_heads"]
    a.head_dim = a.head_dim_value = c["head_dim"]
    a.block_tokens, a.max_blocks, a.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    a.max_context, a.dtype = c["context"], _dtype(c, L)
    a.budget_blocks, a.sink_blocks, a.recent_blocks = c["budget"], c["sink"], c["recent"]
    if "workspace" not in s:
        _workspace(s, lib.sfb_attention_sparse_workspace(ctypes.byref(a)))
    a.workspace = s["workspace"].data_ptr()
    L.check(lib.sfb_k_attention_decode_sparse(ctypes.byref(a), stream))
    return {"out": s["out"], "selected": s["selected"], "bounds": s["bounds"]}


def _own_weights(s):
    from schedforge_b200 import lib as L
    c, lib = s["case"], L.load()
    a = L.WeightsArgs()
    a.q, a.k_pool, a.v_pool = s["q"].data_ptr(), s["k_pool"].data_ptr(), s["v_pool"].data_ptr()
    a.block_table, a.context_len, a.out = s["table"].data_ptr(), s["len"].data_ptr(), s["out"].data_ptr()
    a.weights, a.weights_out = s["weights"].data_ptr(), s["weights_out"].data_ptr()
    a.batch, a.q_heads, a.kv_heads = c["batch"], c["q_heads"], c["kv_heads"]
    a.head_dim = a.head_dim_value = c["head_dim"]
    a.block_tokens, a.max_blocks, a.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    a.max_context, a.weight_stride, a.dtype = c["context"], s["stride"], _dtype(c, L)
    if "workspace" not in s:
        _workspace(s, lib.sfb_attention_weights_workspace(ctypes.byref(a)))
    a.workspace = s["workspace"].data_ptr()
    L.check(lib.sfb_k_attention_decode_weights(ctypes.byref(a), _stream()))
    return {"out": s["out"], "weights": s["weights_out"]}


def _own_evict(s):
    from schedforge_b200 import lib as L
    c, lib = s["case"], L.load()
    a = L.EvictArgs()
    a.k_pool, a.v_pool, a.block_table = s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["table"].data_ptr()
    a.context_len, a.new_len = s["len"].data_ptr(), s["new_len"].data_ptr()
    a.weights, a.weights_out = s["weights"].data_ptr(), s["weights_out"].data_ptr()
    a.positions, a.positions_out = s["positions"].data_ptr(), s["positions_out"].data_ptr()
    a.batch, a.kv_heads, a.max_context, a.weight_stride = c["batch"], c["kv_heads"], c["context"], s["stride"]
    a.head_dim = a.head_dim_value = c["head_dim"]
    a.block_tokens, a.max_blocks, a.num_blocks = c["block"], s["max_blocks"], s["num_blocks"]
    a.budget, a.sink_tokens, a.recent_tokens, a.dtype = c["budget"], c["sink"], c["recent"], _dtype(c, L)
    if "workspace" not in s:
        _workspace(s, lib.sfb_paged_kv_evict_workspace(ctypes.byref(a)))
    a.workspace = s["workspace"].data_ptr()
    L.check(lib.sfb_k_paged_kv_evict(ctypes.byref(a), _stream()))
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], "weights": s["weights_out"], "positions": s["positions_out"],
            "new_len": s["new_len"]}


# ---- plain forms -------------------------------------------------------------------------------------------


def _rows(pool, table):
    """[batch, kv_heads, max_blocks * block, dim] in float32: the pages of every sequence in logical order."""
    x = pool[table.long()]                                    # [b, max_blocks, heads, block, dim]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _softmax(scores, seen):
    """Softmax over the visible entries of the last axis; a row that sees nothing gets zeros."""
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total == 0, torch.ones_like(total), total)


def _plain_tree(s):
    c = s["case"]
    b, hkv, n, d = c["batch"], c["kv_heads"], c["nodes"], c["head_dim"]
    group = c["q_heads"] // hkv
    keys = torch.cat([_rows(s["k_pool"], s["table"]), s["draft_k"].float()], 2)
    values = torch.cat([_rows(s["v_pool"], s["table"]), s["draft_v"].float()], 2)
    node = torch.arange(n, device=keys.device)
    link = torch.eye(n, dtype=torch.float64, device=keys.device) + (s["parents"][:, :, None] == node).double()
    seen_tree = torch.linalg.matrix_power(link, n) > 0        # [b, i, j]: j is i or one of its ancestors
    live = node[None, :] < s["node_count"][:, None]
    seen_context = torch.arange(keys.shape[2] - n, device=keys.device)[None, :] < s["len"][:, None]
    seen = torch.cat([seen_context[:, None, :].expand(b, n, -1), seen_tree & live[:, None, :]], 2)
    q = s["q"].float().reshape(b, hkv, group, n, d).reshape(b, hkv, group * n, d) * (1.0 / math.sqrt(d))
    scores = torch.matmul(q, keys.transpose(2, 3)).reshape(b, hkv, group, n, -1)
    p = _softmax(scores, seen[:, None, None]).reshape(b, hkv, group * n, -1)
    out = torch.matmul(p, values).reshape(b, hkv * group, n, d)
    return (out * live[:, None, :, None]).to(s["q"].dtype)    # rows behind the last node stay as they were: zero


def _plain_accept(s):
    c = s["case"]
    hkv, block = c["kv_heads"], c["block"]
    step = torch.arange(c["path"], device=s["path"].device)
    b, t = (step[None, :] < s["path_len"][:, None]).nonzero(as_tuple=True)
    position = s["len"].long()[b] + t
    page = s["table"].long()[b, position // block]
    node = s["path"].long()[b, t]
    s["k_pool"][page, :, position % block] = s["draft_k"][b, :, node]
    s["v_pool"][page, :, position % block] = s["draft_v"][b, :, node]
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], "new_len": s["len"] + s["path_len"]}


def _plain_sparse(s):
    c = s["case"]
    b, hkv, d, block, budget = c["batch"], c["kv_heads"], c["head_dim"], c["block"], c["budget"]
    group = c["q_heads"] // hkv
    device = s["q"].device
    # bounds of the block that holds the newest token, over its live tokens
    last = (s["len"].long() - 1) // block
    page = s["table"].long()[torch.arange(b, device=device), last]
    slot = last[:, None] * block + torch.arange(block, device=device)
    dead = (slot >= s["len"][:, None])[:, None, :, None]
    newest = s["k_pool"][page]
    s["bounds"][page, :, 0] = newest.masked_fill(dead, math.inf).amin(2)
    s["bounds"][page, :, 1] = newest.masked_fill(dead, -math.inf).amax(2)
    # upper bound of every block's scores, the largest over the heads that share it; 64 bits, since ranks follow from it
    bounds = s["bounds"][s["table"].long()].permute(0, 2, 3, 1, 4).double()    # [b, heads, 2, blocks, dim]
    q = s["q"].double().reshape(b, hkv, group, d)
    upper = torch.matmul(q.clamp(min=0), bounds[:, :, 1].transpose(2, 3)) + torch.matmul(q.clamp(max=0), bounds[:, :, 0].transpose(2, 3))
    upper = upper.amax(2)
    index = torch.arange(s["max_blocks"], device=device)
    blocks = (s["len"].long() + block - 1) // block
    live = index[None, :] < blocks[:, None]
    always = live & ((index[None, :] < c["sink"]) | (index[None, :] >= blocks[:, None] - c["recent"]))
    upper = upper.masked_fill(always[:, None], math.inf).masked_fill(~live[:, None], -math.inf)
    order = upper.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.minimum(blocks, torch.tensor(budget, device=device))
    chosen = torch.arange(order.shape[-1], device=device)[None, :] < kept[:, None]
    order = torch.where(chosen[:, None], order, torch.full_like(order, s["max_blocks"])).sort(-1).values
    chosen = chosen[:, None].expand_as(order)
    selected = torch.full((b, hkv, budget), -1, dtype=torch.int32, device=device)
    selected[..., : order.shape[-1]] = torch.where(chosen, order, torch.full_like(order, -1)).to(torch.int32)
    # attention over the chosen blocks
    logical = torch.where(chosen, order, torch.zeros_like(order))
    page = s["table"].long()[torch.arange(b, device=device)[:, None, None], logical]
    head = torch.arange(hkv, device=device)[None, :, None]
    keys = s["k_pool"][page, head].float().flatten(2, 3)      # [b, heads, budget * block, dim]
    values = s["v_pool"][page, head].float().flatten(2, 3)
    position = logical[..., None] * block + torch.arange(block, device=device)
    seen = (chosen[..., None] & (position < s["len"][:, None, None, None])).flatten(2, 3)
    q = s["q"].float().reshape(b, hkv, group, d) * (1.0 / math.sqrt(d))
    p = _softmax(torch.matmul(q, keys.transpose(2, 3)), seen[:, :, None])
    out = torch.matmul(p, values).reshape(b, hkv * group, d).to(s["q"].dtype)
    return {"out": out, "selected": selected, "bounds": s["bounds"]}


def _plain_weights(s):
    c = s["case"]
    b, hkv, d = c["batch"], c["kv_heads"], c["head_dim"]
    group = c["q_heads"] // hkv
    keys, values = _rows(s["k_pool"], s["table"]), _rows(s["v_pool"], s["table"])
    seen = torch.arange(keys.shape[2], device=keys.device)[None, :] < s["len"][:, None]
    q = s["q"].float().reshape(b, hkv, group, d) * (1.0 / math.sqrt(d))
    p = _softmax(torch.matmul(q, keys.transpose(2, 3)), seen[:, None, None])
    out = torch.matmul(p, values).reshape(b, hkv * group, d).to(s["q"].dtype)
    return {"out": out, "weights": s["weights"] + p.sum(2)}


def _plain_evict(s):
    c = s["case"]
    block = c["block"]
    device = s["weights"].device
    slot = torch.arange(s["stride"], device=device)
    live = (slot[None, :] < s["len"][:, None])[:, None].expand_as(s["weights"])
    new_len = torch.clamp(s["len"], max=c["budget"])
    newest = torch.where(live, s["positions"], torch.full_like(s["positions"], -1)).amax(-1, keepdim=True)
    always = live & ((s["positions"] < c["sink"]) | (s["positions"] > newest - c["recent"]))
    key = s["weights"].masked_fill(always, math.inf).masked_fill(~live, -math.inf)
    rank = key.sort(dim=-1, descending=True, stable=True).indices.argsort(-1)
    kept = rank < new_len[:, None, None]
    front = slot < new_len[:, None, None]
    hole, tail = front & ~kept, ~front & kept                 # equally many in every row, both in ascending order
    b, h, to = hole.nonzero(as_tuple=True)
    since = tail.nonzero(as_tuple=True)[2]
    page_from, page_to = s["table"].long()[b, since // block], s["table"].long()[b, to // block]
    s["k_pool"][page_to, h, to % block] = s["k_pool"][page_from, h, since % block]
    s["v_pool"][page_to, h, to % block] = s["v_pool"][page_from, h, since % block]
    weights = torch.where(front & live, s["weights"], torch.zeros_like(s["weights"]))
    positions = torch.where(front & live, s["positions"], torch.full_like(s["positions"], -1))
    weights[b, h, to] = s["weights"][b, h, since]
    positions[b, h, to] = s["positions"][b, h, since]
    return {"k_pool": s["k_pool"], "v_pool": s["v_pool"], "weights": weights, "positions": positions, "new_len": new_len}


# ---- what one pass cannot do without -------------------------------------------------------------------------


def work(case):
    b, hq, hkv, d = (case[k] for k in ("batch", "q_heads", "kv_heads", "head_dim"))
    e = 2 if case["dtype"] == "bf16" else 4
    # sum of ragged lengths: uniform between a sixteenth and the whole, one sequence at the whole
    mean = case["context"] if not case["ragged"] else case["context"] * 17 / 32
    tokens = mean * (b - 1) + case["context"]
    op = case["op"]
    if op == "tree":
        n = case["nodes"] if not case["ragged"] else case["nodes"] * 0.75
        rows = b * n
        nbytes = (tokens + rows) * hkv * 2 * d * e + 2 * rows * hq * d * e + rows * 4
        return {"bytes": nbytes, "flops": (tokens * n + rows * max(1.0, math.log2(n + 1))) * hq * 4 * d}
    if op == "accept":
        rows = b * (case["path"] if not case["ragged"] else case["path"] / 2)
        return {"bytes": rows * hkv * 4 * d * e + rows * 4 + b * 12, "flops": 0}
    if op == "sparse":
        blocks = tokens / case["block"]
        chosen = min(tokens, b * case["budget"] * case["block"])
        nbytes = (blocks * 2 * d + chosen * 2 * d + b * case["block"] * d) * hkv * e + 2 * b * hq * d * e + b * hkv * case["budget"] * 4
        return {"bytes": nbytes, "flops": (2 * blocks + 4 * chosen) * hq * d}
    if op == "weights":
        return {"bytes": tokens * hkv * (2 * d * e + 8) + 2 * b * hq * d * e, "flops": tokens * hq * 4 * d}
    kept = min(tokens, b * min(case["budget"], case["context"]))
    moved = kept * (1 - kept / tokens)
    return {"bytes": tokens * hkv * 16 + moved * hkv * 4 * d * e, "flops": 0}


# ---- the definition in 64 bits -------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "sparse": _exact_sparse, "weights": _exact_weights,
            "evict": _exact_evict}[case["op"]](case, s)


def _sequence(pool, table, length, block):
    """[kv_heads, length, dim] in float64."""
    pages = table[: -(-length // block)].long()
    return torch.cat(list(pool[pages].double()), 1)[:, :length]


def _attend(q, keys, values):
    """q [rows, d], keys and values [n, d]: rows of softmax(q keys^T / sqrt(d)) and their products with values."""
    x = q @ keys.T / math.sqrt(q.shape[1])
    p = torch.softmax(x, 1)
    return p, p @ values


def _exact_tree(case, s):
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lens"]):
        keys = _sequence(s["k_pool"], s["table"][b], length, case["block"])
        values = _sequence(s["v_pool"], s["table"][b], length, case["block"])
        parents, count = s["parents"][b].tolist(), int(s["node_count"][b])
        line = []
        for i in range(count):
            line.append(([] if parents[i] < 0 else line[parents[i]]) + [i])
        hidden = torch.ones((count, count), dtype=torch.bool)
        for i in range(count):
            hidden[i, line[i]] = False
        hidden = hidden.cuda()
        for h in range(case["kv_heads"]):
            q = s["q"][b, h * group:(h + 1) * group, :count].double()
            x = torch.cat([q @ keys[h].T, (q @ s["draft_k"][b, h, :count].double().T).masked_fill(hidden, -math.inf)], 2)
            p = torch.softmax(x / math.sqrt(case["head_dim"]), 2)
            out[b, h * group:(h + 1) * group, :count] = p[..., :length] @ values[h] + p[..., length:] @ s["draft_v"][b, h, :count].double()
    return out


def _exact_accept(case, s):
    pools = {"k": s["k_pool"].double(), "v": s["v_pool"].double()}
    path, count, table = s["path"].tolist(), s["path_len"].tolist(), s["table"].tolist()
    for b, length in enumerate(s["lens"]):
        for t in range(count[b]):
            block, at = divmod(length + t, case["block"])
            pools["k"][table[b][block], :, at] = s["draft_k"][b, :, path[b][t]].double()
            pools["v"][table[b][block], :, at] = s["draft_v"][b, :, path[b][t]].double()
    new_len = torch.tensor([n + k for n, k in zip(s["lens"], count)], dtype=torch.int32)
    return {"k_pool": pools["k"], "v_pool": pools["v"], "new_len": new_len}


def _exact_sparse(case, s):
    group, block, budget = case["q_heads"] // case["kv_heads"], case["block"], case["budget"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    selected = torch.full(s["selected"].shape, -1, dtype=torch.int32)
    bounds = s["bounds"].double()
    for b, length in enumerate(s["lens"]):
        n = -(-length // block)
        pages = s["table"][b, :n].long()
        rest = s["k_pool"][pages[-1], :, : length - (n - 1) * block].double()
        bounds[pages[-1], :, 0], bounds[pages[-1], :, 1] = rest.min(1).values, rest.max(1).values
        forced = set(range(min(case["sink"], n))) | set(range(max(0, n - case["recent"]), n))
        for h in range(case["kv_heads"]):
            q = s["q"][b, h * group:(h + 1) * group].double()
            score = torch.stack([torch.where(row > 0, bounds[pages, h, 1], bounds[pages, h, 0]) @ row for row in q]).max(0).values
            score = score.tolist()
            ranked = sorted((i for i in range(n) if i not in forced), key=lambda i: (-score[i], i))
            kept = sorted(list(forced) + ranked[: max(0, min(budget, n) - len(forced))])
            selected[b, h, : len(kept)] = torch.tensor(kept, dtype=torch.int32)
            at = torch.tensor(kept, device="cuda")
            live = ((at[:, None] * block + torch.arange(block, device="cuda")) < length).reshape(-1)
            keys = s["k_pool"][pages[at], h].double().reshape(-1, case["head_dim"])[live]
            values = s["v_pool"][pages[at], h].double().reshape(-1, case["head_dim"])[live]
            out[b, h * group:(h + 1) * group] = _attend(q, keys, values)[1]
    return {"out": out, "selected": selected, "bounds": bounds}


def _exact_weights(case, s):
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    weights = s["weights"].double()
    for b, length in enumerate(s["lens"]):
        keys = _sequence(s["k_pool"], s["table"][b], length, case["block"])
        values = _sequence(s["v_pool"], s["table"][b], length, case["block"])
        for h in range(case["kv_heads"]):
            p, o = _attend(s["q"][b, h * group:(h + 1) * group].double(), keys[h], values[h])
            out[b, h * group:(h + 1) * group] = o
            weights[b, h, :length] += p.sum(0)
    return {"out": out, "weights": weights}


def _exact_evict(case, s):
    block, budget = case["block"], case["budget"]
    pools = {"k": s["k_pool"].double(), "v": s["v_pool"].double()}
    weights = torch.zeros(s["weights"].shape, dtype=torch.float64)
    positions = torch.full(s["positions"].shape, -1, dtype=torch.int32)
    w, pos, table = s["weights"].cpu(), s["positions"].cpu(), s["table"].long().cpu()
    new_len = []
    for b, length in enumerate(s["lens"]):
        keep_count = min(length, budget)
        new_len.append(keep_count)
        for h in range(case["kv_heads"]):
            wl, pl = w[b, h, :length].tolist(), pos[b, h, :length].tolist()
            newest = max(pl)
            order = sorted(range(length), key=lambda i: (not (pl[i] < case["sink"] or pl[i] > newest - case["recent"]), -wl[i]
                                                         if not (pl[i] < case["sink"] or pl[i] > newest - case["recent"]) else 0.0, i))
            kept = set(order[:keep_count])
            source = list(range(keep_count))
            free = [i for i in range(keep_count) if i not in kept]
            moved = [i for i in range(keep_count, length) if i in kept]
            for to, since in zip(free, moved):
                source[to] = since
            weights[b, h, :keep_count] = torch.tensor([wl[i] for i in source], dtype=torch.float64)
            positions[b, h, :keep_count] = torch.tensor([pl[i] for i in source], dtype=torch.int32)
            if free:
                to, since = torch.tensor(free), torch.tensor(moved)
                page_to, page_from = table[b, to // block].cuda(), table[b, since // block].cuda()
                to, since = (to % block).cuda(), (since % block).cuda()
                for name, pool in pools.items():
                    pool[page_to, h, to] = s[name + "_pool"][page_from, h, since].double()
    return {"k_pool": pools["k"], "v_pool": pools["v"], "weights": weights, "positions": positions,
            "new_len": torch.tensor(new_len, dtype=torch.int32)}
