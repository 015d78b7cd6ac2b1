"""The calls whose speed this repository answers for beside those of cases.py: drafted trees and ragged
batches over the paged KV cache.

A case is one of three kinds of pass:

* ``tree``:  attention of a tree of drafted tokens over the rows' pages and over the tree's own nodes,
             whose K and V are not in the cache (``PagePool.attend_tree``).
* ``map``:   a kept cache emptied, then for every layer the block tables and the slots of a packed batch
             of prompts, and of ``steps`` further ragged calls (``map_slots_layers``).
* ``write``: packed tokens, or the accepted nodes of drafted trees (``paths``), stored through a slot map
             (``PagePool.write_slots``).

Keys and values are normal, every eighth key channel eight times the others (the outlier channels of
real keys).  Rows are ragged where a case has a ``spread``: lengths from ctx / spread to ctx.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SPARE = 31  # rows of a map pass's pools that no request takes
WINDOW = 128  # positions at a row's end that fp8 pools keep in full precision


def listed():
    tree = dict(kind="tree", batch=16, heads=8, dim=128, group=4, dtype="bf16", page=16, spread=1, fp8=False,
                mask="rows", blind=False)
    maps = dict(kind="map", layers=8, batch=64, page=16, steps=0, spread=32)
    write = dict(kind="write", heads=8, dim=128, dtype="bf16", page=16, nodes=0)
    return [
        # A single token of one user: the smallest call, latency only.
        dict(tree, name="tree-single", batch=1, nodes=1, ctx=700, mask="chain"),
        # A few users of the reference's benchmark model (14 query heads over 2 KV heads x 64), one static
        # tree of 13 nodes for all of them.
        dict(tree, name="tree-small", batch=4, heads=2, dim=64, group=7, nodes=13, ctx=333, mask="shared"),
        # A serving batch, ragged, a tree of 24 nodes for each row.
        dict(tree, name="tree-batch", nodes=24, ctx=2048, spread=4),
        # One long sequence (fp16, page 32), a tree of 64 nodes.
        dict(tree, name="tree-long", batch=1, dtype="fp16", page=32, nodes=64, ctx=32749),
        # Wide trees of a large batch, 8 query heads a KV head: 512 query rows read each K and V, so the
        # matrix products count.  One row is empty, and one node of each tree sees no other.
        dict(tree, name="tree-large", batch=32, group=8, nodes=64, ctx=4096, spread=8, blind=True),
        # Head size 256, a chain of 7 drafted tokens.
        dict(tree, name="tree-wide", batch=12, heads=4, dim=256, group=2, nodes=7, ctx=1500, mask="chain"),
        # fp8 pages behind the residual window.
        dict(tree, name="tree-fp8", nodes=16, ctx=2000, fp8=True),
        # One user's prompt of 37 tokens in a model of two layers.
        dict(maps, name="map-one", layers=2, batch=1, ctx=37, spread=1),
        # 64 ragged prompts for the 32 layers of the benchmark's model, then two steps of 0 to 5 accepted tokens.
        dict(maps, name="map-batch", layers=32, ctx=4096, steps=2),
        # 512 ragged prompts at once.
        dict(maps, name="map-large", batch=512, ctx=4096, spread=16),
        # The accepted nodes of 64 drafted trees of 64 nodes: 0 to 5 of each.
        dict(write, name="write-paths", batch=64, nodes=64, ctx=5),
        # 16 ragged prompts of up to 2,048 tokens, packed.
        dict(write, name="write-prompts", batch=16, ctx=2048),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread evenly over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """A case of the listed ones' kinds: batches of 1 to 64 rows (512 for maps), trees of 1 to 128 nodes,
    contexts of 1 to 32k positions, where it costs no more than the largest listed case."""
    kind = rng.choice(["tree", "tree", "tree", "map", "write"])
    heads, dim = rng.choice([(8, 128), (8, 128), (2, 64), (8, 64), (4, 128), (5, 128), (1, 256), (4, 256)])
    page = rng.choice([16, 16, 32, 8, 64])
    if kind == "map":
        case = dict(kind=kind, layers=rng.randint(1, 32), batch=_spread(rng, 1, 512), page=page,
                    steps=rng.randint(0, 3), spread=rng.choice([1, 4, 32]), ctx=_spread(rng, 1, 4096))
        while work(case)["bytes"] > work(listed()[9])["bytes"]:
            case["ctx"] = max(1, case["ctx"] // 2)
            case["layers"] = max(1, case["layers"] * 3 // 4)
        return case
    dtype = rng.choice(["bf16", "bf16", "fp16"] + ["fp32"] * (kind == "write"))
    case = dict(kind=kind, batch=_spread(rng, 1, 64), heads=heads, dim=dim, dtype=dtype, page=page)
    if kind == "write":
        case.update(nodes=rng.choice([0, 0, _spread(rng, 1, 128)]))
        case["ctx"] = _spread(rng, 1, min(case["nodes"], 8)) if case["nodes"] else _spread(rng, 1, 4096)
    else:
        case.update(group=rng.choice([1, 2, 4, 7, 8]), nodes=_spread(rng, 1, 128), ctx=_spread(rng, 1, 32768),
                    spread=rng.choice([1, 4, 32]), fp8=dim < 256 and page >= 16 and rng.random() < 0.3,
                    mask=rng.choice(["rows", "shared", "chain"]), blind=rng.random() < 0.3)
    limits = [work(c) for c in listed() if c["kind"] == kind]
    while any(work(case)[k] > max(w[k] for w in limits) for k in ("bytes", "flops")):
        if case["ctx"] > 64:
            case["ctx"] = case["ctx"] * 3 // 4
        else:
            case["batch"] = case["batch"] * 3 // 4
    return case


# ------------------------------------------------------------------------------------- inputs
def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((seed * 1009 + part * 31) & 0x7FFFFFFFFFFF)


def _kv(case, seed, part, batch, tokens):
    """K and V [batch, tokens, heads, dim]."""
    g = _generator(seed, part)
    shape = (batch, tokens, case["heads"], case["dim"])
    k = torch.randn(shape, generator=g, device="cuda")
    k[..., ::8] *= 8.0
    v = torch.randn(shape, generator=g, device="cuda")
    return k.to(DTYPES[case["dtype"]]), v.to(DTYPES[case["dtype"]])


def _lengths(case):
    """The rows' lengths; with ``blind`` the first row of several is empty."""
    ctx, spread = case["ctx"], case.get("spread", 1)
    draws = np.random.RandomState(case["batch"] * 7 + spread)
    lens = np.full(case["batch"], ctx, dtype=np.int64)
    if spread > 1:
        lens = draws.randint(max(1, ctx // spread), ctx + 1, case["batch"])
        lens[draws.randint(case["batch"])] = ctx
    if case.get("blind") and case["batch"] > 1:
        lens[0] = 0
    return lens


def _mask(case, seed):
    """The tree's mask, bool [nodes, nodes] or [batch, nodes, nodes]: a node sees itself and its ancestors
    (with ``blind`` the last node sees no node at all); None for a chain."""
    if case["mask"] == "chain":
        return None
    T = case["nodes"]
    draws = np.random.RandomState((seed * 17 + T) & 0x7FFFFFFF)
    trees = 1 if case["mask"] == "shared" else case["batch"]
    mask = np.zeros((trees, T, T), dtype=bool)
    at = np.arange(trees)
    for i in range(T):  # node i hangs on one of the nodes before it, or on the context
        parent = draws.randint(-1, i, trees) if i else np.full(trees, -1)
        mask[:, i] = mask[at, parent] & (parent >= 0)[:, None]
        mask[:, i, i] = True
    if case["blind"]:
        mask[:, -1] = False
    mask = torch.from_numpy(mask).cuda()
    return mask[0] if trees == 1 and case["mask"] == "shared" else mask


def _scales(x, dims):
    """Exponents of the least powers of two that bring the largest of a group within 448, and the E4M3 codes."""
    top = x.abs().amax(dims, keepdim=True)
    mantissa, exponent = torch.frexp(top)
    e = torch.where(top == 0, 0, exponent - 9 + (mantissa > 0.875).to(exponent.dtype))
    return e, torch.ldexp(x, -e).to(torch.float8_e4m3fn)


def _tree_pages(case, k, v, lens, seed):
    """The rows' pages, on scattered places, and their block table; for fp8 also codes [.., page, heads, dim]
    and scales of the blocks wholly before the window: keys' for each channel, values' for each token."""
    B, P, H, D = case["batch"], case["page"], case["heads"], case["dim"]
    blocks = -(-k.shape[1] // P)
    pad = blocks * P - k.shape[1]
    order = torch.randperm(B * blocks, generator=_generator(seed, 5), device="cuda")
    state = dict(table=order.reshape(B, blocks), lens=torch.from_numpy(lens).cuda())
    for name, x in (("key", k), ("value", v)):
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad)).reshape(B * blocks, P, H, D)
        pages = torch.empty_like(x)
        pages[order] = x
        state[name + "_pages"] = pages
        if case["fp8"]:
            e, codes = _scales(x.float(), 1 if name == "key" else 3)
            state[name + "_codes"], state[name + "_scales"] = torch.empty_like(codes), torch.empty_like(e)
            state[name + "_codes"].view(torch.uint8)[order] = codes.view(torch.uint8)
            state[name + "_scales"][order] = e
    return state


def _pool(case, k, v, lens, seed):
    from barqtrain_amd.paged import PagePool, QuantPagePool

    blocks = -(-(case["ctx"] + case["nodes"]) // case["page"])
    geometry = dict(max_batch=case["batch"], max_blocks=blocks, page_size=case["page"], kv_heads=case["heads"],
                    head_dim=case["dim"], dtype=DTYPES[case["dtype"]], device="cuda")
    if case["fp8"]:
        pool = QuantPagePool(window=WINDOW, **geometry)
    else:
        order = torch.randperm(case["batch"] * (blocks + 1), generator=_generator(seed, 5), device="cuda")
        pool = PagePool(page_order=order, **geometry)
    k, v = k.transpose(1, 2), v.transpose(1, 2)
    if (lens == lens[0]).all():
        pool.append(k, v)
    else:
        for row, n in enumerate(lens.tolist()):
            pool.append_rows([row], k[row:row + 1, :, :n], v[row:row + 1, :, :n])
    return pool


def _map_lengths(case, seed=0):
    """Host lengths of a map pass: the prompts, then the accepted tokens of each step; in the seed's order."""
    draws = np.random.RandomState(case["batch"] + case["steps"])
    lengths = [_lengths(case)] + [draws.randint(0, 6, case["batch"]) for _ in range(case["steps"])]
    order = np.random.RandomState((seed * 29 + 1) & 0x7FFFFFFF).permutation(case["batch"])
    return [n[order] for n in lengths]


def _map_rows(case, seed):
    """The requests' rows, among SPARE more."""
    held = case["batch"] + SPARE
    return (np.random.RandomState(case["batch"]).permutation(held)[:case["batch"]] + seed) % held


def _counts(case):
    """Tokens that each row of a write pass stores."""
    draws = np.random.RandomState(case["batch"] * 3 + case["nodes"])
    if case["nodes"]:
        counts = draws.randint(0, min(case["ctx"], case["nodes"]) + 1, case["batch"])
    else:
        counts = draws.randint(max(1, case["ctx"] // 4), case["ctx"] + 1, case["batch"])
    counts[draws.randint(case["batch"])] = min(case["ctx"], case["nodes"] or case["ctx"])
    return counts


def prepare(case, seed):
    kind, B, P = case["kind"], case["batch"], case["page"]
    if kind == "tree":
        lens = _lengths(case)
        k, v = _kv(case, seed, 0, B, case["ctx"])
        nk, nv = _kv(case, seed, 1, B, case["nodes"])
        q = torch.randn((B, case["nodes"], case["heads"] * case["group"], case["dim"]), generator=_generator(seed, 2),
                        device="cuda")
        state = dict(case=case, query=(q * 0.3).to(DTYPES[case["dtype"]]).transpose(1, 2), key=nk.transpose(1, 2),
                     value=nv.transpose(1, 2), mask=_mask(case, seed))
        if own:
            state["pool"] = _pool(case, k, v, lens, seed)
        else:
            state.update(_tree_pages(case, k, v, lens, seed))
        return state
    if kind == "map":
        lengths = _map_lengths(case, seed)
        blocks = -(-int(sum(lengths).max()) // P)
        rows = _map_rows(case, seed)
        held = B + SPARE
        state = dict(case=case, lengths=[n.tolist() for n in lengths], rows=rows.tolist(), blocks=blocks)
        if own:
            from barqtrain_amd.paged import PagePool

            # pages of one element: their contents take no part
            state["pools"] = [PagePool(max_batch=held, max_blocks=blocks, page_size=P, kv_heads=1, head_dim=1,
                                       dtype=torch.bfloat16, device="cuda") for _ in range(case["layers"])]
        else:
            i32 = dict(dtype=torch.int32, device="cuda")
            state.update(lengths_gpu=[torch.tensor(n, device="cuda") for n in state["lengths"]],
                         rows_gpu=torch.tensor(state["rows"], device="cuda"),
                         tables=torch.empty((case["layers"], held, blocks), **i32),
                         free=torch.empty((case["layers"], held * (blocks + 1)), **i32))
        return state
    counts = _counts(case)
    total = int(counts.sum())
    slots, index = _write_places(case, counts, seed)
    k, v = _kv(case, seed, 3, B, case["nodes"]) if case["nodes"] else _kv(case, seed, 3, 1, total)
    state = dict(case=case, slots=slots, index=index, key=k.flatten(0, 1), value=v.flatten(0, 1))
    blocks = -(-case["ctx"] // P) + 1
    if own:
        from barqtrain_amd.paged import PagePool

        pool = PagePool(max_batch=B, max_blocks=blocks, page_size=P, kv_heads=case["heads"], head_dim=case["dim"],
                        dtype=DTYPES[case["dtype"]], device="cuda", num_pages=B * blocks)
        pool.key_pages.zero_()
        pool.value_pages.zero_()
        state["pool"] = pool
    else:
        shape = (B * blocks, P, case["heads"], case["dim"])
        state.update(key_pages=torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda"),
                     value_pages=torch.zeros(shape, dtype=DTYPES[case["dtype"]], device="cuda"))
    return state


def _write_places(case, counts, seed):
    """The slots of each row's tokens, from an odd position on over scattered pages, and which node each is."""
    B, P = case["batch"], case["page"]
    blocks = -(-case["ctx"] // P) + 1
    draws = np.random.RandomState((seed * 23 + B) & 0x7FFFFFFF)
    table = draws.permutation(B * blocks).reshape(B, blocks)
    slots, index = [], []
    for b, n in enumerate(counts.tolist()):
        at = np.arange(n) + (5 * b) % P
        slots.append(table[b, at // P] * P + at % P)
        if case["nodes"]:
            index.append(b * case["nodes"] + np.sort(draws.permutation(case["nodes"])[:n]))
    index = torch.from_numpy(np.concatenate(index).astype(np.int64)).cuda() if case["nodes"] else None
    return torch.from_numpy(np.concatenate(slots).astype(np.int64)).cuda(), index


# --------------------------------------------------------------------------------------- passes
def run(state):
    kind = state["case"]["kind"]
    if kind == "tree":
        if own:
            return state["pool"].attend_tree(state["query"], state["key"], state["value"], state["mask"])
        return _tree_plain(state)
    if kind == "map":
        return _map_own(state) if own else _map_plain(state)
    if own:
        pool = state["pool"]
        pool.write_slots(state["slots"], state["key"], state["value"], state["index"])
        return [pool.key_pages, pool.value_pages]
    at = state["slots"]
    for name in ("key", "value"):
        x = state[name] if state["index"] is None else state[name][state["index"]]
        state[name + "_pages"].flatten(0, 1)[at] = x
    return [state["key_pages"], state["value_pages"]]


def _map_own(state):
    from barqtrain_amd.paged import map_slots_layers, reset_layers

    pools = state["pools"]
    reset_layers(pools)
    maps = [map_slots_layers(pools, n, state["rows"]) for n in state["lengths"]]
    return [[[m.slots, m.positions, m.requests, m.offsets] for m in maps], pools[0].seq_lens,
            [p.block_table for p in pools]]


def _map_plain(state):
    P, blocks = state["case"]["page"], state["blocks"]
    tables, free, rows = state["tables"], state["free"], state["rows_gpu"]
    pages = free.shape[1]
    tables.fill_(-1)
    free.copy_(torch.arange(pages - 1, -1, -1, device=free.device)[None])
    lens = torch.zeros(tables.shape[1], dtype=torch.int64, device=free.device)
    taken, out = torch.zeros((), dtype=torch.int64, device=free.device), []
    for n, host in zip(state["lengths_gpu"], state["lengths"]):
        total = sum(host)
        offsets = torch.cat([n.new_zeros(1), n.cumsum(0)])
        old = lens[rows]
        new = old + n
        first, end = (old + P - 1) // P, (new + P - 1) // P
        before = (end - first).cumsum(0) - (end - first)  # new blocks of the requests before
        j = torch.arange(blocks, device=n.device)[None]
        is_new = (j >= first[:, None]) & (j < end[:, None])
        rank = taken + before[:, None] + j - first[:, None]
        page = free[:, (pages - 1 - rank).clamp(min=0)]
        tables[:, rows] = torch.where(is_new, page, tables[:, rows])
        lens[rows] = new
        taken = taken + (end - first).sum()
        token = torch.arange(total, device=n.device)
        request = torch.searchsorted(offsets[1:], token, right=True)
        position = old[request] + token - offsets[request]
        slots = tables[:, rows[request], position // P].long() * P + position % P
        out.append([slots, position.int(), request.int(), offsets.int()])
    return [out, lens.int(), list(tables.unbind(0))]


def _read(state, name):
    """The rows' cached keys or values in 32 bits, [batch, positions, heads, dim]."""
    case, table = state["case"], state["table"]
    x = state[name + "_pages"][table].float()  # [batch, blocks, page, heads, dim]
    if case["fp8"]:
        read = torch.ldexp(state[name + "_codes"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float(),
                           state[name + "_scales"][table])
        cold = (state["lens"] - WINDOW).clamp(min=0) // case["page"]
        quantised = torch.arange(table.shape[1], device=table.device)[None] < cold[:, None]
        x = torch.where(quantised[:, :, None, None, None], read.to(DTYPES[case["dtype"]]).float(), x)
    return x.flatten(1, 2)


def _tree_plain(state):
    q, nodes = state["query"], state["case"]["nodes"]
    B, Hq, T, D = q.shape
    H = state["case"]["heads"]
    k, v = _read(state, "key"), _read(state, "value")
    cached = torch.arange(k.shape[1], device=q.device)[None] < state["lens"][:, None]
    v = torch.where(cached[:, :, None, None], v, 0.0)
    mask = state["mask"]
    if mask is None:
        mask = torch.ones((nodes, nodes), dtype=torch.bool, device=q.device).tril()
    seen = torch.cat([cached[:, None].expand(B, T, -1), mask.expand(B, T, T)], dim=2)[:, None, None]
    k = torch.cat([k.transpose(1, 2), state["key"].float()], dim=2)  # [batch, heads, positions, dim]
    v = torch.cat([v.transpose(1, 2), state["value"].float()], dim=2)
    s = torch.matmul(q.float().reshape(B, H, -1, D), k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    s = s.reshape(B, H, Hq // H, T, -1).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.flatten(2, 3), v).reshape(B, H, Hq // H, T, D) / torch.where(total == 0, 1.0, total)
    return out.reshape(B, Hq, T, D).to(q.dtype)


# ---------------------------------------------------------------------------------- what it costs
def work(case):
    B = case["batch"]
    if case["kind"] == "map":
        L, total = case["layers"], int(sum(int(n.sum()) for n in _map_lengths(case)))
        rows = sum(_map_lengths(case))
        blocks = -(-int(rows.max()) // case["page"])
        new = int((-(-rows // case["page"])).sum())
        # the emptied tables and free lists, then a page read and entered for each new block, a slot a token and
        # layer, a position and a request a token
        return {"bytes": 4 * L * (B + SPARE) * (2 * blocks + 1) + 8 * L * new + 8 * L * total + 8 * total + 8 * B, "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    row = 2 * case["heads"] * case["dim"] * size
    if case["kind"] == "write":
        n = int(_counts(case).sum())
        return {"bytes": n * (2 * row + 8 + 8 * bool(case["nodes"])), "flops": 0}
    lens, T, Hq = _lengths(case), case["nodes"], case["heads"] * case["group"]
    cold = np.maximum(lens - WINDOW, 0) // case["page"] * case["page"] * case["fp8"]
    scales = cold // case["page"] * case["heads"] * (case["dim"] + case["page"])
    stored = int(((lens - cold) * row + cold * (row // 2) + scales).sum())
    trees = {"chain": 0, "shared": 1, "rows": B}[case["mask"]]
    return {"bytes": stored + B * T * (row + 2 * Hq * case["dim"] * size) + trees * T * T,
            "flops": 4 * Hq * T * case["dim"] * int((lens + T).sum())}


# ------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["kind"] == "write":
        return None  # values are stored as they are
    if case["kind"] == "map":
        return _map_exact(case, seed)
    lens, P, T = _lengths(case), case["page"], case["nodes"]
    k, v = _kv(case, seed, 0, case["batch"], case["ctx"])
    nk, nv = _kv(case, seed, 1, case["batch"], T)
    q = torch.randn((case["batch"], T, case["heads"] * case["group"], case["dim"]), generator=_generator(seed, 2),
                    device="cuda")
    q = (q * 0.3).to(DTYPES[case["dtype"]]).double()
    mask = _mask(case, seed)
    out = torch.zeros((case["batch"], q.shape[2], T, case["dim"]), dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens.tolist()):
        allowed = torch.ones((T, T), dtype=torch.bool, device="cuda").tril() if mask is None else mask
        allowed = allowed[b] if allowed.dim() == 3 else allowed
        cold = max(n - WINDOW, 0) // P * P if case["fp8"] else 0
        for h in range(case["heads"]):
            rows = []
            for x, dims in ((k, 1), (v, 2)):  # a group is a channel of a page's keys, a token of its values
                x = x[b, :n, h]
                if cold:
                    e, codes = _scales(x[:cold].float().reshape(-1, P, case["dim"]), dims)
                    read = torch.ldexp(codes.float(), e).reshape(cold, -1).to(x.dtype)
                    x = torch.cat([read, x[cold:]])
                rows.append(x.double())
            keys, values = torch.cat([rows[0], nk[b, :, h].double()]), torch.cat([rows[1], nv[b, :, h].double()])
            seen = torch.cat([torch.ones((T, n), dtype=torch.bool, device="cuda"), allowed], dim=1)
            for g in range(case["group"]):
                s = (q[b, :, h * case["group"] + g] @ keys.t()) / math.sqrt(case["dim"])
                p = torch.softmax(s.masked_fill(~seen, -math.inf), dim=1).nan_to_num(0.0)
                out[b, h * case["group"] + g] = p @ values
    return out


def _map_exact(case, seed):
    """The same by counting: every token of every request takes the next position of its row."""
    B, P, L = case["batch"], case["page"], case["layers"]
    lengths, rows = _map_lengths(case, seed), _map_rows(case, seed)
    blocks = -(-int(sum(lengths).max()) // P)
    table = np.full((B + SPARE, blocks), -1, dtype=np.int32)
    lens, page, out = np.zeros(B + SPARE, dtype=np.int64), 0, []
    for n in lengths:
        slots, positions, requests = [], [], []
        for i, count in enumerate(n.tolist()):
            at = np.arange(lens[rows[i]], lens[rows[i]] + count)
            fresh = np.unique(at[table[rows[i], at // P] < 0] // P)
            table[rows[i], fresh] = np.arange(page, page + len(fresh))
            page += len(fresh)
            slots.append(table[rows[i], at // P].astype(np.int64) * P + at % P)
            positions.append(at)
            requests.append(np.full(count, i))
            lens[rows[i]] += count
        join = lambda parts: np.concatenate(parts).astype(np.int32)  # noqa: E731
        out.append([np.repeat(np.concatenate(slots)[None], L, 0), join(positions), join(requests),
                    np.concatenate([[0], np.cumsum(n)]).astype(np.int32)])
    return [out, lens.astype(np.int32), [table] * L]
