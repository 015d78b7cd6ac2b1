"""Slot maps, stores through them and tree attention on pools in host memory, their refusals, and the C ABI of
include/barq_ragged.h without a GPU."""

import ctypes
import subprocess
import types

import numpy as np
import pytest
import torch

from barqtrain_amd import _capi, build
from barqtrain_amd.kv_cache import create_paged_kv_cache
from barqtrain_amd.paged import (
    PagedKVCapacityError,
    PagedKVPoolExhausted,
    PagePool,
    QuantPagePool,
    map_slots_layers,
)
from tree_ref import tree_bound, tree_reference


def pool_of(batch=4, blocks=6, page=4, heads=2, dim=8, dtype=torch.float32, pages=None, cls=PagePool, **kw):
    pool = cls(max_batch=batch, max_blocks=blocks, page_size=page, kv_heads=heads, head_dim=dim, dtype=dtype,
               device="cpu", num_pages=pages, **kw)
    pool.key_pages.zero_()
    pool.value_pages.zero_()
    return pool


def state_of(pool):
    return [t.clone() for t in pool.tensors] + [pool.lens.copy(), pool.hw.copy(), pool.free_count]


def same_state(a, b):
    return all(np.array_equal(np.asarray(x), np.asarray(y)) for x, y in zip(a, b))


def packed(pool, total, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn((total, pool.kv_heads, pool.head_dim), generator=g).to(pool.dtype)
    return k, torch.randn((total, pool.kv_heads, pool.head_dim), generator=g).to(pool.dtype)


# --------------------------------------------------------------------------------------- C ABI
@pytest.fixture(scope="module")
def built():
    if not build.is_built():
        build.build()
    return _capi.load_library()


def test_library_exports_the_ragged_header(built):
    declared = _capi.header_functions(_capi.RAGGED_HEADER)
    assert declared == sorted(_capi._RAGGED_SIGNATURES)
    out = subprocess.run(["nm", "-D", "--defined-only", str(build.lib_path())], capture_output=True, text=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T barq_" in line}
    assert exported == set(declared) | set(_capi.header_functions())


def fake_pool(**kw):
    """A plausible descriptor whose addresses are never followed: only calls that return before a launch."""
    addr = 0x7F0000000000
    pool = _capi.BarqKVPool(*(addr + i * 2**32 for i in range(8)), 64, 4, 8, 16, 8, 128, 2)
    for name, value in kw.items():
        setattr(pool, name, value)
    return pool


def test_invalid_arguments_are_refused_before_any_launch(built):
    addr = ctypes.c_void_p(0x7F0000000000)
    i32 = lambda *v: (ctypes.c_int32 * max(len(v), 1))(*v)  # noqa: E731

    def mapped(pools, n_pools, rows, lengths, n, slots=addr, stride=1 << 20):
        return built.barq_map_slots(pools, n_pools, rows, lengths, n, slots, stride, None, None, None, None)

    good = fake_pool()
    assert mapped(None, 1, None, i32(1), 1) == 1
    assert mapped(ctypes.byref(good), 0, None, i32(1), 1) == 1
    assert mapped(ctypes.byref(good), 1, None, i32(1), 0) == 0                      # no requests: nothing to do
    assert mapped(ctypes.byref(good), 1, None, None, 1) == 1
    assert mapped(ctypes.byref(good), 1, None, i32(-1), 1) == 1
    assert mapped(ctypes.byref(good), 1, None, i32(129), 1) == 1                    # past the row's capacity
    assert mapped(ctypes.byref(good), 1, None, i32(1, 1, 1, 1, 1), 5) == 1          # more requests than rows
    assert mapped(ctypes.byref(good), 1, i32(4), i32(1), 1) == 1
    assert mapped(ctypes.byref(good), 1, i32(-1), i32(1), 1) == 1
    assert mapped(ctypes.byref(good), 1, i32(2, 2), i32(1, 1), 2) == 1
    assert mapped(ctypes.byref(good), 1, None, i32(1), 1, None) == 1
    assert mapped((_capi.BarqKVPool * 2)(good, good), 2, None, i32(1), 1) == 1      # one pool twice
    other = fake_pool(page_size=8, ctrl=0x7FF000000000, seq_lens=0x7FF100000000)
    assert mapped((_capi.BarqKVPool * 2)(good, other), 2, None, i32(1), 1) == 1

    def write(pool, slots=addr, index=None, count=1, key=addr, value=addr, tokens=1, sn=1024, sh=128):
        return built.barq_write_slots(ctypes.byref(pool), slots, index, count, key, value, tokens, sn, sh, None)

    assert write(good, count=0, key=None) == 0
    assert write(good, slots=None) == 1 and write(good, key=None) == 1 and write(good, value=None) == 1
    assert write(good, count=-1) == 1 and write(good, count=2) == 1 and write(good, tokens=0) == 1
    assert write(good, sn=-1) == 1 and write(fake_pool(elem_bytes=3)) == 1

    def tree(pool, cold=None, nodes=4, heads=32, batch=4, q=addr, st=128, flags=0, ws=addr, ws_bytes=1 << 40, out=addr,
             max_seq=0):
        return built.barq_tree_attention(ctypes.byref(pool), cold, q, batch, heads, nodes, 0, st, 0, addr, addr, 0, 128, 0,
                                         None, 0, 0, 0, out, 0, 128, 0, 1.0, max_seq, 0, flags, ws, ws_bytes, None)

    assert tree(fake_pool(elem_bytes=4)) == 1 and tree(fake_pool(head_dim=96)) == 1
    assert tree(good, nodes=0) == 1 and tree(good, nodes=257) == 1 and tree(good, heads=30) == 1 and tree(good, batch=5) == 1
    assert tree(good, q=ctypes.c_void_p(0x7F0000000008)) == 1 and tree(good, st=12) == 1
    assert tree(good, out=ctypes.c_void_p(0x7F0000000004)) == 1 and tree(good, flags=4) == 1
    assert tree(good, max_seq=-1) == 1
    long = fake_pool(max_blocks=512)
    assert built.barq_tree_attention_workspace_bytes(ctypes.byref(long), 0, 1, 32, 4, 0, 0) > 0
    assert built.barq_tree_attention_workspace_bytes(ctypes.byref(long), 0, 1, 33, 4, 0, 0) == -1
    assert tree(long, batch=1, ws_bytes=0) == 1 and tree(long, batch=1, ws=None) == 1
    cold = _capi.BarqKVCold(*([0x7F0000000000] * 6), 16, 128, 1)  # fp16 codes of a bf16 call
    assert tree(good, cold=ctypes.byref(cold)) == 1
    cold.element_type = 0
    assert tree(fake_pool(page_size=8), cold=ctypes.byref(cold)) == 1
    assert tree(fake_pool(head_dim=256), cold=ctypes.byref(cold)) == 1


# --------------------------------------------------------------------------------------- slot maps
@pytest.mark.parametrize("page", [1, 4, 5])
def test_mapped_slots_are_the_append_s(page):
    """Mapped and stored tokens leave the pool as append_rows leaves it, and read back the same."""
    a, b = (pool_of(page=page, blocks=24 // page) for _ in range(2))
    draws = np.random.RandomState(page)
    for step in range(4):
        rows = draws.permutation(4)[:draws.randint(1, 5)].tolist()
        lengths = draws.randint(0, 6, len(rows)).tolist()
        k, v = packed(a, sum(lengths), step)
        got = a.map_slots(lengths, rows)
        a.write_slots(got.slots, k, v)
        at = 0
        for i, (r, n) in enumerate(zip(rows, lengths)):
            assert got.offsets[i] == at and (got.requests[at:at + n] == i).all()
            assert got.positions[at:at + n].tolist() == list(range(int(b.lens[r]), int(b.lens[r]) + n))
            b.append_rows([r], *(t[at:at + n].transpose(0, 1)[None] for t in (k, v)))
            at += n
        assert got.offsets[-1] == at == len(got.slots)
        assert same_state(state_of(a), state_of(b))
        if step == 1:
            a.crop(4, 3), b.crop(4, 3)
        if step == 2:
            a.free_rows([1]), b.free_rows([1])
    assert a.errors() == 0


def test_map_slots_of_layers_is_each_pool_s():
    one, layers = [pool_of() for _ in range(3)], [pool_of() for _ in range(3)]
    got = map_slots_layers(layers, [3, 0, 7], [2, 0, 1])
    for l, p in enumerate(one):
        want = p.map_slots([3, 0, 7], [2, 0, 1])
        assert torch.equal(got.slots[l], want.slots)
        assert all(torch.equal(x, y) for x, y in zip(got[1:], want[1:]))
        assert same_state(state_of(layers[l]), state_of(p))


def test_map_slots_refusals_change_nothing():
    pool = pool_of(pages=7)
    pool.map_slots([5, 3])
    before = state_of(pool)
    cases = [
        (ValueError, dict(lengths=[1, 2], rows=[0])), (ValueError, dict(lengths=[1, 2], rows=[1, 1])),
        (IndexError, dict(lengths=[1], rows=[4])), (IndexError, dict(lengths=[1], rows=[-1])),
        (IndexError, dict(lengths=[1] * 5)), (ValueError, dict(lengths=[-1])), (ValueError, dict(lengths=np.array([1.5]))),
        (ValueError, dict(lengths=[1.5])), (ValueError, dict(lengths=[2], rows=[0.5])), (ValueError, dict(lengths=torch.ones((1, 1), dtype=torch.int64))),
        (PagedKVCapacityError, dict(lengths=[20])), (PagedKVCapacityError, dict(lengths=[4], max_length=8)),
        (PagedKVPoolExhausted, dict(lengths=[0, 0, 16, 4])),
    ]
    for error, kw in cases:
        with pytest.raises(error):
            pool.map_slots(**kw)
        assert same_state(state_of(pool), before)
    with pytest.raises(ValueError):
        map_slots_layers([], [1])
    with pytest.raises(ValueError, match="twice"):
        map_slots_layers([pool, pool], [1])
    with pytest.raises(ValueError, match="page size"):
        map_slots_layers([pool, pool_of(page=8)], [1])
    with pytest.raises(ValueError, match="different lengths"):
        map_slots_layers([pool, pool_of()], [1])
    assert same_state(state_of(pool), before)
    # what a call leaves out keeps its state: a full row may stand by with length 0
    pool.map_slots([0, 2], max_length=5)
    assert pool.map_slots([]).slots.numel() == 0
    with pytest.raises(PagedKVCapacityError):
        pool.map_slots([1], max_length=5)


def test_write_slots_refusals_and_what_is_passed_over():
    pool = pool_of()
    k, v = packed(pool, 5)
    slots = torch.tensor([3, -1, 9, 10**9, 0])
    pool.write_slots(slots, k, v, torch.tensor([4, 0, 9, 1, 2]))
    flat = pool.key_pages.flatten(0, 1)
    assert torch.equal(flat[3], k[4]) and torch.equal(flat[0], k[2]) and (flat[9] == 0).all()
    assert pool.errors() == 4
    before = state_of(pool)
    bad = [(slots, k[:, :1], v[:, :1]), (slots, k, v[:4]), (slots, k.double(), v.double()), (slots.int(), k, v),
           (slots[None], k, v), (slots, k[:4], v[:4]), (slots, k, v, slots[:4]), (slots, k, v, slots.float()),
           (slots, k[:0], v[:0], slots)]
    for args in bad:
        with pytest.raises(ValueError):
            pool.write_slots(*args)
    assert same_state(state_of(pool), before)
    pool.write_slots(slots[:0], k, v)


# --------------------------------------------------------------------------------------- tree attention
def tree_inputs(pool, batch, nodes, group, seed=0):
    g = torch.Generator().manual_seed(seed)
    shape = (batch, nodes, pool.kv_heads, pool.head_dim)
    q = torch.randn((batch, nodes, pool.kv_heads * group, pool.head_dim), generator=g).to(pool.dtype)
    k, v = (torch.randn(shape, generator=g).to(pool.dtype) for _ in range(2))
    return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)


@pytest.mark.parametrize("mask", ["chain", "shared", "rows"])
def test_host_tree_attention(mask):
    pool = pool_of(dim=16)
    k, v = packed(pool, 13)
    pool.write_slots(pool.map_slots([5, 0, 8]).slots, k, v)
    q, nk, nv = tree_inputs(pool, 3, 6, 2)
    g = torch.Generator().manual_seed(1)
    m = {"chain": None, "shared": torch.rand((6, 6), generator=g) < 0.4, "rows": torch.rand((3, 6, 6), generator=g) < 0.4}[mask]
    if mask == "rows":
        m[1, 2] = False  # an empty row's node that sees no node: nothing at all
    got = pool.attend_tree(q, nk, nv, m)
    ko, vo = pool.gather(3)
    out, weight, score = tree_reference(q, ko, vo, pool.lens, nk, nv, m, 16**-0.5)
    assert got.shape == q.shape and (got.double() - out).abs().le(tree_bound(out, weight, score, torch.float32, 14, 16)).all()
    if mask == "rows":
        assert (got[1, :, 2] == 0).all()


def test_tree_attention_refusals():
    pool = pool_of(dim=16)
    q, k, v = tree_inputs(pool, 2, 3, 2)
    mask = torch.ones((3, 3), dtype=torch.bool)
    big = tree_inputs(pool, 1, 257, 1)
    bad = [(q[..., :8], k, v), (q[:, :3], k, v), (q, k[:1], v), (q, k, v[:, :, :2]), (q.double(), k, v), (q, k, v, mask.int()),
           (q, k, v, mask[:2]), (q, k, v, mask.expand(3, 3, 3)), (q[0], k, v), big, tree_inputs(pool, 5, 1, 1)]
    for args in bad:
        with pytest.raises(ValueError):
            pool.attend_tree(*args)
    with pytest.raises(ValueError):
        pool.attend_tree(q, k, v, out=torch.empty((1, 1)))
    with pytest.raises(ValueError):
        pool.attend_tree(q, k, v, out_dtype=torch.float16)
    with pytest.raises(ValueError):
        pool.attend_tree(q, k, v, max_seq=25)
    assert pool.attend_tree(q[:0], k[:0], v[:0]).shape == (0, 4, 3, 16)


def run_steps(cache, layers, device, batch=3, nodes=5, steps=3, seed=0):
    """A run as a program makes it: ragged prompts, then per step tree attention in every layer and the accepted
    paths stored.  Returns the outputs and each row's stored (K, V) by layer, kept apart."""
    g = torch.Generator().manual_seed(seed)
    draws = np.random.RandomState(seed)
    shape = lambda n: (layers, n, 2, 64)  # noqa: E731
    prompts = [7, 1, 4]
    k, v = (torch.randn(shape(sum(prompts)), generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    got = cache.map_slots(prompts)
    kept = [[[k[l][got.requests.cpu() == b], v[l][got.requests.cpu() == b]] for b in range(batch)] for l in range(layers)]
    for l in range(layers):
        cache.layers[l].write_slots(got.slots[l], k[l], v[l])
    outs = []
    for _ in range(steps):
        parents = [draws.randint(-1, i) if i else -1 for i in range(nodes)]
        mask = torch.zeros((nodes, nodes), dtype=torch.bool)
        for i, p in enumerate(parents):
            mask[i] = mask[p] if p >= 0 else False
            mask[i, i] = True
        q = torch.randn((layers, batch, nodes, 4, 64), generator=g).to(torch.bfloat16).to(device)
        nk, nv = (torch.randn((layers, batch, nodes, 2, 64), generator=g).to(torch.bfloat16).to(device) for _ in range(2))
        for l in range(layers):
            outs.append((cache.layers[l].attend_tree(q[l].transpose(1, 2), nk[l].transpose(1, 2), nv[l].transpose(1, 2),
                                                     mask.to(device)),
                         q[l].transpose(1, 2), nk[l].transpose(1, 2), nv[l].transpose(1, 2), mask,
                         [[t.clone() for t in kept[l][b]] for b in range(batch)]))
        paths = [sorted(draws.permutation(nodes)[:draws.randint(0, nodes + 1)].tolist()) for _ in range(batch)]
        index = torch.tensor([b * nodes + i for b, path in enumerate(paths) for i in path], dtype=torch.int64)
        got = cache.map_slots([len(p) for p in paths])
        for l in range(layers):
            cache.layers[l].write_slots(got.slots[l], nk[l].flatten(0, 1), nv[l].flatten(0, 1), index.to(device))
            for b, path in enumerate(paths):
                kept[l][b] = [torch.cat([old, new[l, b][path]]) for old, new in zip(kept[l][b], (nk, nv))]
    return outs, kept


def check_run(cache, outs, kept, dim=64):
    for out, q, nk, nv, mask, rows in outs:
        lens = [r[0].shape[0] for r in rows]
        k, v = (torch.nn.utils.rnn.pad_sequence([r[i] for r in rows], batch_first=True).transpose(1, 2) for i in (0, 1))
        ref, weight, score = tree_reference(q, k, v, lens, nk, nv, mask, dim**-0.5)
        bound = tree_bound(ref, weight, score, out.dtype, max(lens) + mask.shape[0], dim)
        assert (out.double().cpu() - ref).abs().le(bound).all()
    for l, layer in enumerate(cache.layers):
        k, v = layer.current_tensors()
        for b, (kk, vv) in enumerate(kept[l]):
            n = kk.shape[0]
            assert layer.pool.lens[b] == n
            assert torch.equal(k[b, :, :n].transpose(0, 1), kk) and torch.equal(v[b, :, :n].transpose(0, 1), vv)


def make_cache(device, layers=2, batch=3, **kw):
    cache = create_paged_kv_cache(types.SimpleNamespace(num_hidden_layers=layers), max_batch_size=batch,
                                  max_cache_len=64, page_size=16, **kw)
    like = torch.empty((batch, 2, 0, 64), dtype=torch.bfloat16, device=device)
    for layer in cache.layers:
        layer.lazy_initialization(like)
    return cache


def test_speculative_steps_on_the_host():
    cache = make_cache("cpu")
    check_run(cache, *run_steps(cache, 2, "cpu"))


def test_cache_map_slots_needs_its_layers():
    cache = create_paged_kv_cache(types.SimpleNamespace(num_hidden_layers=2), max_batch_size=2, max_cache_len=32)
    with pytest.raises(ValueError):
        cache.map_slots([1, 1])


def test_quantised_pools_quantise_what_a_map_left_behind():
    """Blocks that mapped tokens pushed out of the window are quantised by the next map (or append)."""
    pool = pool_of(cls=QuantPagePool, page=4, blocks=8, dim=8, window=4, chunk=8)
    other = pool_of(cls=QuantPagePool, page=4, blocks=8, dim=8, window=4, chunk=8)
    for step, n in enumerate([6, 6, 5, 1]):
        k, v = packed(pool, 2 * n, step)
        pool.write_slots(pool.map_slots([n, n]).slots, k, v)
        other.append(*(t.reshape(2, n, 2, 8).transpose(1, 2) for t in (k, v)))
        if step >= 2:  # 12 positions, 4 of them in the window: two blocks of 4
            assert (pool.cold_blocks > 0)[:2].all()
    pool._settle()
    for x, y in zip(pool.gather(2), other.gather(2)):
        assert torch.equal(x, y)
    assert pool.errors() == 0
