"""Slot maps and stores through them on the GPU: against the host pool's, and against appends."""

import numpy as np
import pytest
import torch

from barqtrain_amd.paged import PagedKVCapacityError, PagedKVPoolExhausted, PagePool, QuantPagePool, map_slots_layers, reset_layers
from test_ragged import check_run, make_cache, run_steps

pytestmark = pytest.mark.gpu


def pool_of(device, batch=4, blocks=6, page=4, heads=2, dim=8, dtype=torch.bfloat16, cls=PagePool, **kw):
    pool = cls(max_batch=batch, max_blocks=blocks, page_size=page, kv_heads=heads, head_dim=dim, dtype=dtype,
               device=device, **kw)
    pool.key_pages.zero_()
    pool.value_pages.zero_()
    return pool


def same_metadata(gpu, host):
    for a, b in zip(gpu.tensors[2:6], host.tensors[2:6]):
        assert torch.equal(a.cpu(), b)
    assert gpu.ctrl[0].item() == host.ctrl[0].item() and gpu.errors() == host.errors() == 0
    assert (gpu.ctrl[32:] == 0).all()
    assert (gpu.lens == host.lens).all() and (gpu.hw == host.hw).all() and gpu.free_count == host.free_count


@pytest.mark.parametrize("page,batch,longest", [(1, 3, 5), (3, 7, 9), (16, 64, 40), (16, 300, 12), (16, 520, 3), (64, 5, 5000)])
def test_map_slots_matches_the_host_pool(hip, page, batch, longest):
    blocks = -(-3 * longest // page)
    order = torch.randperm(batch * (blocks + 1), generator=torch.Generator().manual_seed(page))
    gpu, host = (pool_of(d, batch, blocks, page, 1, 1, page_order=order) for d in ("cuda", "cpu"))
    draws = np.random.RandomState(batch)
    for step in range(3):
        rows = draws.permutation(batch)[:draws.randint(1, batch + 1)].tolist()
        if step == 2:
            rows = None
        lengths = draws.randint(0, longest + 1, batch if rows is None else len(rows)).tolist()
        a, b = gpu.map_slots(lengths, rows), host.map_slots(lengths, rows)
        assert all(torch.equal(x.cpu(), y) and x.dtype == y.dtype for x, y in zip(a, b))
        same_metadata(gpu, host)
        if step == 0:  # stale mapped blocks past a row's length, and freed rows
            gpu.crop(batch, longest // 2), host.crop(batch, longest // 2)
            gpu.free_rows([0, batch - 1]), host.free_rows([0, batch - 1])
            assert gpu.free_count == host.free_count
            host.free_pages.copy_(gpu.free_pages.cpu())  # the freed pages' order on the stack is not fixed


@pytest.mark.parametrize("layers", [1, 2, 32, 35])
def test_map_slots_layers(hip, layers):
    gpu = [pool_of("cuda", 5, 9) for _ in range(layers)]
    host = pool_of("cpu", 5, 9)
    for lengths, rows in (([7, 0, 30], [4, 1, 0]), ([1, 1, 1, 1, 1], None), ([2], [2])):
        a, b = map_slots_layers(gpu, lengths, rows), host.map_slots(lengths, rows)
        assert a.slots.shape == (layers, sum(lengths))
        for l in range(layers):
            assert torch.equal(a.slots[l].cpu(), b.slots)
            same_metadata(gpu[l], host)
        assert all(torch.equal(x.cpu(), y) for x, y in zip(a[1:], b[1:]))
    reset_layers(gpu)
    assert map_slots_layers(gpu, [3]).slots[layers - 1].tolist() == [0, 1, 2]


def test_map_slots_refusals_change_nothing(hip):
    pool = pool_of("cuda", num_pages=7)
    pool.map_slots([5, 3])
    before = [t.clone() for t in pool.tensors[2:]], pool.lens.copy(), pool.free_count
    for error, args in ((ValueError, ([1, 2], [1, 1])), (IndexError, ([1], [4])), (IndexError, ([1] * 5,)), (ValueError, ([-1],)),
                        (PagedKVCapacityError, ([20],)), (PagedKVPoolExhausted, ([0, 0, 16, 4],)),
                        (ValueError, (torch.ones(1, dtype=torch.int64, device="cuda"),)),
                        (ValueError, ([1.5],)), (ValueError, ([2], [0.5])), (ValueError, ([1 << 40 | 1, 1.0],))):
        with pytest.raises(error):
            pool.map_slots(*args)
    with pytest.raises(ValueError):
        map_slots_layers([pool, pool], [1])
    with pytest.raises(ValueError):
        map_slots_layers([pool, pool_of("cpu")], [1])
    assert all(torch.equal(a, b) for a, b in zip(before[0], pool.tensors[2:]))
    assert (pool.lens == before[1]).all() and pool.free_count == before[2]
    for lengths in ((0, 0), np.zeros(2, dtype=np.int32), torch.zeros(2, dtype=torch.int64), [False, np.int64(0)]):
        assert pool.map_slots(lengths).offsets.tolist() == [0, 0, 0]
    assert pool.map_slots([]).slots.numel() == 0 and pool.map_slots([0, 0]).offsets.tolist() == [0, 0, 0]


def test_a_pool_that_runs_out_on_the_device_is_flagged(hip):
    """What a graph's replays can meet: the host has checked nothing for them."""
    pool = pool_of("cuda", num_pages=3)
    pool.free_count = 100  # a host count that does not hold
    got = pool.map_slots([9, 8])
    assert got.slots.tolist() == list(range(9)) + [-1] * 8
    assert pool.errors() == 1 and pool.ctrl[0].item() == 0
    assert (pool.block_table[1, :2] == -1).all()
    k = torch.ones((17, 2, 8), dtype=torch.bfloat16, device="cuda")
    pool.write_slots(got.slots, k, k)  # the tokens without a page are passed over
    assert (pool.key_pages.flatten(0, 1)[:9] == 1).all() and (pool.key_pages.flatten(0, 1)[9:] == 0).all()


@pytest.mark.parametrize("dtype,heads,dim", [(torch.bfloat16, 8, 128), (torch.float32, 5, 64), (torch.float16, 1, 256),
                                             (torch.bfloat16, 3, 20), (torch.float64, 2, 3), (torch.uint8, 3, 5),
                                             (torch.float16, 1, 1)])
@pytest.mark.parametrize("layout", ["packed", "nodes", "heads"])
def test_write_slots(hip, dtype, heads, dim, layout):
    """Every width of vector, packed tokens, [batch, heads, nodes, dim] states and strided heads, with and
    without an index; what no slot names stays."""
    pool = pool_of("cuda", 4, 8, 16, heads, dim, dtype)
    g = torch.Generator().manual_seed(dim)
    k, v = (torch.randint(0, 100, (3 * 21, heads, dim), generator=g).to(dtype).cuda() for _ in range(2))
    if layout == "nodes":  # contiguous [batch, heads, nodes, dim]: the flattened view is a copy unless heads is 1
        k, v = (t.reshape(3, 21, heads, dim).transpose(1, 2).contiguous().transpose(1, 2).flatten(0, 1) for t in (k, v))
    if layout == "heads":
        k, v = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (k, v))
    slots = torch.randperm(pool.num_pages * 16, generator=g)[:40]
    slots[[3, 17]] = -1
    index = torch.randint(0, 63, (40,), generator=g)
    want = [torch.zeros_like(pool.key_pages).flatten(0, 1) for _ in range(2)]
    for x, t in zip(want, (k, v)):
        x[slots[slots >= 0].cuda()] = t[index[slots >= 0].cuda()]
    pool.write_slots(slots.cuda(), k, v, index.cuda())
    assert torch.equal(pool.key_pages.flatten(0, 1), want[0]) and torch.equal(pool.value_pages.flatten(0, 1), want[1])
    for x, t in zip(want, (k, v)):
        x[slots[slots >= 0].cuda()] = t[:40][(slots >= 0).cuda()]
    pool.write_slots(slots.cuda()[None, :].expand(2, 40)[1], k, v)
    assert torch.equal(pool.key_pages.flatten(0, 1), want[0]) and torch.equal(pool.value_pages.flatten(0, 1), want[1])
    assert pool.errors() == 0


def test_write_slots_passes_over_what_names_nothing(hip):
    pool = pool_of("cuda")
    k = torch.arange(5, device="cuda", dtype=torch.bfloat16)[:, None, None].expand(5, 2, 8)  # stride 0: copied
    slots = torch.tensor([3, -1, 9, 10**12, 0, pool.num_pages * 4], device="cuda")
    pool.write_slots(slots, k, k, torch.tensor([4, 0, 5, 1, 2, 2], device="cuda"))
    flat = pool.key_pages.flatten(0, 1)[:, 0, 0]
    assert flat[3] == 4 and flat[0] == 2 and int((flat != 0).sum()) == 2 and pool.errors() == 4
    pool.write_slots(slots[:0], k, k)
    for args in ((slots, k[:, :1], k[:, :1]), (slots, k.float(), k.float()), (slots.int(), k, k), (slots, k, k),
                 (slots.cpu(), k, k, slots), (slots, k, k, slots[:4])):
        with pytest.raises(ValueError):
            pool.write_slots(*args)


def test_slots_and_offsets_past_32_bits(hip):
    """A pool of more than 2^31 slots and more than 2^32 bytes: the last page's slots are stored and read."""
    pages, page = 80, 1 << 25
    pool = PagePool(max_batch=2, max_blocks=60, page_size=page, kv_heads=1, head_dim=2, dtype=torch.uint8, device="cuda",
                    num_pages=pages, page_order=torch.arange(pages - 1, -1, -1))
    got = pool.map_slots([3, 2])
    assert got.slots.tolist() == [(pages - 1) * page + i for i in range(3)] + [(pages - 2) * page + i for i in range(2)]
    k = torch.arange(10, dtype=torch.uint8, device="cuda").reshape(5, 1, 2)
    pool.write_slots(got.slots, k, k + 100)
    assert torch.equal(pool.key_pages[pages - 1, :3], k[:3]) and torch.equal(pool.value_pages[pages - 2, :2], k[3:] + 100)


def test_mapped_and_written_rows_equal_appends(hip):
    a, b = (pool_of("cuda", 6, 20, 16, 8, 128) for _ in range(2))
    g = torch.Generator(device="cuda").manual_seed(0)
    for rows, lengths in (([5, 0, 3], [100, 37, 1]), ([3, 0, 2], [4, 0, 200])):
        k, v = (torch.randn((sum(lengths), 8, 128), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
        a.write_slots(a.map_slots(lengths, rows).slots, k, v)
        at = 0
        for r, n in zip(rows, lengths):
            b.append_rows([r], *(t[at:at + n].transpose(0, 1)[None] for t in (k, v)))
            at += n
    for x, y in zip(a.gather(6), b.gather(6)):
        assert torch.equal(x, y)
    for x, y in zip(a.tensors[2:6], b.tensors[2:6]):
        assert torch.equal(x, y)


def test_another_stream_and_captured_replays(hip):
    """A captured map takes the lengths of its recording and the rows' state of each replay; a captured store
    reads its buffers anew."""
    pool = pool_of("cuda", 3, 40, 4)
    k, v = (torch.zeros((5, 2, 8), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool.map_slots([1, 2, 3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pool.map_slots([3, 0, 2], [2, 0, 1])
        pool.write_slots(got.slots, k, v)
    for replay in range(4):
        k.fill_(replay + 1)
        v.fill_(-replay - 1)
        graph.replay()
        torch.cuda.synchronize()
        assert pool.seq_lens.tolist() == [1, 2 + 2 * (replay + 1), 3 + 3 * (replay + 1)]
        assert got.positions.tolist() == [3 + 3 * replay + i for i in range(3)] + [2 + 2 * replay + i for i in range(2)]
        pool.lens[:] = pool.seq_lens.cpu().numpy()
        pool.hw[:] = pool.lens
        pool.free_count = int(pool.ctrl[0])
        ko, vo = pool.gather(3)
        assert (ko[2, :, -3:] == replay + 1).all() and (vo[1, :, 2 + 2 * replay:4 + 2 * replay] == -replay - 1).all()
        assert (ko[2, :, 3:6] == 1).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        more = pool.map_slots([2])
        pool.write_slots(more.slots, k[:2], v[:2])
    side.synchronize()
    assert more.positions.tolist() == [1, 2] and pool.errors() == 0


@pytest.mark.parametrize("kw", [{}, {"kv_quant": "fp8_e4m3", "residual_window": 64}])
def test_speculative_steps(hip, kw):
    """Prompts by slot map, trees attended, accepted paths stored, in every layer of a cache."""
    cache = make_cache("cuda", **kw)
    check_run(cache, *run_steps(cache, 2, "cuda"))
    assert all(l.pool.errors() == 0 for l in cache.layers)


def test_speculative_steps_after_a_beam_selection(hip):
    """Rows that share full pages, after a selection and a crop: stores go to pages of the row's own."""
    pool = pool_of("cuda", 3, 12, 4, 2, 64)
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda n: (torch.randn((n, 2, 64), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))  # noqa: E731
    k, v = new(11)
    pool.write_slots(pool.map_slots([11]).slots, k, v)
    pool.select_rows([0, 0, 0])
    pool.crop(3, 9)
    k2, v2 = new(9)
    pool.write_slots(pool.map_slots([2, 3, 4]).slots, k2, v2)
    ko, vo = pool.gather(3)
    for b, (lo, n) in enumerate([(0, 2), (2, 3), (5, 4)]):
        assert torch.equal(ko[b, :, :9 + n].transpose(0, 1), torch.cat([k[:9], k2[lo:lo + n]]))
        assert torch.equal(vo[b, :, :9 + n].transpose(0, 1), torch.cat([v[:9], v2[lo:lo + n]]))
    assert pool.errors() == 0


def test_quantised_pool_maps_and_quantises(hip):
    gpu, host = (pool_of(d, 2, 12, 16, 2, 64, torch.bfloat16, QuantPagePool, window=32, chunk=64) for d in ("cuda", "cpu"))
    for step, lengths in enumerate([[40, 10], [30, 0], [20, 60], [1, 1]]):
        g = torch.Generator().manual_seed(step)
        k, v = (torch.randn((sum(lengths), 2, 64), generator=g).to(torch.bfloat16) for _ in range(2))
        for pool in (gpu, host):
            pool.write_slots(pool.map_slots(lengths).slots, k.to(pool.device), v.to(pool.device))
        assert (gpu.cold_blocks == host.cold_blocks).all() and gpu.cold_free == host.cold_free
        for x, y in zip(gpu.gather(2), host.gather(2)):
            assert torch.equal(x.cpu(), y)
    assert (gpu.cold_blocks == [3, 2]).all() and gpu.errors() == 0
