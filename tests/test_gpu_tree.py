"""Attention of drafted trees over the page pool on the GPU, against float64."""

import math

import numpy as np
import pytest
import torch

from barqtrain_amd.paged import PagePool, QuantPagePool
from tree_ref import tree_bound, tree_reference

pytestmark = pytest.mark.gpu


def filled(lens, page=16, heads=2, dim=128, dtype=torch.bfloat16, seed=0, extra=1, quant=False, scale=1.0, **kw):
    """Rows of the given lengths on scattered pages; every slot not written holds NaN."""
    blocks = max(-(-max(lens) // page), 1) + extra
    g = torch.Generator().manual_seed(seed)
    geometry = dict(max_batch=len(lens), max_blocks=blocks, page_size=page, kv_heads=heads, head_dim=dim, dtype=dtype,
                    device="cuda", **kw)
    if quant:
        pool = QuantPagePool(**geometry)
    else:
        pool = PagePool(page_order=torch.randperm(len(lens) * (blocks + 1), generator=g), **geometry)
    pool.key_pages.fill_(math.nan)
    pool.value_pages.fill_(math.nan)
    for b, n in enumerate(lens):
        k, v = ((torch.randn((1, heads, n, dim), generator=g) * scale).to(dtype).cuda() for _ in range(2))
        pool.append_rows([b], k, v)
    return pool


def nodes_of(pool, batch, nodes, group, seed=0, layout="projection"):
    g = torch.Generator().manual_seed(seed + 100)
    H, D = pool.kv_heads, pool.head_dim
    q, k, v = (torch.randn((batch, nodes, n, D), generator=g).to(pool.dtype).cuda() for n in (H * group, H, H))
    if layout == "heads":
        q, k, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    return q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)


def mask_of(kind, batch, nodes, seed=0):
    g = torch.Generator().manual_seed(seed + 200)
    if kind == "chain":
        return None
    m = torch.rand((batch, nodes, nodes), generator=g) < 0.3
    m |= torch.eye(nodes, dtype=torch.bool)
    m[:, nodes // 2] = False  # a node that sees no node
    return m[0].cuda() if kind == "shared" else m.cuda()


def check(pool, q, k, v, mask, got, scale=None):
    batch = q.shape[0]
    longest = max(int(pool.lens[:batch].max()), 1)
    ko, vo = pool.gather(batch, longest)
    scale = pool.head_dim**-0.5 if scale is None else scale
    out, weight, score = tree_reference(q, ko, vo, pool.lens, k, v, mask, scale)
    bound = tree_bound(out, weight, score, got.dtype, longest + q.shape[2], pool.head_dim)
    off = (got.double().cpu() - out).abs()
    assert got.shape == q.shape and off.le(bound).all(), f"off by {(off / bound).max().item():.3g} bounds"
    assert pool.errors() == 0


# Calls of little work are cut by the host, the others on the device, by the length that the call may have:
# with a bound of `LONG` positions all are cut on the device (but where the page size or the tree does not allow it).
LONG = 9000


def listed_pool(listed, lens, page=16, **kw):
    return filled(lens, page=page, extra=-(-LONG // page) if listed else 1, **kw)


def attend(pool, listed, *args, **kw):
    return pool.attend_tree(*args, max_seq=LONG if listed else None, **kw)


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nodes,group", [(1, 1), (1, 4), (5, 7), (13, 4), (17, 8), (64, 2), (100, 3)])
@pytest.mark.parametrize("mask", ["chain", "shared", "rows"])
def test_shapes(hip, dim, nodes, group, mask, listed):
    """Every head size and count of query rows, empty rows among rows that end inside tiles and pages."""
    lens = [0, 1, 63, 64, 65, 300]
    pool = listed_pool(listed, lens, dim=dim, seed=nodes)
    q, k, v = nodes_of(pool, len(lens), nodes, group, nodes)
    m = mask_of(mask, len(lens), nodes, nodes)
    check(pool, q, k, v, m, attend(pool, listed, q, k, v, m))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 3, 4, 8, 16, 24, 64, 200])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pages_and_types(hip, page, dtype, dim, listed):
    lens = [199, 5, 128]
    pool = listed_pool(listed, lens, page=page, heads=3, dim=dim, dtype=dtype, seed=page)
    q, k, v = nodes_of(pool, 3, 9, 2, page)
    m = mask_of("rows", 3, 9)
    check(pool, q, k, v, m, attend(pool, listed, q, k, v, m))
    got = attend(pool, listed, q, k, v, m, 0.3, out_dtype=torch.float32)
    assert got.dtype == torch.float32
    check(pool, q, k, v, m, got, 0.3)


@pytest.mark.parametrize("dim,nodes,group", [(128, 3, 4), (128, 12, 4), (128, 30, 8), (64, 4, 7), (256, 16, 2), (256, 40, 4)])
@pytest.mark.parametrize("out", [None, torch.float32])
def test_long_rows_are_split_and_joined(hip, dim, nodes, group, out):
    lens = [4001, 130, 0]
    pool = filled(lens, heads=2, dim=dim, seed=dim + nodes)
    q, k, v = nodes_of(pool, 3, nodes, group, nodes)
    m = mask_of("rows", 3, nodes)
    check(pool, q, k, v, m, pool.attend_tree(q, k, v, m, out_dtype=out))
    check(pool, q, k, v, m, pool.attend_tree(q, k, v, m, max_seq=pool.capacity))
    one = pool.attend_tree(q[:1], k[:1], v[:1], m[:1])
    check(pool, q[:1], k[:1], v[:1], m[:1], one)


@pytest.mark.parametrize("dim,nodes,group", [(128, 5, 4), (64, 12, 8), (256, 3, 4)])
def test_many_rows_of_few_positions(hip, dim, nodes, group):
    """More rows than a wave has lanes, most of them short: ranges of many pairs, and pairs of many ranges."""
    lens = [(i * 37) % 90 for i in range(150)] + [2500]
    pool = filled(lens, heads=3, dim=dim, seed=2)
    q, k, v = nodes_of(pool, len(lens), nodes, group, 2)
    check(pool, q, k, v, None, pool.attend_tree(q, k, v))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dim,nodes", [(128, 128), (128, 256), (64, 256), (256, 128), (256, 129)])
def test_largest_trees(hip, dim, nodes, listed):
    pool = listed_pool(listed, [70, 0], heads=4, dim=dim)
    q, k, v = nodes_of(pool, 2, nodes, 1)
    m = mask_of("rows", 2, nodes)
    check(pool, q, k, v, m, attend(pool, listed, q, k, v, m))
    check(pool, q, k, v, None, attend(pool, listed, q, k, v))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dim,group", [(64, 1), (128, 4), (128, 8), (256, 4)])
def test_what_a_node_does_not_see_takes_no_part(hip, dim, group, listed):
    """Infinities and NaN in nodes that others do not see, keys and values; what sees them has them."""
    nodes = 40
    pool = listed_pool(listed, [150, 0], dim=dim, heads=4, seed=5)
    q, k, v = nodes_of(pool, 2, nodes, group, 5)
    k, v = k.clone(), v.clone()
    m = torch.eye(nodes, dtype=torch.bool).expand(2, nodes, nodes).clone()
    m[:, :, 7] = True
    wild = {3: math.nan, 20: math.inf, 33: -math.inf, 39: math.nan}
    for j, x in wild.items():
        k[:, :, j, ::3] = x
        v[:, :, j, 1::5] = x
    clean = [i for i in range(nodes) if i not in wild]
    got = attend(pool, listed, q, k, v, m.cuda())
    ko, vo = pool.gather(2, 150)
    out, weight, score = tree_reference(q, ko, vo, pool.lens, k, v, m, dim**-0.5)
    bound = tree_bound(out, weight, score, got.dtype, 200, dim)
    assert (got.double().cpu() - out).abs()[:, :, clean].le(bound[:, :, clean]).all()
    # finite keys, an infinite value that its node alone sees: infinite there, and nowhere else
    k2, v2 = nodes_of(pool, 2, nodes, group, 6)[1:]
    v2 = v2.clone()
    v2[:, :, 20, 1::5] = math.inf
    got = attend(pool, listed, q, k2, v2, m.cuda()).float().cpu()
    assert (got[:, :, 20, 1::5] == math.inf).all()
    got[:, :, 20, 1::5] = 0
    assert got.isfinite().all()
    out, weight, score = tree_reference(q, ko, vo, pool.lens, k2, v2, m, dim**-0.5)
    bound = tree_bound(out, weight, score, torch.bfloat16, 200, dim)
    rest = [i for i in range(nodes) if i != 20]
    assert (got.double() - out).abs()[:, :, rest].le(bound[:, :, rest]).all()


@pytest.mark.parametrize("listed", [False, True])
def test_large_scores(hip, listed):
    """Scores of some hundreds, rising along the row, so that the running maximum moves often; and all equal."""
    pool = listed_pool(listed, [700], heads=5, dim=128, scale=1.0, seed=3)
    q, k, v = nodes_of(pool, 1, 6, 4, 3)
    q = q * 16
    check(pool, q, k, v, None, attend(pool, listed, q, k, v))
    zero = torch.zeros_like(q)
    check(pool, zero, k, v, None, attend(pool, listed, zero, k, v))


@pytest.mark.parametrize("listed", [False, True])
def test_layouts_and_outputs(hip, listed):
    """Strided and misaligned inputs, an out of the caller's, masks of any strides, fewer rows than the pool."""
    lens = [90, 31, 200]
    pool = listed_pool(listed, lens, heads=2, dim=64)
    q, k, v = nodes_of(pool, 3, 10, 3, layout="heads")
    m = mask_of("rows", 3, 10)
    want = attend(pool, listed, q, k, v, m)
    check(pool, q, k, v, m, want)
    flat = torch.zeros((3 * 10 * 6 * 64 + 1,), dtype=q.dtype, device="cuda")
    odd = flat[1:].view(3, 6, 10, 64).copy_(q)
    wide = torch.zeros((3, 2, 10, 65), dtype=q.dtype, device="cuda")
    wide[..., :64] = k
    turned = v.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(attend(pool, listed, odd, wide[..., :64], turned, m.transpose(1, 2).contiguous().transpose(1, 2)), want)
    for dtype in (q.dtype, torch.float32):
        for shape, turn in (((3, 6, 10, 64), False), ((3, 10, 6, 64), True), ((3, 6, 10, 67), False)):
            buffer = torch.full(shape, 7.0, dtype=dtype, device="cuda")
            out = buffer.transpose(1, 2) if turn else buffer[..., :64]
            got = attend(pool, listed, q, k, v, m, out=out)
            assert got.data_ptr() == out.data_ptr() and torch.equal(got.to(q.dtype), want)
            assert (buffer[..., 64:] == 7).all()
    two = attend(pool, listed, q[:2], k[:2], v[:2], m[:2])
    check(pool, q[:2], k[:2], v[:2], m[:2], two)
    expanded = m[:1].expand(3, 10, 10)
    assert torch.equal(attend(pool, listed, q, k, v, expanded), attend(pool, listed, q, k, v, m[0]))
    assert torch.equal(attend(pool, listed, q, k, v, m[:1]), attend(pool, listed, q, k, v, m[0]))
    one = torch.zeros((1, 2, 1, 64), dtype=q.dtype, device="cuda")  # dimensions of one: their strides do not count
    check(pool, q[:1, :, :1], one, one, None, attend(pool, listed, q[:1, :, :1], one.as_strided((1, 2, 1, 64), (3, 64, 5, 1)), one))


def test_refusals(hip):
    pool = filled([20], dim=64)
    q, k, v = nodes_of(pool, 1, 3, 2)
    m = torch.ones((3, 3), dtype=torch.bool, device="cuda")
    big = nodes_of(pool, 1, 257, 1)
    for args in ((q[..., :32], k, v), (q[:, :3], k, v), (q, k[:, :1], v[:, :1]), (q, k, v[:, :, :2]), (q.float(), k, v),
                 (q, k, v, m.int()), (q, k, v, m[:2]), (q, k, v, m.cpu()), (q.cpu(), k, v), big):
        with pytest.raises(ValueError):
            pool.attend_tree(*args)
    with pytest.raises(ValueError):
        pool.attend_tree(q, k, v, out=torch.empty_like(q)[:, :1])
    with pytest.raises(ValueError):
        pool.attend_tree(q, k, v, max_seq=10**6)
    for dtype, dim in ((torch.float32, 64), (torch.bfloat16, 96)):
        other = PagePool(max_batch=1, max_blocks=2, page_size=16, kv_heads=2, head_dim=dim, dtype=dtype, device="cuda")
        x = torch.zeros((1, 2, 3, dim), dtype=dtype, device="cuda")
        with pytest.raises(ValueError):
            other.attend_tree(x, x, x)
    assert pool.attend_tree(q[:, :, :0], k[:, :, :0], v[:, :, :0]).shape == (1, 4, 0, 64)
    assert pool.attend_tree(q[:0], k[:0], v[:0]).shape == (0, 4, 3, 64)


@pytest.mark.parametrize("heads", [2, 130])
def test_rows_longer_than_max_seq_and_bad_pages_are_flagged(hip, heads):
    pool = filled([100, 40], dim=64, heads=heads)
    q, k, v = nodes_of(pool, 2, 4, 2)
    got = pool.attend_tree(q, k, v, max_seq=50)
    assert pool.errors() == 16  # BARQ_KV_ERRBIT_ATTN_SHORT
    ko, vo = pool.gather(2, 100)
    out, weight, score = tree_reference(q, ko, vo, [50, 40], k, v, None, 64**-0.5)
    assert (got.double().cpu() - out).abs().le(tree_bound(out, weight, score, got.dtype, 54, 64)).all()
    pool.ctrl[1] = 0
    pool.key_pages.nan_to_num_(0.0)
    pool.value_pages.nan_to_num_(0.0)
    pool.block_table[1, 0] = pool.num_pages
    pool.attend_tree(q, k, v)
    assert pool.errors() == 4  # BARQ_KV_ERRBIT_BAD_INDEX


@pytest.mark.parametrize("blocks", [8, 600])
def test_page_offsets_past_32_bits(hip, blocks):
    pages = 140000  # 4.6 GB of keys
    pool = PagePool(max_batch=1, max_blocks=blocks, page_size=16, kv_heads=8, head_dim=128, dtype=torch.bfloat16, device="cuda",
                    num_pages=pages, page_order=torch.arange(pages - 1, -1, -1))
    g = torch.Generator().manual_seed(0)
    pool.append(*(torch.randn((1, 8, 77, 128), generator=g).to(torch.bfloat16).cuda() for _ in range(2)))
    q, k, v = nodes_of(pool, 1, 4, 2)
    check(pool, q, k, v, None, pool.attend_tree(q, k, v, max_seq=pool.capacity))


@pytest.mark.parametrize("extra", [8, 600])
def test_streams_and_captured_replays(hip, extra):
    """Two captured graphs of one pool and eager calls between their replays; rows grow between replays."""
    pool = filled([300, 10], dim=128, heads=2, extra=extra)
    inputs = [nodes_of(pool, 2, n, 4, n) for n in (5, 20)]
    masks = [mask_of("rows", 2, n, n) for n in (5, 20)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for (q, k, v), m in zip(inputs, masks):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pool.attend_tree(q, k, v, m))
        graphs.append(graph)
    side = torch.cuda.Stream()
    for replay in range(3):
        for i in (replay % 2, 1 - replay % 2):
            inputs[i][0].mul_(-1.01)
            graphs[i].replay()
            eager = pool.attend_tree(*inputs[1 - i], masks[1 - i])
            torch.cuda.synchronize()
            check(pool, *inputs[i], masks[i], outs[i])
            check(pool, *inputs[1 - i], masks[1 - i], eager)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = pool.attend_tree(*inputs[0], masks[0])
        side.synchronize()
        check(pool, *inputs[0], masks[0], got)
        g = torch.Generator().manual_seed(replay)
        pool.append(*(torch.randn((2, 2, 30, 128), generator=g).to(torch.bfloat16).cuda() for _ in range(2)))


def test_the_same_call_gives_the_same_bits(hip):
    pool = filled([2000, 100, 7000], dim=128, heads=4)
    q, k, v = nodes_of(pool, 3, 24, 4)
    m = mask_of("rows", 3, 24)
    first = pool.attend_tree(q, k, v, m)
    for _ in range(5):
        assert torch.equal(pool.attend_tree(q, k, v, m), first)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,page,nodes,group", [(128, 16, 6, 4), (64, 32, 20, 3), (128, 48, 70, 2), (64, 16, 1, 1),
                                                  (64, 16, 33, 4), (128, 32, 40, 4), (128, 16, 9, 4),
                                                  (64, 8, 5, 2), (256, 16, 5, 2)])
def test_fp8_pages(hip, dtype, dim, page, nodes, group):
    """Quantised blocks as the dequantising gather gives them; page sizes and heads the kernel does not decode too."""
    lens = [500, 129, 20, 0]
    pool = filled(lens, page=page, dim=dim, dtype=dtype, quant=True, window=64)
    assert pool.cold_blocks[0] > 0 and pool.cold_blocks[3] == 0
    q, k, v = nodes_of(pool, 4, nodes, group)
    m = mask_of("rows", 4, nodes)
    check(pool, q, k, v, m, pool.attend_tree(q, k, v, m))
    got = pool.attend_tree(q, k, v, m, out=torch.empty(q.shape, dtype=torch.float32, device="cuda"))
    check(pool, q, k, v, m, got)
    odd = torch.zeros((q.numel() + 1,), dtype=dtype, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(pool.attend_tree(odd, k, v, m, out_dtype=torch.float32), got)


def test_fp8_codes_of_every_kind(hip):
    """Zero, subnormal and saturating codes and far-apart scales: the element path of the decoder."""
    pool = QuantPagePool(max_batch=1, max_blocks=20, page_size=16, kv_heads=2, head_dim=128, dtype=torch.bfloat16,
                         device="cuda", window=16)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((1, 2, 300, 128), generator=g) * torch.exp(torch.randn((1, 2, 300, 128), generator=g) * 3) for _ in range(2))
    k[:, :, 5:9] = 0.0
    v[:, :, ::7] = 0.0
    pool.append((k * 0.05).to(torch.bfloat16).cuda(), v.to(torch.bfloat16).cuda())
    q, nk, nv = nodes_of(pool, 1, 4, 4)
    check(pool, q, nk, nv, None, pool.attend_tree(q, nk, nv))


@pytest.mark.parametrize("dtype,scales", [(torch.bfloat16, (12, 64, 127, 200, 238)), (torch.float16, (112, 119, 127, 133))])
@pytest.mark.parametrize("dim", [64, 128])
def test_fp8_every_code_at_far_scales(hip, dtype, scales, dim):
    """All codes but NaN's, of values at one scale a call and of keys at a scale a channel, as the gather gives them."""
    pool = QuantPagePool(max_batch=1, max_blocks=4, page_size=16, kv_heads=2, head_dim=dim, dtype=dtype, device="cuda", window=16)
    zeros = torch.zeros((1, 2, 48, dim), dtype=dtype, device="cuda")
    pool.append(zeros, zeros)
    assert pool.cold_blocks[0] == 2
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    codes[codes & 127 == 127] = 0
    q, k, v = nodes_of(pool, 1, 2, 3)
    for scale in scales:
        pool.value_scales.fill_(scale)
        for part in codes.view(-1, dim):
            pool.value_codes.copy_(part.expand_as(pool.value_codes))
            check(pool, q * 0, k * 0, v * 0, None, pool.attend_tree(q * 0, k * 0, v * 0))
    g = torch.Generator().manual_seed(dim)
    pool.value_scales.fill_(120)
    pool.key_codes.copy_(codes[torch.randint(0, 256, pool.key_codes.shape, generator=g).cuda()])
    pool.key_scales.copy_(torch.randint(116, 124, pool.key_scales.shape, generator=g).to(torch.uint8))
    check(pool, q, k, v, None, pool.attend_tree(q, k, v))


def test_single_tokens_agree_with_decode_attention(hip):
    """A chain of T nodes over the cache is decode attention of T tokens after their append."""
    pool = filled([257, 31], dim=128, heads=2, extra=2)
    q, k, v = nodes_of(pool, 2, 2, 4)
    tree = pool.attend_tree(q, k, v, out_dtype=torch.float32)
    pool.append(k, v)
    decode = pool.attend(q, out_dtype=torch.float32)
    ko, vo = pool.gather(2)
    out, weight, score = tree_reference(q, ko, vo, np.array(pool.lens) - 2, k, v, None, 128**-0.5)
    assert (tree.double().cpu() - out).abs().le(tree_bound(out, weight, score, torch.float32, 260, 128)).all()
    assert (tree - decode).abs().max() <= 2 * tree_bound(out, weight, score, torch.float32, 260, 128).max()
