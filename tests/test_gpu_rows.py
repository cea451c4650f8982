"""Pages copied and token rows moved together, in the caches of several layers, byte for byte."""

import random

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from turboquant_vllm.kernels import ops as _ops

    return _ops


def random_caches(layers, blocks, bs, width, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (blocks, bs, width), dtype=torch.uint8, generator=g) for _ in range(layers)]


# heads, head_dim, bytes of a row: padded, 16-byte pieces; odd heads (8-byte pieces); rows without padding; 4-byte pieces
ROWS = [(8, 128, 2048), (1, 128, 256), (2, 64, 144), (5, 96, 520), (1, 128, 140), (4, 256, 1056), (128, 256, 33792)]


# ---- pages ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("h,d,width", ROWS)
@pytest.mark.parametrize("pairs,layers,bs", [(1, 1, 16), (7, 3, 16), (40, 2, 1), (12, 33, 24)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_copy(ops, h, d, width, pairs, layers, bs, dtype):
    if width > 30000 and layers > 3:
        layers = 3
    caches = random_caches(layers, 2 * pairs + 3, bs, width)
    order = list(range(2 * pairs + 3))
    random.Random(pairs).shuffle(order)
    src, dst = order[:pairs], order[pairs : 2 * pairs]
    src[-1] = src[0]  # a source of two
    got = [c.cuda() for c in caches]
    ops.tq4_copy_blocks(got, torch.tensor(list(zip(src, dst)), dtype=dtype).cuda(), h, d)
    data = h * (d + 8)
    for c, x in zip(caches, got):
        c[dst, :, :data] = c[src, :, :data]
        assert torch.equal(x.cpu(), c)
    assert ops.read_and_clear_errors(got[0].device) == 0


@pytest.mark.parametrize("many", [False, True])
def test_copies_that_clash_are_decided_by_the_list(ops, many):
    """The same rule for lists that every block scans and for those with a map of the pages."""
    from turboquant_vllm import _native as nv

    caches = random_caches(2, 4000, 16, 144)
    filler = [(2000 + 2 * i, 2001 + 2 * i) for i in range(900 if many else 5)] * (2 if many else 1)  # (listed twice: harmless)

    def run(pairs, flag, result):
        got = [c.cuda() for c in caches]
        ops.tq4_copy_blocks(got, torch.tensor(pairs + filler).cuda(), 2, 64)
        assert ops.read_and_clear_errors(got[0].device) == flag
        for c, x in zip(caches, got):
            want = c.clone()
            for s, t in filler + result:
                want[t, :, :144] = c[s, :, :144]
            assert torch.equal(x.cpu(), want)

    run([(1, 2), (3, 2), (4, 5)], nv.DEV_PAGE_CONFLICT, [(1, 2), (4, 5)])     # one destination twice: the first
    run([(1, 2), (1, 2), (4, 5)], 0, [(1, 2), (4, 5)])                        # the same pair twice
    run([(1, 2), (2, 3), (4, 5)], nv.DEV_PAGE_CONFLICT, [(1, 2), (4, 5)])     # a source that is written
    run([(2, 3), (1, 2)], nv.DEV_PAGE_CONFLICT, [(1, 2)])
    run([(1, 2), (2, 1)], nv.DEV_PAGE_CONFLICT, [])                           # a swap: neither
    run([(6, 6), (6, 7)], 0, [(6, 7)])                                        # onto itself: nothing
    run([(1, 4000), (-1, 2), (1, -5), (4, 5)], nv.DEV_BAD_BLOCK, [(4, 5)])    # pages that are not there
    run([(1, 1 << 40), (4, 5)], nv.DEV_BAD_BLOCK, [(4, 5)])


def test_copy_of_many_pages_and_of_more_layers_than_a_launch_takes(ops):
    caches = torch.randint(0, 256, (130, 40, 4, 144), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    got = caches.cuda()
    ops.tq4_copy_blocks(list(got), torch.tensor([(0, 39), (5, 6)]).cuda(), 2, 64)
    caches[:, [39, 6]] = caches[:, [0, 5]]
    assert torch.equal(got.cpu(), caches)
    big = torch.randint(0, 256, (6000, 16, 144), dtype=torch.uint8, generator=torch.Generator().manual_seed(2))
    pairs = torch.randperm(6000, generator=torch.Generator().manual_seed(3)).view(-1, 2)
    got = big.cuda()
    ops.tq4_copy_blocks(got, pairs.cuda(), 2, 64)
    big[pairs[:, 1]] = big[pairs[:, 0]]
    assert torch.equal(got.cpu(), big)
    assert ops.read_and_clear_errors(got.device) == 0


def test_strided_caches(ops):
    """The caches of all layers interleaved in one buffer (layers inside blocks)."""
    full = torch.randint(0, 256, (20, 3, 16, 272), dtype=torch.uint8, generator=torch.Generator().manual_seed(1))
    got = full.cuda()
    ops.tq4_copy_blocks([got[:, i] for i in range(3)], torch.tensor([(0, 19), (5, 6)]).cuda(), 2, 128)
    full[[19, 6]] = full[[0, 5]]
    assert torch.equal(got.cpu(), full)


# ---- rows ----------------------------------------------------------------------------------------
def compact_reference(cache, table, bs, starts, keep, lens, data):
    flat = cache.flatten(0, 1)
    before = flat.clone()
    for i, n in enumerate(lens):
        for j in range(n):
            a, b = starts[i] + keep[i][j], starts[i] + j
            s = int(table[i, a // bs]) * bs + a % bs
            t = int(table[i, b // bs]) * bs + b % bs
            flat[t, :data] = before[s, :data]
    return cache


def compact_case(held, of, kept, bs, width, layers, seed, extra=1):
    """Sequences of held + of tokens in shuffled pages, of which sorted random `kept` stay."""
    rng = random.Random(seed)
    need = [-(-(a + b) // bs) for a, b in zip(held, of)]
    order = list(range(sum(need) + extra))
    rng.shuffle(order)
    table = torch.full((len(held), max(need) + 1), 1 << 20, dtype=torch.int32)
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[sum(need[:i]) : sum(need[:i]) + n], dtype=torch.int32)
    keep = [sorted(rng.sample(range(b), n)) for b, n in zip(of, kept)]
    return random_caches(layers, sum(need) + extra, bs, width, seed), table, keep


def run_compact(ops, caches, table, starts, keep, width, h, d, lens=None):
    places = torch.full((len(keep), max(1, width)), -7, dtype=torch.int32)
    for i, k in enumerate(keep):
        places[i, : len(k)] = torch.tensor(k, dtype=torch.int32)
    got = [c.cuda() for c in caches]
    out = torch.empty(len(keep), dtype=torch.int32, device="cuda")
    lens = [len(k) for k in keep] if lens is None else lens
    ops.tq4_compact_rows(got, table.cuda(), torch.tensor(starts, dtype=torch.int32).cuda(), places.cuda(),
                         torch.tensor(lens, dtype=torch.int32).cuda(), h, d, seq_lens_out=out)
    assert out.tolist() == [a + b for a, b in zip(starts, lens)]
    return [x.cpu() for x in got]


@pytest.mark.parametrize("h,d,width", ROWS)
@pytest.mark.parametrize("held,of,kept,bs,layers", [
    ([100, 7, 0], [16, 16, 16], [3, 0, 16], 16, 5),
    ([33], [64], [40], 16, 2),                      # a batch and a half of rows
    ([0, 15, 1], [1, 1, 60], [1, 0, 60], 24, 3),
    ([5, 0], [500, 300], [250, 299], 16, 2),        # long lists
    ([0, 3, 9], [900, 70, 66], [1, 65, 66], 32, 3),
])
def test_compact(ops, h, d, width, held, of, kept, bs, layers):
    if width > 30000:
        layers = 1
    caches, table, keep = compact_case(held, of, kept, bs, width, layers, seed=len(held) + width)
    got = run_compact(ops, caches, table, held, keep, max(kept), h, d)
    for c, x in zip(caches, got):
        assert torch.equal(x, compact_reference(c, table, bs, held, keep, kept, h * (d + 8)))
    assert ops.read_and_clear_errors(torch.device("cuda")) == 0


@pytest.mark.parametrize("pattern", ["last", "first", "every other", "shift by one", "all", "two halves"])
@pytest.mark.parametrize("n", [64, 65, 1000, 5000])
def test_orders_in_which_rows_overwrite_one_another(ops, pattern, n):
    of = 2 * n + 1
    keep = {"last": list(range(of - n, of)), "first": list(range(n)), "every other": list(range(0, 2 * n, 2)),
            "shift by one": list(range(1, n + 1)), "all": list(range(n)), "two halves": list(range(n // 2)) + list(range(of - n + n // 2, of))}[pattern]
    caches, table, _ = compact_case([3], [of], [1], 16, 272, 2, seed=n)
    for _ in range(3):
        got = run_compact(ops, caches, table, [3], [keep], n, 2, 128)
        for c, x in zip(caches, got):
            assert torch.equal(x, compact_reference(c.clone(), table, 16, [3], [keep], [n], 272))
    assert ops.read_and_clear_errors(torch.device("cuda")) == 0


@pytest.mark.parametrize("n", [6, 300])
def test_bad_lists_and_pages(ops, n):
    """A list out of order leaves its sequence as it is, a bad page its rows; the others are moved."""
    from turboquant_vllm import _native as nv

    caches, table, keep = compact_case([2, 2], [n + 20, n + 20], [n, n], 16, 272, 2, seed=n)
    bad_lists = [keep[0][:3] + [keep[0][2]] + keep[0][4:], keep[0][:-2] + keep[0][:-3:-1], [-1] + keep[0][1:]]
    for bad in bad_lists:
        got = run_compact(ops, caches, table, [2, 2], [bad, keep[1]], n, 2, 128)
        assert ops.read_and_clear_errors(torch.device("cuda")) == nv.DEV_KEEP_ORDER
        for c, x in zip(caches, got):
            assert torch.equal(x, compact_reference(c.clone(), table, 16, [2, 2], [[], keep[1]], [0, n], 272))
    for lens in ([n + 1, n], [-1, n]):
        got = run_compact(ops, caches, table, [2, 2], keep, n, 2, 128, lens=lens)
        assert ops.read_and_clear_errors(torch.device("cuda")) == nv.DEV_KEEP_ORDER
        for c, x in zip(caches, got):
            assert torch.equal(x, compact_reference(c.clone(), table, 16, [2, 2], [[], keep[1]], [0, n], 272))
    # positions past the table, before it, and pages that are not there
    far = [k + (1 << 29 if j == n - 1 else 0) for j, k in enumerate(keep[0])]
    got = run_compact(ops, caches, table, [2, 2], [far, keep[1]], n, 2, 128)
    assert ops.read_and_clear_errors(torch.device("cuda")) == nv.DEV_BAD_BLOCK
    for c, x in zip(caches, got):
        assert torch.equal(x, compact_reference(c.clone(), table, 16, [2, 2], [far[:-1], keep[1]], [n - 1, n], 272))
    got = run_compact(ops, caches, table, [-(1 << 30), 2], keep, n, 2, 128)
    assert ops.read_and_clear_errors(torch.device("cuda")) == nv.DEV_BAD_BLOCK
    for c, x in zip(caches, got):
        assert torch.equal(x, compact_reference(c.clone(), table, 16, [2, 2], [[], keep[1]], [0, n], 272))
    broken = table.clone()
    broken[0] = -1
    got = run_compact(ops, caches, broken, [2, 2], keep, n, 2, 128)
    assert ops.read_and_clear_errors(torch.device("cuda")) == nv.DEV_BAD_BLOCK
    for c, x in zip(caches, got):
        assert torch.equal(x, compact_reference(c.clone(), table, 16, [2, 2], [[], keep[1]], [0, n], 272))


def test_refusals(ops):
    cache = torch.zeros(4, 16, 272, dtype=torch.uint8, device="cuda")
    pairs = torch.zeros(1, 2, dtype=torch.int64, device="cuda")
    table, ints = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    keep = torch.zeros(2, 3, dtype=torch.int32, device="cuda")

    def refused(error, match, f, *args, **kw):
        with pytest.raises(error, match=match):
            f(*args, **kw)

    copy, compact = ops.tq4_copy_blocks, ops.tq4_compact_rows
    refused(RuntimeError, "CUDA", copy, cache.cpu(), pairs, 2, 128)
    refused(AssertionError, "hold a cache", copy, [], pairs, 2, 128)
    refused(AssertionError, "uint8", copy, cache.float(), pairs, 2, 128)
    refused(AssertionError, "alike", copy, [cache, cache[:3]], pairs, 2, 128)
    refused(AssertionError, "once", copy, [cache, cache], pairs, 2, 128)
    refused(AssertionError, "block_mapping", copy, cache, pairs[0], 2, 128)
    refused(AssertionError, "block_mapping", copy, cache, pairs.float(), 2, 128)
    refused(RuntimeError, "invalid argument", copy, cache, pairs, 3, 128)  # more heads than a row has bytes for
    refused(NotImplementedError, "head_dim", copy, cache, pairs, 2, 80)
    refused(RuntimeError, "invalid argument", copy, cache, pairs, 0, 128)
    refused(AssertionError, "keep must", compact, cache, table, ints, keep.long(), ints, 2, 128)
    refused(AssertionError, "block_table", compact, cache, table[:1], ints, keep, ints, 2, 128)
    refused(AssertionError, "starts", compact, cache, table, ints[:1], keep, ints, 2, 128)
    refused(AssertionError, "keep_lens", compact, cache, table, ints, keep, ints.long(), 2, 128)
    refused(AssertionError, "overlap", compact, cache, table, ints, keep, ints, 2, 128, seq_lens_out=ints)
    refused(RuntimeError, "CUDA", compact, cache, table, ints.cpu(), keep, ints, 2, 128)
    copy(cache, pairs[:0], 2, 128)
    compact(cache, table[:0], ints[:0], keep[:0], ints[:0], 2, 128)
    compact(cache, table, ints, keep[:, :0], ints, 2, 128)
    assert ops.read_and_clear_errors(cache.device) == 0


@pytest.mark.parametrize("n", [5, 300])
def test_captured(ops, n):
    caches, table, keep = compact_case([2], [n + 20], [n], 16, 272, 3, seed=n)
    got = [c.cuda() for c in caches]
    args = (got, table.cuda(), torch.tensor([2], dtype=torch.int32).cuda(), torch.tensor([keep[0]], dtype=torch.int32).cuda(),
            torch.tensor([n], dtype=torch.int32).cuda(), 2, 128)
    many = torch.stack((torch.zeros(1100, dtype=torch.long), torch.full((1100,), 1)), dim=1).cuda()  # (one pair, many times)
    ops.tq4_compact_rows(*args)
    ops.tq4_copy_blocks(got, many, 2, 128)
    torch.cuda.synchronize()
    for x, c in zip(got, caches):
        x.copy_(c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tq4_compact_rows(*args)
        ops.tq4_copy_blocks(got, many, 2, 128)
    want = [c.clone() for c in caches]
    for _ in range(3):
        graph.replay()
        for c in want:
            compact_reference(c, table, 16, [2], keep, [n], 272)
            c[1] = c[0]
    for x, c in zip(got, want):
        assert torch.equal(x.cpu(), c)
