"""Steps of decoding with a tree of drafts, as a server makes them, against sequences that never drafted anything.

Rotary positions, cache write, mask, attention of the tree, compaction of the accepted branch, the next step on what it left, and
pages copied where a sequence is forked.  What is kept in the cache has to be, byte for byte, what a cache holds into which the same tokens
were written one after the other; attention over equal bytes is the same call.
"""

import math
import random

import pytest
import torch

from tests.helpers import Prims
from turboquant_vllm.rotary import rotary_inv_freq

pytestmark = pytest.mark.gpu

BS = 16


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from turboquant_vllm.kernels import ops as _ops

    return _ops


class Server:
    """Caches of a few layers, a block table of its own order, and projections that depend on the token alone."""

    def __init__(self, ops, pr, layers, seqs, hq, hkv, pages, seed):
        self.ops, self.hq, self.hkv, self.d, self.layers = ops, hq, hkv, pr.d, layers
        self.p = pr.cuda()
        self.data = hkv * (pr.d + 8)
        width = hkv * (1 << (pr.d + 7).bit_length())
        order = list(range(seqs * pages + 4))
        random.Random(seed).shuffle(order)
        self.table = torch.tensor(order[: seqs * pages], dtype=torch.int32).view(seqs, pages).cuda()
        self.spare = order[seqs * pages :]
        self.caches = [torch.zeros(len(order), BS, width, dtype=torch.uint8, device="cuda") for _ in range(layers)]
        self.freq = rotary_inv_freq(pr.d, 10000.0)[0].cuda()

    def qkv(self, tokens, layer):
        """Rows of a token: the same whenever and wherever it is run."""
        def rows(heads, what):
            return torch.stack([torch.randn(heads, self.d, generator=torch.Generator().manual_seed(1000 * t + 10 * layer + what))
                                for t in tokens]).bfloat16().cuda()
        return rows(self.hq, 0), rows(self.hkv, 1), rows(self.hkv, 2)

    def write(self, tokens, seqs, slots_at, positions, layer):
        """Rotates, writes at places `slots_at` of sequences `seqs`; returns the rotated queries."""
        q, k, v = self.qkv(tokens, layer)
        q, k = self.ops.tq4_rotary(q, k, positions, self.freq)
        pages = self.table[seqs.long(), (slots_at // BS).long()].long()
        self.ops.tq4_write_paged(k, v, self.caches[layer], pages * BS + slots_at % BS, self.p["even"], self.p["odd"], self.p["kb"], self.p["vb"])
        return q

    def causal(self, q, layer, lens, starts):
        return self.ops.paged_tq4_attention(q, self.caches[layer], self.table, lens, self.p["kc"], self.p["vc"], self.p["rot"], self.hkv, BS,
                                            query_start_loc=starts, out_dtype=torch.float32)

    def rows(self, layer, seq, n):
        at = torch.arange(n, device="cuda")
        return self.caches[layer][self.table[seq, at // BS].long(), at % BS][:, : self.data]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("d,hq,hkv", [(128, 32, 8), (64, 14, 2), (96, 4, 4), (256, 8, 4)])
@pytest.mark.parametrize("held", [[1, 15, 16, 130], [700]])
def test_accepted_branches_leave_the_cache_of_plain_decoding(ops, d, hq, hkv, held):
    pr, rng, steps = Prims(d), random.Random(d + len(held)), 3
    seqs, layers = len(held), 2
    drafting, plain = (Server(ops, pr, layers, seqs, hq, hkv, max(held) // BS + 10, seed) for seed in (1, 2))
    text = [[rng.randrange(100) for _ in range(n)] for n in held]  # tokens so far
    for s in (drafting, plain):
        for layer in range(layers):
            for i, t in enumerate(text):
                at = torch.arange(len(t), dtype=torch.int32, device="cuda")
                s.write(t, ints([i] * len(t)), at, at, layer)
    lens = ints(held)
    for step in range(steps):
        # a tree a sequence: parents come first, branches of random length
        nodes = [rng.choice((1, 9, 33)) for _ in range(seqs)]
        parents = [[rng.randint(max(-1, j - 4), j - 1) for j in range(n)] for n in nodes]
        tokens = [[rng.randrange(100) for _ in range(n)] for n in nodes]
        starts = ints([sum(nodes[:i]) for i in range(seqs + 1)])
        mask, depth = ops.tq4_tree_mask(ints(sum(parents, [])), starts, max(nodes))
        owner = ints(sum(([i] * n for i, n in enumerate(nodes)), []))
        place = torch.cat([torch.arange(n, dtype=torch.int32, device="cuda") for n in nodes])
        base = lens[owner.long()]
        # the accepted branch: a node and its ancestors
        keep = []
        for i, n in enumerate(nodes):
            path, j = [], rng.randrange(n)
            while j >= 0:
                path.append(j)
                j = parents[i][j]
            keep.append(path[::-1])
        first = [sum(nodes[:i]) for i in range(seqs)]
        accepted = [[tokens[i][j] for j in path] for i, path in enumerate(keep)]
        after = ints([len(t) + len(a) for t, a in zip(text, accepted)])
        a_starts = ints([sum(len(a) for a in accepted[:i]) for i in range(seqs + 1)])
        a_owner = ints(sum(([i] * len(a) for i, a in enumerate(accepted)), []))
        a_at = ints(sum((list(range(len(t), len(t) + len(a))) for t, a in zip(text, accepted)), []))
        for layer in range(layers):
            q = drafting.write(sum(tokens, []), owner, base + place, base + depth, layer)
            out = ops.paged_tq4_tree_attention(q, drafting.caches[layer], drafting.table, lens + ints(nodes), starts, mask, drafting.p["kc"],
                                               drafting.p["vc"], drafting.p["rot"], hkv, BS, out_dtype=torch.float32)
            want = plain.causal(plain.write(sum(accepted, []), a_owner, a_at, a_at, layer), layer, after, a_starts)
            got = out[torch.tensor([first[i] + j for i, path in enumerate(keep) for j in path], device="cuda")]
            # The same bytes through the same fp16 tables.  Queries and weights are two fp16 terms in every kernel, 22 bits: a score
            # of up to 16 moves by 2^-18, a weight with it, and both kernels have both.  Sums of 64 keys in tensor memory truncate
            # by at most 8 * 2^-23.
            assert (got - want).norm() <= (8 * (int(after.max()) / 64 + 1) * 2 ** -23 + 2 ** -16) * want.norm()
        places = torch.full((seqs, max(map(len, keep)) + 1), -1, dtype=torch.int32)
        for i, path in enumerate(keep):
            places[i, : len(path)] = torch.tensor(path, dtype=torch.int32)
        new_lens = torch.empty_like(lens)
        ops.tq4_compact_rows(drafting.caches, drafting.table, lens, places.cuda(), ints([len(path) for path in keep]), hkv, d,
                             seq_lens_out=new_lens)
        assert torch.equal(new_lens, after)
        lens = new_lens
        text = [t + a for t, a in zip(text, accepted)]
        for layer in range(layers):
            for i, t in enumerate(text):
                assert torch.equal(drafting.rows(layer, i, len(t)), plain.rows(layer, i, len(t)))
    # one more token by plain decoding: the same bytes, so the same numbers
    for layer in range(layers):
        at = ints([len(t) for t in text])
        outs = [s.ops.paged_tq4_attention(s.write([7] * seqs, ints(range(seqs)), at, at, layer), s.caches[layer], s.table, at + 1, s.p["kc"],
                                          s.p["vc"], s.p["rot"], hkv, BS, out_dtype=torch.float32) for s in (drafting, plain)]
        assert torch.equal(*outs)
    assert ops.read_and_clear_errors(lens.device) == 0


def test_a_fork_copies_its_last_page_and_goes_its_own_way(ops):
    """Two branches of one context: full pages are shared, the half full one is copied before either writes."""
    pr, layers, length = Prims(128), 3, 37
    server = Server(ops, pr, layers, 2, 8, 2, 4, 3)
    tokens, at = [t % 91 for t in range(length)], torch.arange(length, dtype=torch.int32, device="cuda")
    for layer in range(layers):
        server.write(tokens, ints([0] * length), at, at, layer)
    last, own = int(server.table[0, length // BS]), server.spare[0]
    server.table[1] = server.table[0]
    server.table[1, length // BS] = own
    ops.tq4_copy_blocks(server.caches, ints([[last, own]]), 2, 128)
    for layer in range(layers):
        q = server.write([5, 6], ints([0, 1]), ints([length, length]), ints([length, length]), layer)
        assert torch.equal(server.rows(layer, 0, length), server.rows(layer, 1, length))
        assert not torch.equal(server.rows(layer, 0, length + 1), server.rows(layer, 1, length + 1))
        both = server.ops.paged_tq4_attention(q, server.caches[layer], server.table, ints([length + 1] * 2), server.p["kc"], server.p["vc"],
                                              server.p["rot"], 2, BS, out_dtype=torch.float32)
        assert torch.isfinite(both).all() and not torch.equal(both[0], both[1])
    assert ops.read_and_clear_errors(server.table.device) == 0


def test_an_evicted_context_is_the_context_of_the_rows_that_stay(ops):
    """Rows chosen by a score stay, in their order, rotated as they were; attention over them is attention that sees nothing else."""
    pr, n, left = Prims(128), 300, 77
    server = Server(ops, pr, 1, 1, 8, 2, 20, 4)
    at = torch.arange(n, dtype=torch.int32, device="cuda")
    server.write([t % 91 for t in range(n)], ints([0] * n), at, at, 0)
    keep = sorted(random.Random(0).sample(range(n), left))
    before = server.rows(0, 0, n)[keep]
    q = torch.randn(1, 8, 128, generator=torch.Generator().manual_seed(0)).half().cuda()
    # a draft behind a context that it does not see but for the rows that stay: the mask's words cover the whole context
    words = [0] * (-(-n // 32))
    for k in keep:
        words[k // 32] |= 1 << k % 32
    # (n drafts, of which one asks: the others are hidden from the output)
    rows = torch.zeros(n, 8, 128, dtype=torch.float16, device="cuda")
    rows[-1] = q[0]
    mask = torch.zeros(n, len(words), dtype=torch.int64)
    mask[-1] = torch.tensor(words)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32).cuda()
    seen = ops.paged_tq4_tree_attention(rows, server.caches[0], server.table, ints([n]), ints([0, n]), mask, server.p["kc"], server.p["vc"],
                                        server.p["rot"], 2, BS, out_dtype=torch.float32)[-1:]
    lens = torch.empty(1, dtype=torch.int32, device="cuda")
    ops.tq4_compact_rows(server.caches[0], server.table, ints([0]), ints([keep]), ints([left]), 2, 128, seq_lens_out=lens)
    assert lens.tolist() == [left] and torch.equal(server.rows(0, 0, left), before)
    alone = ops.paged_tq4_attention(q, server.caches[0], server.table, lens, server.p["kc"], server.p["vc"], server.p["rot"], 2, BS,
                                    out_dtype=torch.float32)
    # (as above, over five tiles)
    assert (seen - alone).norm() <= (8 * (math.ceil(n / 64) + 1) * 2 ** -23 + 2 ** -16) * alone.norm()
    assert ops.read_and_clear_errors(lens.device) == 0
