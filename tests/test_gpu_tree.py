"""Masks of trees of drafted tokens, and attention with them over the packed cache, against 64-bit arithmetic from the definitions."""

import math
import random

import numpy as np
import pytest
import torch

from tests.helpers import Prims, build_paged_case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from turboquant_vllm.kernels import ops as _ops

    return _ops


def offsets(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32)


def random_parents(nodes, rng, reach=5):
    return [rng.randint(max(-1, j - reach), j - 1) for n in nodes for j in range(n)]


def ancestor_matrix(nodes, parents):
    """Per sequence the bool matrix [T, T]: row j sees itself and its ancestors."""
    out, first = [], 0
    for n in nodes:
        m = np.zeros((n, n), dtype=bool)
        for j in range(n):
            p = parents[first + j]
            if 0 <= p < j:
                m[j] = m[p]
            m[j, j] = True
        out.append(m)
        first += n
    return out


def pack(matrices, words):
    """Masks as words: [rows, words] int32 (bits past the last word are dropped)."""
    rows = []
    for m in matrices:
        bits = np.zeros((m.shape[0], 32 * words), dtype=np.uint64)
        keep = min(m.shape[1], 32 * words)
        bits[:, :keep] = m[:, :keep]
        word = (bits.reshape(m.shape[0], words, 32) << np.arange(32, dtype=np.uint64)).sum(axis=2)
        rows.append(word.astype(np.uint32).view(np.int32).reshape(m.shape[0], words))
    return torch.from_numpy(np.concatenate(rows)) if rows else torch.zeros(0, words, dtype=torch.int32)


def reference(q, case, nodes, matrices, pr, hkv, bs, scale, window=None):
    """float64: out [rows, Hq, D], lse [rows, Hq], and the rms of the visible scores."""
    rows, hq, d = q.shape
    group = hq // hkv
    out = torch.zeros(rows, hq, d, dtype=torch.float64)
    lse = torch.full((rows, hq), -math.inf, dtype=torch.float64)
    kc, vc, rot = pr.kc.double(), pr.vc.double(), pr.rot.double()
    squares = count = 0.0
    r0 = 0
    for i, (n, m) in enumerate(zip(nodes, matrices)):
        length = int(case["seq_lens"][i])
        base = length - n
        pos = torch.arange(length)
        held = case["cache"][case["block_table"][i, pos // bs].long(), pos % bs]
        vec, at = [], 0
        for cents in (kc, vc):
            idx = held[:, at : at + hkv * d // 2].reshape(length, hkv, d // 2).long()
            at += hkv * d // 2
            norm = held[:, at : at + 4 * hkv].contiguous().view(torch.float32).double()
            at += 4 * hkv
            vec.append((cents[torch.stack((idx >> 4, idx & 15), dim=-1).flatten(2)] @ rot) * norm[..., None])
        for j in range(n):
            sees = torch.zeros(length, dtype=torch.bool)
            low = max(0, base + int(m[j].sum()) - window) if window else 0
            sees[low : max(base, 0)] = True
            for k in np.nonzero(m[j])[0]:
                if 0 <= base + k < length:
                    sees[base + k] = True
            if not sees.any():
                continue
            for h in range(hq):
                s = vec[0][sees, h // group] @ q[r0 + j, h].double() * scale
                squares, count = squares + float(s.square().sum()), count + s.numel()
                lse[r0 + j, h] = torch.logsumexp(s, 0)
                out[r0 + j, h] = torch.softmax(s, 0) @ vec[1][sees, h // group]
        r0 += n
    return out, lse, math.sqrt(squares / max(count, 1))


# ---- masks -------------------------------------------------------------------------------------
@pytest.mark.parametrize("nodes,reach", [
    ([1], 1), ([0, 3, 0, 1], 3), ([31, 32, 33, 64, 65], 4), ([5, 24, 7, 200], 40), ([2500, 3], 2), ([700], 1),  # (a chain of 700)
])
def test_mask_is_the_ancestors(ops, nodes, reach):
    parents = random_parents(nodes, random.Random(sum(nodes)), reach)
    want = ancestor_matrix(nodes, parents)
    widest = max(nodes)
    mask, depth = ops.tq4_tree_mask(torch.tensor(parents, dtype=torch.int32).cuda(), offsets(nodes).cuda(), widest)
    assert mask.dtype == depth.dtype == torch.int32 and mask.shape == (sum(nodes), -(-widest // 32))
    assert torch.equal(mask.cpu(), pack(want, -(-widest // 32)))
    assert depth.tolist() == [int(r.sum()) - 1 for m in want for r in m]
    assert ops.read_and_clear_errors(mask.device) == 0


def test_mask_of_rows_behind_the_last_sequence_and_of_bad_parents(ops):
    from turboquant_vllm import _native as nv

    starts = torch.tensor([0, 3], dtype=torch.int32).cuda()
    mask, depth = ops.tq4_tree_mask(torch.tensor([-1, 0, 1, 0, -1], dtype=torch.int32).cuda(), starts, 40)
    assert mask.tolist() == [[1, 0], [3, 0], [7, 0], [0, 0], [0, 0]] and depth.tolist() == [0, 1, 2, -1, -1]
    assert ops.read_and_clear_errors(mask.device) == 0
    # a parent that is the row itself, a later one, or below -1: the row starts a branch, and it is reported
    for bad in (1, 2, -2, 1 << 30):
        mask, depth = ops.tq4_tree_mask(torch.tensor([-1, bad, 1], dtype=torch.int32).cuda(), starts, 3)
        assert mask.flatten().tolist() == [1, 2, 6] and depth.tolist() == [0, 0, 1]
        assert ops.read_and_clear_errors(mask.device) == nv.DEV_BAD_TREE
    # a draft without a bit of its own
    parents = torch.tensor([-1] + list(range(39)), dtype=torch.int32).cuda()
    mask, depth = ops.tq4_tree_mask(parents, torch.tensor([0, 40], dtype=torch.int32).cuda(), 32)
    assert mask.shape == (40, 1) and mask[39].item() == -1 and depth[39].item() == 39
    assert ops.read_and_clear_errors(mask.device) == nv.DEV_BAD_TREE


def test_mask_refusals(ops):
    starts, parents = torch.tensor([0, 2], dtype=torch.int32).cuda(), torch.tensor([-1, 0], dtype=torch.int32).cuda()
    with pytest.raises(AssertionError, match="parents"):
        ops.tq4_tree_mask(parents.long(), starts, 2)
    with pytest.raises(AssertionError, match="query_start_loc"):
        ops.tq4_tree_mask(parents, starts.long(), 2)
    with pytest.raises(AssertionError, match="max_nodes"):
        ops.tq4_tree_mask(parents, starts, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.tq4_tree_mask(parents.cpu(), starts, 2)
    mask, depth = ops.tq4_tree_mask(parents[:0], starts[:1], 7)
    assert mask.shape == (0, 1) and depth.shape == (0,)


# ---- attention ---------------------------------------------------------------------------------
CASES = [  # head_dim, q heads, KV heads, lengths, drafts, block size, window, row format, query type
    (128, 28, 4, [40], [8], 16, None, True, "bf16"),
    (128, 4, 4, [1], [1], 16, None, True, "fp16"),                       # nothing held, one draft
    (128, 8, 2, [7, 0, 300], [7, 0, 1], 16, None, True, "bf16"),         # drafts alone, an empty sequence, a single draft
    (128, 32, 8, [700, 130, 64, 65], [16, 9, 24, 1], 16, None, True, "fp16"),
    (128, 32, 8, [3000], [33], 16, None, True, "bf16"),                  # cut along the keys, two words
    (128, 8, 2, [600, 90], [200, 70], 16, None, True, "bf16"),           # several row blocks beside one stream of two
    (128, 28, 4, [500, 129], [37, 100], 32, None, False, "bf16"),        # groups of 7, rows without padding
    (128, 4, 1, [333], [40], 256, None, False, "bf16"),                  # 136-byte rows
    (64, 14, 2, [200, 1000], [30, 64], 16, None, True, "bf16"),
    (64, 64, 1, [150], [9], 24, None, True, "fp16"),                     # a group of 64: two rows a block; pages that end in tiles
    (96, 4, 4, [300, 41], [64, 9], 16, None, True, "bf16"),
    (96, 32, 32, [257], [100], 16, None, "dense", "bf16"),
    (256, 8, 4, [300, 90, 3], [12, 90, 3], 16, 64, True, "bf16"),
    (256, 2, 2, [900], [17], 16, None, True, "fp16"),
    (128, 8, 4, [500, 100, 20], [20, 33, 20], 16, 48, True, "bf16"),     # a window
    (128, 8, 4, [500, 100], [20, 70], 16, 3, True, "bf16"),              # ... shorter than the branches
    (128, 8, 8, [90], [40], 16, None, True, "fp32"),
    (128, 32, 8, [3000, 70], [30, 3], 16, None, True, "bf16"),           # few drafts, cut along the keys
    (128, 2, 2, [130], [40], 48, None, True, "bf16"),                    # rows whose values start on 8 bytes; pages of three boxes
    (64, 3, 3, [100, 257], [5, 40], 16, 100, False, "fp16"),             # ... rows of 216 bytes
    (96, 8, 1, [77], [16], 16, None, True, "bf16"),
]
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _call(ops, q, case, nodes, mask, p, hkv, bs, **kw):
    return ops.paged_tq4_tree_attention(
        q.cuda(), case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(), offsets(nodes).cuda(), mask.cuda(), p["kc"],
        p["vc"], p["rot"], hkv, bs, **kw)


def _check(got, lse, want, want_lse, spread, out_dtype=torch.float32):
    # Keys and values are centroids on the tensor cores' fp16 grid (half a step: 2^-11 of the value); an error of 2^-11 in a key moves
    # its score, and with it its weight, by 2^-11 of the score.  16-bit outputs add half a step of their own.
    # Calls with a bf16 output may round queries and weights to fp16 as well (2^-11 of the score, and of the weight, once more).
    tol = 2 ** -11 * (1 + spread) * (2 if out_dtype == torch.bfloat16 else 1)
    tol += 0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2
    assert torch.isfinite(got).all()
    assert (got.double() - want).norm() <= tol * want.norm() + 1e-30
    if lse is not None:
        seen = want_lse > -math.inf
        assert torch.equal(lse > -math.inf, seen)
        # (a score of `spread` moves by 2^-11 of it, at most some four times that for the largest; fp32 sums and log2 add 1e-5)
        assert (lse.double() - want_lse)[seen].abs().max() <= 2 ** -11 * 4 * (1 + spread) + 1e-5 if seen.any() else True


@pytest.mark.parametrize("d,hq,hkv,lens,nodes,bs,window,padded,dtype", CASES)
def test_tree_attention(ops, d, hq, hkv, lens, nodes, bs, window, padded, dtype):
    pr = Prims(d)
    case = build_paged_case(lens, hkv, d, bs, pr, seed=5, padded=padded)
    rng = random.Random(d + sum(lens))
    matrices = ancestor_matrix(nodes, random_parents(nodes, rng))
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype])
    lse = torch.full((sum(nodes), hq), math.nan, device="cuda")
    got = _call(ops, q, case, nodes, pack(matrices, -(-max(nodes) // 32)), pr.cuda(), hkv, bs, sliding_window=window,
                out_dtype=torch.float32, lse_out=lse)
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, hkv, bs, d ** -0.5, window)
    _check(got.cpu(), lse.cpu(), want, want_lse, spread)
    for out_dtype in (torch.bfloat16, torch.float16):
        got = _call(ops, q, case, nodes, pack(matrices, -(-max(nodes) // 32)), pr.cuda(), hkv, bs, sliding_window=window, out_dtype=out_dtype)
        _check(got.cpu(), None, want, None, spread, out_dtype)
    assert ops.read_and_clear_errors(got.device) == 0


@pytest.mark.parametrize("d,hq,hkv,lens,nodes", [(128, 8, 2, [40, 30, 12], [20, 30, 12]), (256, 8, 4, [70, 5], [40, 5]), (64, 4, 4, [33], [33])])
def test_any_mask_also_one_that_leaves_a_row_empty(ops, d, hq, hkv, lens, nodes):
    """Masks that no tree has: rows without any bit, without their own, with later drafts."""
    pr = Prims(d)
    case = build_paged_case(lens, hkv, d, 16, pr, seed=8, padded=True)
    rng = np.random.default_rng(d)
    matrices = [rng.random((n, n)) < 0.3 for n in nodes]
    for m in matrices:
        m[::5] = False
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(2)).bfloat16()
    lse = torch.empty(sum(nodes), hq, device="cuda")
    got = _call(ops, q, case, nodes, pack(matrices, 2), pr.cuda(), hkv, 16, out_dtype=torch.float32, lse_out=lse)
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, hkv, 16, d ** -0.5)
    _check(got.cpu(), lse.cpu(), want, want_lse, spread)
    empty = (want_lse == -math.inf).all(dim=1)
    assert empty.any() and (got.cpu()[empty] == 0).all()


def test_drafts_behind_the_masks_last_bit_are_hidden(ops):
    pr, nodes = Prims(128), [50]
    case = build_paged_case([90], 2, 128, 16, pr, seed=3, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3))
    q = torch.randn(50, 8, 128, generator=torch.Generator().manual_seed(3)).half()
    got = _call(ops, q, case, nodes, pack(matrices, 1), pr.cuda(), 2, 16, out_dtype=torch.float32)
    matrices[0][:, 32:] = False
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, 2, 16, 128 ** -0.5)
    _check(got.cpu(), None, want, want_lse, spread)
    got = _call(ops, q, case, nodes, torch.zeros(50, 0, dtype=torch.int32), pr.cuda(), 2, 16, out_dtype=torch.float32)  # no bits at all
    matrices[0][:] = False
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, 2, 16, 128 ** -0.5)
    _check(got.cpu(), None, want, want_lse, spread)


def test_more_drafts_than_tokens(ops):
    """A length below the number of drafts: the first drafts have no keys."""
    pr, nodes = Prims(128), [20]
    case = build_paged_case([12], 2, 128, 16, pr, seed=3, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3))
    q = torch.randn(20, 4, 128, generator=torch.Generator().manual_seed(3)).half()
    lse = torch.empty(20, 4, device="cuda")
    got = _call(ops, q, case, nodes, pack(matrices, 1), pr.cuda(), 2, 16, out_dtype=torch.float32, lse_out=lse)
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, 2, 16, 128 ** -0.5)
    _check(got.cpu(), lse.cpu(), want, want_lse, spread)


@pytest.mark.parametrize("d,hq,hkv,length,n", [(128, 32, 8, 900, 12), (256, 8, 4, 333, 20), (64, 14, 2, 2000, 40)])
def test_a_chain_is_causal_attention(ops, d, hq, hkv, length, n):
    """A tree that is one branch: the chunked prefill of the same rows."""
    pr = Prims(d)
    p = pr.cuda()
    case = build_paged_case([length], hkv, d, 16, pr, seed=9, padded=True)
    q = torch.randn(n, hq, d, generator=torch.Generator().manual_seed(4)).bfloat16()
    mask, _ = ops.tq4_tree_mask(torch.arange(-1, n - 1, dtype=torch.int32).cuda(), offsets([n]).cuda(), n)
    got = _call(ops, q, case, [n], mask, p, hkv, 16, out_dtype=torch.float32)
    want = ops.paged_tq4_attention(q.cuda(), case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(), p["kc"], p["vc"],
                                   p["rot"], hkv, 16, query_start_loc=offsets([n]).cuda(), out_dtype=torch.float32)
    # (the same tables and two-term products; sums in tensor memory truncate, at most 8 * 2^-23 a tile of 64 keys, as in the prefill kernel)
    assert (got - want).norm() <= (8 * (length / 64 + 1) * 2 ** -23 + 2 ** -18) * want.norm()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_16bit_output_strided_queries_and_rows_behind_the_last_sequence(ops, dtype):
    pr, nodes = Prims(128), [9, 5]
    p = pr.cuda()
    case = build_paged_case([200, 77], 2, 128, 16, pr, seed=3, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3))
    fused = torch.randn(17, 8 + 4, 128, generator=torch.Generator().manual_seed(3)).to(DTYPES[dtype])  # q | k | v of a projection
    mask = torch.cat((pack(matrices, 1), torch.full((3, 1), -1, dtype=torch.int32)))
    out = torch.full((17, 8, 160), 7.0, dtype=DTYPES[dtype], device="cuda")
    q = fused.cuda()[:, :8]
    got = ops.paged_tq4_tree_attention(q, case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(), offsets(nodes).cuda(),
                                       mask.cuda(), p["kc"], p["vc"], p["rot"], 2, 16, out=out[..., :128])
    assert got.data_ptr() == out.data_ptr() and (out[..., 128:] == 7).all()
    full = _call(ops, fused[:, :8].contiguous(), case, nodes, mask, p, 2, 16, out_dtype=torch.float32)
    if dtype == "fp16":  # (the rounded fp32 output; a bf16 output's queries and weights are rounded, too)
        assert torch.equal(out[..., :128], full.to(out.dtype))
    want, want_lse, spread = reference(fused[:14, :8], case, nodes, matrices, pr, 2, 16, 128 ** -0.5)
    _check(out[:14, :, :128].cpu(), None, want, want_lse, spread, DTYPES[dtype])
    assert (out[14:, :, :128] == 0).all()


def test_rotated_output_and_its_merge(ops):
    """Rotated partials with their lse, as the shards of a long context are merged."""
    pr, nodes = Prims(128), [12]
    p = pr.cuda()
    case = build_paged_case([700], 4, 128, 16, pr, seed=3, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3))
    q = torch.randn(12, 8, 128, generator=torch.Generator().manual_seed(3)).half()
    lse = torch.empty(12, 8, device="cuda")
    rotated = _call(ops, q, case, nodes, pack(matrices, 1), p, 4, 16, out_dtype=torch.float32, lse_out=lse, out_rotated=True)
    got = ops.combine_partials(rotated[None], lse[None], p["rot"])
    want, _, spread = reference(q, case, nodes, matrices, pr, 4, 16, 128 ** -0.5)
    _check(got.cpu(), None, want, None, spread)


def test_bad_pages_and_lengths_are_reported_and_hidden(ops):
    from turboquant_vllm import _native as nv

    pr, nodes = Prims(128), [6]
    p = pr.cuda()
    case = build_paged_case([100], 2, 128, 16, pr, seed=3, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3))
    q = torch.randn(6, 8, 128, generator=torch.Generator().manual_seed(3)).half()
    mask = pack(matrices, 1)
    good = _call(ops, q, case, nodes, mask, p, 2, 16, out_dtype=torch.float32)
    bad = dict(case, block_table=case["block_table"].clone())
    bad["block_table"][0, 2] = 1 << 30
    out = _call(ops, q, bad, nodes, mask, p, 2, 16, out_dtype=torch.float32)
    assert ops.read_and_clear_errors(out.device) == nv.DEV_BAD_BLOCK
    assert torch.isfinite(out).all() and not torch.equal(out, good)
    # a length past the table's row is cut there; the row stride may be wider than the row
    wide = torch.zeros(1, 64, dtype=torch.int32)
    wide[0, :7] = case["block_table"][0, :7]
    far = dict(case, seq_lens=torch.tensor([500], dtype=torch.int32))
    out = ops.paged_tq4_tree_attention(q.cuda(), case["cache"].cuda(), wide.cuda()[:, :7], far["seq_lens"].cuda(), offsets(nodes).cuda(),
                                       mask.cuda(), p["kc"], p["vc"], p["rot"], 2, 16, out_dtype=torch.float32)
    assert ops.read_and_clear_errors(out.device) == nv.DEV_BAD_BLOCK and torch.isfinite(out).all()


def test_refusals(ops):
    pr, nodes = Prims(128), [6]
    p = pr.cuda()
    case = build_paged_case([100], 2, 128, 16, pr, seed=3, padded=True)
    q, mask = torch.zeros(6, 8, 128, dtype=torch.float16), torch.zeros(6, 1, dtype=torch.int32)

    def call(error, match, q=q, case=case, mask=mask, hkv=2, bs=16, starts=offsets(nodes), **kw):
        with pytest.raises(error, match=match):
            ops.paged_tq4_tree_attention(q.cuda(), case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(),
                                         starts.cuda(), mask.cuda(), p["kc"], p["vc"], p["rot"], hkv, bs, **kw)

    call(AssertionError, "tree_mask", mask=mask[:5])
    call(AssertionError, "tree_mask", mask=mask.long())
    call(AssertionError, "multiple of the KV heads", hkv=3)
    call(AssertionError, "block_size", bs=32)
    call(AssertionError, "query_start_loc", starts=offsets([3, 3]))
    call(AssertionError, "seq_lens", case=dict(case, seq_lens=case["seq_lens"].long()))
    call(AssertionError, "out must", out=torch.empty(6, 8, 64, device="cuda"))
    call(ValueError, "workspace has", workspace=torch.empty(64, dtype=torch.uint8, device="cuda"))
    call(AssertionError, "rotation", q=torch.zeros(6, 8, 80, dtype=torch.float16))
    call(TypeError, "float32/float16/bfloat16", q=q.double())
    with pytest.raises(ValueError):
        ops.tree_attention_workspace_bytes(4, 129, 1, 128)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.paged_tq4_tree_attention(q, case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(), offsets(nodes).cuda(),
                                     mask.cuda(), p["kc"], p["vc"], p["rot"], 2, 16)


def test_captured_calls_on_two_streams_and_an_own_workspace(ops):
    """Two captured graphs, replayed on two streams at a time, give what eager calls give; so does a workspace of the caller's."""
    pr = Prims(128)
    p = pr.cuda()
    cases = []
    for seed, lens, nodes in ((1, [900, 40], [7, 20]), (2, [64, 2000], [64, 3])):
        case = build_paged_case(lens, 2, 128, 16, pr, seed=seed, padded=True)
        matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(seed), 3))
        q = torch.randn(sum(nodes), 8, 128, generator=torch.Generator().manual_seed(seed)).half().cuda()
        args = [q, case["cache"].cuda(), case["block_table"].cuda(), case["seq_lens"].cuda(), offsets(nodes).cuda(), pack(matrices, 2).cuda(),
                p["kc"], p["vc"], p["rot"], 2, 16]
        out = torch.empty(sum(nodes), 8, 128, device="cuda")
        eager = ops.paged_tq4_tree_attention(*args, out_dtype=torch.float32)
        ws = torch.empty(ops.tree_attention_workspace_bytes(sum(nodes), 8, 2, 128), dtype=torch.uint8, device="cuda")
        assert torch.equal(ops.paged_tq4_tree_attention(*args, out_dtype=torch.float32, workspace=ws), eager)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_tq4_tree_attention(*args, out=out)
        cases.append((graph, out, eager, torch.cuda.Stream(), args))  # (the graph reads its inputs where they are)
    for _ in range(3):
        for _, out, *_ in cases:
            out.fill_(math.nan)
        torch.cuda.synchronize()
        for graph, _, _, stream, _ in cases:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, eager, *_ in cases:
            assert torch.equal(out, eager)


@pytest.mark.parametrize("lens,nodes", [([100], [20]), ([3000, 70], [30, 3]), ([400], [200])])  # one part, parts of the keys, many drafts
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("where", ["key", "value"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_norm_that_is_not_finite_reaches_the_rows_that_see_it(ops, lens, nodes, dtype, where, bad):
    """In a draft, and in front of the window: rows that do not see the token are what they were, the others NaN."""
    d, hkv, bs, window = 128, 2, 16, 40
    pr = Prims(d)
    p = pr.cuda()
    case = build_paged_case(lens, hkv, d, bs, pr, seed=6, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(2), 3))
    mask = pack(matrices, -(-max(nodes) // 32))
    q = torch.randn(sum(nodes), 8, d, generator=torch.Generator().manual_seed(3)).to(DTYPES[dtype])
    for window_, token in ((None, lens[0] - nodes[0] + 4), (window, lens[0] - nodes[0] - window)):
        good = _call(ops, q, case, nodes, mask, p, hkv, bs, sliding_window=window_)
        assert torch.isfinite(good).all()
        hurt = dict(case, cache=case["cache"].clone())
        at = hkv * d // 2 if where == "key" else hkv * d + 4 * hkv
        row = hurt["cache"][case["block_table"][0, token // bs].long(), token % bs]
        row[at : at + 4] = torch.tensor([bad]).view(torch.uint8)  # (the first KV head's)
        got = _call(ops, q, hurt, nodes, mask, p, hkv, bs, sliding_window=window_)
        sees = torch.zeros(sum(nodes), dtype=torch.bool)
        if window_ is None:
            sees[: nodes[0]] = torch.from_numpy(matrices[0][:, 4])
        else:  # (the position of a row of depth n - 1 is that of the last token held plus n)
            sees[: nodes[0]] = torch.from_numpy(token >= lens[0] - nodes[0] + matrices[0].sum(axis=1) - window)
        hit = torch.zeros(sum(nodes), 8, dtype=torch.bool)
        hit[sees, :4] = True
        assert 0 < int(sees.sum()) < sum(nodes) or window_ is not None
        assert torch.isnan(got.cpu()[hit]).all()
        assert torch.equal(got.cpu()[~hit], good.cpu()[~hit])
    assert ops.read_and_clear_errors(q.cuda().device) == 0


def test_more_sequences_than_a_warp_has_lanes_cut_along_the_keys(ops):
    """Seventy sequences of very different lengths, some empty, on one KV head: the shares of the keys are found 32 sequences at a time."""
    rng = random.Random(7)
    d, hq, hkv, bs = 128, 4, 1, 16
    nodes = [rng.choice((0, 1, 5, 30)) for _ in range(70)]
    lens = [n + rng.choice((0, 3, 64, 500, 1500)) for n in nodes]
    pr = Prims(d)
    case = build_paged_case(lens, hkv, d, bs, pr, seed=5, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, rng))
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(1)).half()
    lse = torch.full((sum(nodes), hq), math.nan, device="cuda")
    got = _call(ops, q, case, nodes, pack(matrices, 1), pr.cuda(), hkv, bs, out_dtype=torch.float32, lse_out=lse)
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, hkv, bs, d ** -0.5)
    _check(got.cpu(), lse.cpu(), want, want_lse, spread)
    assert ops.read_and_clear_errors(got.device) == 0


@pytest.mark.parametrize("d,hq,hkv", [(128, 8, 2), (256, 8, 4)])
def test_a_replayed_graph_follows_lengths_offsets_and_masks(ops, d, hq, hkv):
    """The step that a server captures once: its inputs change in place, sequences come and go, the mask is part of a wider buffer."""
    pr = Prims(d)
    p = pr.cuda()
    cases = [([900, 40, 0], [7, 20, 0]), ([5, 0, 1700], [5, 0, 31]), ([64, 2000, 33], [1, 2, 3])]
    rows, words = 40, 2
    built = [build_paged_case(lens, hkv, d, 16, pr, seed=i, padded=True) for i, (lens, _) in enumerate(cases)]
    pages = max(b["cache"].shape[0] for b in built)
    width = max(b["block_table"].shape[1] for b in built) + 3
    cache = torch.zeros(pages, *built[0]["cache"].shape[1:], dtype=torch.uint8, device="cuda")
    table = torch.zeros(3, width, dtype=torch.int32, device="cuda")
    lens_, starts = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    mask = torch.full((rows, words + 3), -1, dtype=torch.int32, device="cuda")
    q = torch.zeros(rows, hq, d, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.zeros(rows, hq, d, device="cuda"), torch.zeros(rows, hq, device="cuda")

    def step():
        ops.paged_tq4_tree_attention(q, cache, table, lens_, starts, mask[:, 1 : 1 + words], p["kc"], p["vc"], p["rot"], hkv, 16, out=out, lse_out=lse)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (0, 1, 2, 0):
        (lens, nodes), case = cases[i], built[i]
        n = sum(nodes)
        matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(i)))
        cache[: case["cache"].shape[0]].copy_(case["cache"])
        table.zero_()
        table[:, : case["block_table"].shape[1]].copy_(case["block_table"])
        lens_.copy_(case["seq_lens"])
        starts.copy_(offsets(nodes))
        mask[:n, 1 : 1 + words].copy_(pack(matrices, words))
        new = torch.randn(rows, hq, d, generator=torch.Generator().manual_seed(i)).bfloat16()
        q.copy_(new)
        out.fill_(math.nan)
        lse.fill_(math.nan)
        graph.replay()
        want, want_lse, spread = reference(new[:n], case, nodes, matrices, pr, hkv, 16, d ** -0.5)
        _check(out[:n].cpu(), lse[:n].cpu(), want, want_lse, spread)
        assert (out[n:] == 0).all() and (lse[n:] == -math.inf).all()
    assert ops.read_and_clear_errors(out.device) == 0


@pytest.mark.parametrize("lens,nodes", [([100], [20]), ([3000, 70], [30, 3]), ([400], [200])])  # one part, parts of the keys, many drafts
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_query_that_is_not_finite_is_its_own_rows_alone(ops, lens, nodes, dtype, bad):
    pr = Prims(128)
    case = build_paged_case(lens, 2, 128, 16, pr, seed=6, padded=True)
    mask = pack(ancestor_matrix(nodes, random_parents(nodes, random.Random(2), 3)), -(-max(nodes) // 32))
    q = torch.randn(sum(nodes), 8, 128, generator=torch.Generator().manual_seed(3)).to(DTYPES[dtype])
    good = _call(ops, q, case, nodes, mask, pr.cuda(), 2, 16)
    hit = torch.zeros(sum(nodes), 8, dtype=torch.bool)
    hit[4, 5] = hit[17, 0] = True
    q[hit] = q[hit].clone().index_fill_(1, torch.tensor([9]), bad)
    got = _call(ops, q, case, nodes, mask, pr.cuda(), 2, 16)
    assert torch.isnan(got.cpu()[hit]).all()  # (an infinite coordinate makes scores of both signs, and the rotation of it NaN)
    assert torch.equal(got.cpu()[~hit], good.cpu()[~hit])
    assert ops.read_and_clear_errors(got.device) == 0


@pytest.mark.parametrize("d,hq,hkv,lens,nodes", [
    (128, 8, 2, [100], [20]), (128, 8, 2, [3000, 70], [30, 3]), (128, 8, 2, [400], [200]),  # one part, parts of the keys, many drafts
    (256, 8, 4, [100], [20]), (256, 8, 4, [3000], [12]), (96, 4, 4, [2000], [9])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("where", ["key", "value", "query"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_the_lse_of_a_row_that_is_not_finite_is_nan(ops, d, hq, hkv, lens, nodes, dtype, where, bad):
    """Whether or not the keys are cut; and a merge with another part of the context hands it on instead of leaving the row's keys out."""
    pr, bs = Prims(d), 16
    p = pr.cuda()
    case = build_paged_case(lens, hkv, d, bs, pr, seed=6, padded=True)
    other = build_paged_case([200, 50][: len(lens)], hkv, d, bs, pr, seed=7, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(2), 3))
    mask = pack(matrices, -(-max(nodes) // 32))
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(3)).to(DTYPES[dtype])

    def run(q, case):
        lse = torch.zeros(sum(nodes), hq, device="cuda")
        out = _call(ops, q, case, nodes, mask, p, hkv, bs, out_dtype=torch.float32, out_rotated=True, lse_out=lse)
        return out, lse

    good, good_lse = run(q, case)
    healthy, healthy_lse = run(q, other)
    assert torch.isfinite(good_lse).all() and torch.isfinite(healthy_lse).all()
    hit = torch.zeros(sum(nodes), hq, dtype=torch.bool)
    if where == "query":
        hit[4, hq - 1] = hit[8, 0] = True
        hurt_q, hurt = q.clone(), case
        hurt_q[hit] = q[hit].index_fill(1, torch.tensor([9]), bad)
    else:
        hurt_q, hurt = q, dict(case, cache=case["cache"].clone())
        token = lens[0] - nodes[0] + 4
        at = hkv * d // 2 if where == "key" else hkv * d + 4 * hkv
        row = hurt["cache"][case["block_table"][0, token // bs].long(), token % bs]
        row[at : at + 4] = torch.tensor([bad]).view(torch.uint8)  # (the first KV head's)
        hit[: nodes[0], : hq // hkv] = torch.from_numpy(matrices[0][:, 4])[:, None]
        assert hit.any() and not hit.all()
    hit = hit.cuda()
    got, lse = run(hurt_q, hurt)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], good[~hit])
    assert torch.isnan(lse[hit]).all() and torch.equal(lse[~hit], good_lse[~hit])
    merged = ops.combine_partials(torch.stack((got, healthy)), torch.stack((lse, healthy_lse)), p["rot"])
    want = ops.combine_partials(torch.stack((good, healthy)), torch.stack((good_lse, healthy_lse)), p["rot"])
    assert torch.isnan(merged[hit]).all() and torch.equal(merged[~hit], want[~hit])
    assert ops.read_and_clear_errors(got.device) == 0


FORMS = [  # head_dim, q heads, KV heads, lengths, drafts
    (128, 8, 2, [100, 70], [20, 3]), (128, 8, 2, [3000, 70], [30, 3]), (128, 8, 2, [400], [200]),  # one part, parts of the keys, many drafts
    (64, 14, 2, [200, 1000], [30, 17]), (96, 4, 4, [300, 41], [20, 9]), (256, 8, 4, [300, 90], [12, 40]), (256, 8, 4, [3000], [12])]


@pytest.mark.parametrize("d,hq,hkv,lens,nodes", FORMS)
@pytest.mark.parametrize("scale", [1.0, 32.0])
def test_a_bf16_output_is_the_rounded_fp32_one(ops, d, hq, hkv, lens, nodes, scale):
    """No caller's choice of output or lse changes how queries and weights enter the products, whatever the size of the scores."""
    pr = Prims(d)
    case = build_paged_case(lens, hkv, d, 16, pr, seed=5, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(4)))
    mask = pack(matrices, -(-max(nodes) // 32))
    q = (scale * torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(1))).bfloat16()
    full = _call(ops, q, case, nodes, mask, pr.cuda(), hkv, 16, out_dtype=torch.float32)
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, hkv, 16, d ** -0.5)
    _check(full.cpu(), None, want, None, spread)
    lse = torch.empty(sum(nodes), hq, device="cuda")
    for kw in ({}, {"lse_out": lse}, {"mode": 3}):
        assert torch.equal(_call(ops, q, case, nodes, mask, pr.cuda(), hkv, 16, **kw), full.bfloat16())


@pytest.mark.parametrize("d,hq,hkv,lens,nodes", FORMS)
def test_single_terms_where_the_caller_asks_for_them(ops, d, hq, hkv, lens, nodes):
    pr = Prims(d)
    p = pr.cuda()
    case = build_paged_case(lens, hkv, d, 16, pr, seed=5, padded=True)
    matrices = ancestor_matrix(nodes, random_parents(nodes, random.Random(4)))
    mask = pack(matrices, -(-max(nodes) // 32))
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    want, want_lse, spread = reference(q, case, nodes, matrices, pr, hkv, 16, d ** -0.5)
    lse = torch.empty(sum(nodes), hq, device="cuda")
    got = _call(ops, q, case, nodes, mask, p, hkv, 16, mode=4, lse_out=lse)
    _check(got.cpu(), lse.cpu(), want, want_lse, spread, torch.bfloat16)
    assert torch.equal(_call(ops, q, case, nodes, mask, p, hkv, 16, mode=4), got)
    full = _call(ops, q, case, nodes, mask, p, hkv, 16, mode=4, out_dtype=torch.float32)
    assert torch.equal(full.bfloat16(), got)
    # one row that sees a token without a finite norm, one query that is not finite: their rows alone
    hurt, hurt_q = dict(case, cache=case["cache"].clone()), q.clone()
    token = lens[0] - nodes[0] + 4
    hurt["cache"][case["block_table"][0, token // 16].long(), token % 16][hkv * d // 2 : hkv * d // 2 + 4] = torch.tensor([math.nan]).view(torch.uint8)
    hurt_q[9, hq - 1, 3] = math.inf
    hit = torch.zeros(sum(nodes), hq, dtype=torch.bool)
    hit[: nodes[0], : hq // hkv] = torch.from_numpy(matrices[0][:, 4])[:, None]
    hit[9, hq - 1] = True
    bad = _call(ops, hurt_q, hurt, nodes, mask, p, hkv, 16, mode=4)
    assert torch.isnan(bad.cpu()[hit]).all() and torch.equal(bad.cpu()[~hit], got.cpu()[~hit])
    assert ops.read_and_clear_errors(got.device) == 0


def test_modes_that_there_are_not(ops):
    pr, nodes = Prims(128), [6]
    case = build_paged_case([100], 2, 128, 16, pr, seed=3, padded=True)
    q, mask = torch.zeros(6, 8, 128, dtype=torch.float16), torch.zeros(6, 1, dtype=torch.int32)
    for mode in (1, 2, 5, -1, 1 << 32):
        with pytest.raises(AssertionError, match="mode"):
            _call(ops, q, case, nodes, mask, pr.cuda(), 2, 16, mode=mode)
    for dtype in (torch.float16, torch.float32):
        with pytest.raises(NotImplementedError):
            _call(ops, q.to(dtype), case, nodes, mask, pr.cuda(), 2, 16, mode=4)


@pytest.mark.parametrize("d,hq,hkv,lens,nodes", [
    (128, 4, 2, [12, 1], [20, 9]), (256, 8, 4, [12, 1], [20, 9]), (128, 8, 2, [150], [200]), (128, 28, 4, [3000], [8])])
@pytest.mark.parametrize("window", [1 << 20, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5])
def test_a_window_wider_than_every_context_is_none(ops, d, hq, hkv, lens, nodes, window):
    """Also where there are more drafts than tokens; and it leaves the choice of key parts alone."""
    from turboquant_vllm import _native as nv

    pr = Prims(d)
    case = build_paged_case(lens, hkv, d, 16, pr, seed=3, padded=True)
    mask = pack(ancestor_matrix(nodes, random_parents(nodes, random.Random(1), 3)), -(-max(nodes) // 32))
    q = torch.randn(sum(nodes), hq, d, generator=torch.Generator().manual_seed(3)).half()
    got = []
    for w in (None, window):
        lse = torch.empty(sum(nodes), hq, device="cuda")
        nv.profile_start(8)
        out = _call(ops, q, case, nodes, mask, pr.cuda(), hkv, 16, lse_out=lse, sliding_window=w)
        got.append((out, lse, len(nv.profile_read(nv.PROF_COMBINE, 8))))
        nv.profile_stop()
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1]) and got[0][2] == got[1][2]
    assert (got[0][1] > -math.inf).any()
