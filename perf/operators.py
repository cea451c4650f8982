"""The operators of a server that drafts several tokens a step over the packed cache, as cases to measure.

One step of such a server: the queries and keys of the drafted tokens get their rotary positions (``tq4_rotary``), the tree of
drafts becomes bits (``tq4_tree_mask``), every layer attends over its pages (``paged_tq4_tree_attention``), the token rows of
the accepted path move together (``tq4_compact_rows``, which also serves an eviction from long contexts), and a sequence that
is forked takes copies of pages along (``tq4_copy_blocks``).

Model shapes are the ones of this repository's benchmark configurations and tests.  Keys and values are N(0, 1) with four
outlier channels scaled by 8, queries N(0, 1); block tables are shuffled; token rows are vLLM's padded ones (heads x next power
of two of head_dim + 8 bytes) or, in some drawn cases, the unpadded ones.
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False  # whether run() makes the framework's calls or computes the plain form

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
OUTLIERS = (3, 17, 41, 52)
POOL = 16384  # distinct cached token rows; a cache draws its tokens from them
BLOCK = 16    # tokens per page


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------
def _tree(batch, nodes_lo, nodes_hi, ctx_lo, ctx_hi, hq, hkv, dim, dtype, window=0, dense=False):
    """``batch`` sequences of [ctx_lo, ctx_hi] tokens held, each with a tree of [nodes_lo, nodes_hi] drafted ones behind them."""
    return {"op": "tree", "batch": batch, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype, "window": window, "dense": dense}


def _mask(batch, nodes_lo, nodes_hi, reach):
    """Trees of [nodes_lo, nodes_hi] drafts whose parents lie at most ``reach`` drafts back."""
    return {"op": "mask", "batch": batch, "nodes_lo": nodes_lo, "nodes_hi": nodes_hi, "reach": reach}


def _rotary(seqs, new, far, hq, hkv, dim, rot, dtype, interleaved=False, factor=1.0, base=10000.0, inverse=False):
    """``new`` tokens of each of ``seqs`` sequences, at positions up to ``far``; the first ``rot`` dimensions of a head turn."""
    return {"op": "rotary", "seqs": seqs, "new": new, "far": far, "hq": hq, "hkv": hkv, "dim": dim, "rot": rot, "dtype": dtype,
            "interleaved": interleaved, "factor": factor, "base": base, "inverse": inverse}


def _copy(pairs, layers, hkv, dim, dense=False):
    return {"op": "copy", "pairs": pairs, "layers": layers, "hkv": hkv, "dim": dim, "dense": dense}


def _compact(batch, held, of, keep_lo, keep_hi, layers, hkv, dim, dense=False):
    """[keep_lo, keep_hi] of the ``of`` tokens behind the first ``held`` ones stay."""
    return {"op": "compact", "batch": batch, "held": held, "of": of, "keep_lo": keep_lo, "keep_hi": keep_hi, "layers": layers,
            "hkv": hkv, "dim": dim, "dense": dense}


def listed():
    return [
        # one user's chat with a small tree, groups of 7 heads: latency
        dict(_tree(1, 8, 8, 1024, 1024, 28, 4, 128, "bf16"), name="tree-1"),
        # an ordinary moment of a server: sequences and trees of all sizes, fp16 model
        dict(_tree(16, 5, 24, 300, 8100, 32, 8, 128, "fp16"), name="tree-16-ragged"),
        # the benchmark's headline batch, each sequence with 16 drafts
        dict(_tree(64, 16, 16, 4096, 4096, 32, 8, 128, "bf16"), name="tree-64x4096"),
        # long documents with wide trees, a model without grouped queries and an odd head dimension (the largest case)
        dict(_tree(8, 48, 64, 65536, 65536, 32, 32, 96, "bf16"), name="tree-8x65536-d96"),
        # the masks of the ordinary moment above, and of a batch of large trees
        dict(_mask(16, 5, 24, 5), name="mask-16"),
        dict(_mask(64, 200, 512, 40), name="mask-64x512"),
        # queries and keys of 16 sequences with 8 drafts each, far into long contexts
        dict(_rotary(16, 8, 131072, 32, 8, 128, 128, "bf16", base=500000.0), name="rotary-16x8"),
        # a full prefill step
        dict(_rotary(8, 2048, 10240, 32, 8, 128, 128, "bf16"), name="rotary-8x2048"),
        # eight sequences forked: each copies its last page, in all layers
        dict(_copy(8, 32, 8, 128), name="copy-8"),
        # a prefix of 32 768 tokens duplicated
        dict(_copy(2048, 8, 8, 128), name="copy-2048"),
        # the accepted drafts of a batch of 64 with trees of 16, in all layers
        dict(_compact(64, 1000, 16, 1, 6, 32, 8, 128), name="accept-64x16"),
        # half of four long contexts evicted
        dict(_compact(4, 0, 16384, 8192, 8192, 8, 8, 128), name="evict-4x16384"),
    ]


# query heads, KV heads, head_dim, sliding window: the shapes of the benchmark configurations and the tests
SHAPES = ((32, 8, 128, 0), (32, 8, 128, 0), (28, 4, 128, 0), (4, 1, 128, 0), (32, 32, 96, 0), (14, 2, 64, 0), (8, 4, 256, 4096))


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    hq, hkv, dim, window = rng.choice(SHAPES)
    dense = rng.random() < 0.25
    op = rng.choice(("tree", "tree", "tree", "tree", "mask", "rotary", "rotary", "copy", "compact", "compact"))
    if op == "tree":
        batch, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
        # bytes, scores and operations of a case stay below those of the largest listed one
        most = int(min(65536, 1.7e9 / (batch * hkv * (dim + 8)), 1e9 / (batch * hq * nodes), 4e11 / (4 * dim * hq * nodes * batch)))
        ctx = _log_int(rng, 30, max(30, most))
        return _tree(batch, max(1, nodes // rng.choice((1, 1, 4))), nodes, max(0, ctx // rng.choice((1, 20))), ctx, hq, hkv, dim,
                     rng.choice(("bf16", "bf16", "fp16")), window, dense)
    if op == "mask":
        nodes = _log_int(rng, 1, 512)
        return _mask(_log_int(rng, 1, 64), max(1, nodes // 3), nodes, _log_int(rng, 1, 64))
    if op == "rotary":
        seqs = _log_int(rng, 1, 64)
        return _rotary(seqs, _log_int(rng, 1, 16384 // seqs), rng.choice((20000, 131072, 1000000)), hq, hkv, dim,
                       rng.choice((dim, dim, dim // 2, 2 * rng.randint(1, dim // 2))), rng.choice(("bf16", "bf16", "fp16", "fp32")),
                       rng.random() < 0.4, rng.choice((1.0, 1.0, 1.1386)), rng.choice((10000.0, 500000.0)), rng.random() < 0.2)
    if op == "copy":
        layers = rng.choice((1, 8, 32))
        return _copy(_log_int(rng, 1, min(4096, int(2.8e8 / (layers * BLOCK * hkv * (dim + 8))))), layers, hkv, dim, dense)
    layers = rng.choice((1, 8, 32))
    if rng.random() < 0.5:
        of = _log_int(rng, 1, 64)
        return _compact(_log_int(rng, 1, 64), rng.randint(1, 2000), of, 0, min(of, 8), layers, hkv, dim, dense)
    batch = _log_int(rng, 1, 8)
    of = _log_int(rng, 100, min(16384, int(5.6e8 / (layers * batch * hkv * (dim + 8)))))
    return _compact(batch, rng.choice((0, 4)), of, of // 3, of - of // 4, layers, hkv, dim, dense)


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------
def _spread(n: int, lo: int, hi: int) -> list[int]:
    """``n`` numbers spread evenly over [lo, hi] (a case is of one size for every seed)."""
    return [lo + round((hi - lo) * (i + 0.5) / n) for i in range(n)]


def _shuffled(items: list, seed: int) -> list:
    items = list(items)
    random.Random(seed).shuffle(items)
    return items


_codebooks: dict = {}


def _codebook(dim: int):
    """Rotation, centroids and boundaries of a model's cache (a program makes them once)."""
    if dim not in _codebooks:
        x = torch.randn(dim, dim, generator=torch.Generator().manual_seed(42))
        rotation = torch.linalg.qr(x)[0]
        sd = dim ** -0.5
        cents = [sd * (-3 + 6 * (i + 0.5) / 16) for i in range(16)]
        pdf = lambda z: math.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)  # noqa: E731
        cdf = lambda z: 0.5 * (1 + math.erf(z / math.sqrt(2)))  # noqa: E731
        for _ in range(200):  # Lloyd-Max for N(0, 1 / dim) within three standard deviations
            edge = [-3.0] + [(a + b) / 2 / sd for a, b in zip(cents, cents[1:])] + [3.0]
            cents = [sd * (pdf(a) - pdf(b)) / (cdf(b) - cdf(a)) for a, b in zip(edge, edge[1:])]
        bounds = [(a + b) / 2 for a, b in zip(cents, cents[1:])]
        _codebooks[dim] = tuple(t.to("cuda", torch.float32).contiguous() for t in (rotation, torch.tensor(cents), torch.tensor(bounds)))
    return _codebooks[dim]


def _width(hkv: int, dim: int, dense: bool) -> int:
    return (hkv * (dim + 8) + 15) // 16 * 16 if dense else hkv * (1 << (dim + 7).bit_length())


def _cached_rows(n: int, hkv: int, dim: int, dense: bool, gen) -> torch.Tensor:
    """``n`` token rows [K indices | K norms | V indices | V norms | padding] of keys and values as they are cached."""
    rotation, _, bounds = _codebook(dim)
    pool = min(n, max(64, POOL // hkv))
    parts = []
    for _ in range(2):
        x = torch.randn(pool * hkv, dim, device="cuda", generator=gen)
        x[:, list(OUTLIERS)] *= 8.0
        norm = x.norm(dim=1, keepdim=True)
        idx = torch.bucketize((x / (norm + 1e-10)) @ rotation.T, bounds).to(torch.uint8)
        parts += [((idx[:, 0::2] << 4) | idx[:, 1::2]).reshape(pool, -1), norm.reshape(pool, hkv).view(torch.uint8)]
    rows = torch.zeros(pool, _width(hkv, dim, dense), dtype=torch.uint8, device="cuda")
    data = torch.cat(parts, dim=1)
    rows[:, : data.shape[1]] = data
    return rows.view(torch.int64)[torch.randint(pool, (n,), device="cuda", generator=gen)].view(torch.uint8)


def _table(lens: list[int], gen, extra: int = 2):
    """A shuffled block table for sequences of these lengths, and how many pages the cache has."""
    need = [max(1, -(-n // BLOCK)) for n in lens]
    blocks = sum(need) + extra
    order = torch.randperm(blocks, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda")
    at = torch.arange(max(need), device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[at] = order[: sum(need)]
    return table, blocks


def _parents(nodes: list[int], reach: int, rng: random.Random) -> list[int]:
    """Of every draft the one it continues, by its place in its tree (-1: the first drafts, behind the tokens held)."""
    return [rng.randint(max(-1 if j < 3 else 0, j - reach), j - 1) for n in nodes for j in range(n)]


def _ancestor_bits(nodes: list[int], parents: list[int], words: int) -> list[list[int]]:
    bits, first = [], 0
    for n in nodes:
        for j in range(n):
            p = parents[first + j]
            bits.append((bits[first + p] if p >= 0 else 0) | 1 << j)
        first += n
    word = [[b >> 32 * w & 0xFFFFFFFF for w in range(words)] for b in bits]
    return [[x - (1 << 32) if x >> 31 else x for x in w] for w in word]


def _starts(counts: list[int]) -> torch.Tensor:
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")


def _nodes(c, seed):
    return _shuffled(_spread(c["batch"], c["nodes_lo"], c["nodes_hi"]), seed)


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed)
    s = {"case": c}
    if c["op"] == "tree":
        nodes = _nodes(c, seed)
        lens = [a + b for a, b in zip(_shuffled(_spread(c["batch"], c["ctx_lo"], c["ctx_hi"]), seed + 1), nodes)]
        s["table"], blocks = _table(lens, gen)
        s["cache"] = _cached_rows(blocks * BLOCK, c["hkv"], c["dim"], c["dense"], gen).view(blocks, BLOCK, -1)
        s["lens"], s["starts"] = torch.tensor(lens, dtype=torch.int32, device="cuda"), _starts(nodes)
        words = -(-max(nodes) // 32)
        s["mask"] = torch.tensor(_ancestor_bits(nodes, _parents(nodes, 5, rng), words), dtype=torch.int32, device="cuda")
        s["q"] = torch.randn(sum(nodes), c["hq"], c["dim"], device="cuda", generator=gen).to(DTYPES[c["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["rotation"], s["cents"], _ = _codebook(c["dim"])
        s["longest"], s["widest"] = max(lens), max(nodes)
    elif c["op"] == "mask":
        nodes = _nodes(c, seed)
        s["parents"] = torch.tensor(_parents(nodes, c["reach"], rng), dtype=torch.int32, device="cuda")
        s["starts"], s["widest"] = _starts(nodes), max(nodes)
    elif c["op"] == "rotary":
        first = torch.randint(0, max(1, c["far"] - c["new"]), (c["seqs"], 1), device="cuda", generator=gen)
        s["positions"] = (first + torch.arange(c["new"], device="cuda")).reshape(-1)
        n, dtype = c["seqs"] * c["new"], DTYPES[c["dtype"]]
        s["q"] = torch.randn(n, c["hq"], c["dim"], device="cuda", generator=gen).to(dtype)
        s["k"] = torch.randn(n, c["hkv"], c["dim"], device="cuda", generator=gen).to(dtype)
        s["out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        s["inv_freq"] = c["base"] ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
    else:
        s["data"] = c["hkv"] * (c["dim"] + 8)
        if c["op"] == "copy":
            blocks = 2 * c["pairs"] + 2
            order = torch.randperm(blocks, device="cuda", generator=gen)
            s["pairs"] = torch.stack((order[: c["pairs"]], order[c["pairs"] : 2 * c["pairs"]]), dim=1)
        else:
            lens = [c["held"] + c["of"]] * c["batch"]
            s["table"], blocks = _table(lens, gen)
            kept = _shuffled(_spread(c["batch"], c["keep_lo"], c["keep_hi"]), seed)
            order = torch.rand(c["batch"], c["of"], device="cuda", generator=gen).argsort(dim=1)
            s["kept"] = torch.tensor(kept, dtype=torch.int32, device="cuda")
            pick = torch.where(torch.arange(c["of"], device="cuda") < s["kept"][:, None], order, c["of"])
            s["keep"] = pick.sort(dim=1).values[:, : max(1, max(kept))].to(torch.int32).contiguous()
            s["first"] = torch.full((c["batch"],), c["held"], dtype=torch.int32, device="cuda")
            s["lens"] = torch.empty(c["batch"], dtype=torch.int32, device="cuda")
        s["kv"] = torch.randint(0, 256, (c["layers"], blocks, BLOCK, _width(c["hkv"], c["dim"], c["dense"])), device="cuda",
                                generator=gen, dtype=torch.uint8)
        s["layers"] = list(s["kv"])  # a cache tensor a layer, as an engine holds them
    return s


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if own:
        K = _kernels()
        if c["op"] == "tree":
            return K.paged_tq4_tree_attention(
                s["q"], s["cache"], s["table"], s["lens"], s["starts"], s["mask"], s["cents"], s["cents"], s["rotation"], c["hkv"],
                BLOCK, sliding_window=c["window"] or None, out=s["out"], max_seq_len=s["longest"])
        if c["op"] == "mask":
            return K.tq4_tree_mask(s["parents"], s["starts"], s["widest"])
        if c["op"] == "rotary":
            return K.tq4_rotary(s["q"], s["k"], s["positions"], s["inv_freq"], interleaved=c["interleaved"],
                                attention_factor=c["factor"], inverse=c["inverse"], out=s["out"])
        if c["op"] == "copy":
            K.tq4_copy_blocks(s["layers"], s["pairs"], c["hkv"], c["dim"])
            return s["kv"]
        K.tq4_compact_rows(s["layers"], s["table"], s["first"], s["keep"], s["kept"], c["hkv"], c["dim"], seq_lens_out=s["lens"])
        return s["kv"], s["lens"]
    return {"tree": _plain_tree, "mask": _plain_mask, "rotary": _plain_rotary, "copy": _plain_copy, "compact": _plain_compact}[c["op"]](s)


def _kernels():
    package = os.path.join(os.getcwd(), "turboquant-vllm_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    import turboquant_vllm.kernels as kernels

    return kernels


def _places(starts: torch.Tensor, rows: int):
    """Sequence and place within it of every row."""
    row = torch.arange(rows, device=starts.device)
    seq = (row[:, None] >= starts[None, 1:]).sum(dim=1)
    return seq, row - starts.long()[seq]


def _plain_tree(s):
    c = s["case"]
    hkv, dim, group = c["hkv"], c["dim"], c["hq"] // c["hkv"]
    rows, most = s["q"].shape[0], s["longest"]
    seq, place = _places(s["starts"], rows)
    pos = torch.arange(most, device="cuda")
    held = s["cache"].flatten(0, 1)[s["table"].long()[:, pos // BLOCK] * BLOCK + pos % BLOCK]  # [B, L, width]
    half = hkv * (dim // 2 + 4)

    def vectors(part):  # centroids times norm, in rotated space: [B, H, L, D]
        idx, norm = part[..., : hkv * dim // 2].unflatten(2, (hkv, dim // 2)), part[..., hkv * dim // 2 :].contiguous().view(torch.float32)
        both = torch.stack((idx >> 4, idx & 15), dim=4).flatten(3)
        return (s["cents"][both.int()] * norm[..., None]).transpose(1, 2)

    q = s["q"].float() @ s["rotation"].T
    padded = q.new_zeros(c["batch"], s["widest"], c["hq"], dim)
    padded[seq, place] = q
    padded = padded.unflatten(2, (hkv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, H, group * T, D]
    score = padded @ vectors(held[..., :half]).transpose(2, 3) * dim ** -0.5
    score = score.unflatten(2, (group, s["widest"]))
    # what a row sees: the tokens held (within its window), and of the drafts those of its bits
    lens, count = s["lens"].long(), s["starts"].long().diff()
    base = (lens - count)[seq]
    node = pos[None, :] - base[:, None]
    bit = s["mask"].gather(1, (node.clamp(0, 32 * s["mask"].shape[1] - 1) >> 5)) >> (node & 31) & 1
    bits = s["mask"][:, :, None] >> torch.arange(32, device="cuda") & 1
    low = base + bits.sum(dim=(1, 2)) - c["window"] if c["window"] else torch.zeros_like(base)
    sees = torch.where(node < 0, pos[None, :] >= low[:, None], bit.bool()) & (node < count[seq][:, None])
    visible = torch.zeros(c["batch"], s["widest"], most, dtype=torch.bool, device="cuda")
    visible[seq, place] = sees
    score = score.masked_fill(~visible[:, None, None], -math.inf)
    top = score.amax(dim=-1, keepdim=True)
    weight = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = weight.sum(dim=-1, keepdim=True)
    mixed = (weight.flatten(2, 3) @ vectors(held[..., half : 2 * half])).unflatten(2, (group, s["widest"]))
    mixed = torch.where(total > 0, mixed / total, 0.0).permute(0, 3, 1, 2, 4).flatten(2, 3)[seq, place]
    return (mixed @ s["rotation"]).to(s["q"].dtype)


def _plain_mask(s):
    rows, widest = s["parents"].shape[0], s["widest"]
    seq, place = _places(s["starts"], rows)
    step = torch.zeros(s["starts"].shape[0] - 1, widest, widest, device="cuda")
    has = s["parents"] >= 0
    step[seq[has], place[has], s["parents"][has].long()] = 1.0
    one = torch.eye(widest, device="cuda").expand_as(step)
    reach = torch.linalg.solve_triangular(one - step, one, upper=False)  # 1 + step + step^2 + ...: itself and its ancestors
    reach = reach[seq, place] > 0.5
    words = -(-widest // 32)
    bits = torch.zeros(rows, 32 * words, dtype=torch.int64, device="cuda")
    bits[:, :widest] = reach
    word = (bits.unflatten(1, (words, 32)) << torch.arange(32, device="cuda")).sum(dim=2)
    return torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32), (reach.sum(dim=1) - 1).to(torch.int32)


def _plain_rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["inv_freq"] * (-1 if c["inverse"] else 1)
    cos, sin = ((f(angle) * c["factor"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(x):
        part, rest = x.float()[..., : c["rot"]], x[..., c["rot"] :]
        a, b = (part[..., 0::2], part[..., 1::2]) if c["interleaved"] else part.chunk(2, dim=-1)
        a, b = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack((a, b), dim=-1).flatten(-2) if c["interleaved"] else torch.cat((a, b), dim=-1)
        return torch.cat((turned.to(x.dtype), rest), dim=-1)

    return turn(s["q"]), turn(s["k"])


def _plain_copy(s):
    s["kv"][:, s["pairs"][:, 1], :, : s["data"]] = s["kv"][:, s["pairs"][:, 0], :, : s["data"]]
    return s["kv"]


def _plain_compact(s):
    rows = s["kv"].flatten(1, 2)
    slot = torch.arange(s["keep"].shape[1], device="cuda")
    there = (slot < s["kept"][:, None]).reshape(-1)

    def flat(pos):
        pos = pos.clamp(max=BLOCK * s["table"].shape[1] - 1)
        return (s["table"].long().gather(1, pos // BLOCK) * BLOCK + pos % BLOCK).reshape(-1)[there]

    first = s["first"].long()[:, None]
    rows[:, flat(first + slot), : s["data"]] = rows[:, flat(first + s["keep"]), : s["data"]]
    s["lens"].copy_(s["first"] + s["kept"])
    return s["kv"], s["lens"]


# --------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "tree":
        nodes = _spread(c["batch"], c["nodes_lo"], c["nodes_hi"])
        ctx = [min(n, c["window"] or n) for n in _spread(c["batch"], c["ctx_lo"], c["ctx_hi"])]
        rows = sum(nodes)
        # (the order of the trees among the sequences changes with the seed: on average)
        keys, pairs = sum(ctx) + rows, rows * sum(ctx) / c["batch"] + rows
        return {"bytes": keys * c["hkv"] * (c["dim"] + 8) + 4 * rows * c["hq"] * c["dim"],
                "flops": 4 * c["dim"] * c["hq"] * pairs + 4 * rows * c["hq"] * c["dim"] ** 2}
    if c["op"] == "mask":
        rows = sum(_spread(c["batch"], c["nodes_lo"], c["nodes_hi"]))
        return {"bytes": rows * 4 * (2 + -(-c["nodes_hi"] // 32)), "flops": 0}
    if c["op"] == "rotary":
        vectors = c["seqs"] * c["new"] * (c["hq"] + c["hkv"])
        return {"bytes": 2 * vectors * c["dim"] * (4 if c["dtype"] == "fp32" else 2) + 8 * c["seqs"] * c["new"],
                "flops": 3 * vectors * c["rot"]}
    rows = BLOCK * c["pairs"] if c["op"] == "copy" else sum(_spread(c["batch"], c["keep_lo"], c["keep_hi"]))
    return {"bytes": max(1, 2 * rows * c["layers"] * c["hkv"] * (c["dim"] + 8)), "flops": 0}


# --------------------------------------------------------------------------------------------------
# the same in 64 bits, from the definitions
# --------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] not in ("tree", "rotary"):
        return None  # (bytes and whole numbers)
    s, c = prepare(case, seed), case
    if c["op"] == "rotary":
        turn = torch.polar(torch.full((), c["factor"], dtype=torch.float64, device="cuda"),
                           s["positions"].double()[:, None, None] * s["inv_freq"])
        turn = turn.conj() if c["inverse"] else turn
        outs = []
        for x in (s["q"].double(), s["k"].double()):
            r, h = c["rot"], c["rot"] // 2
            even, odd = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, h), slice(h, r))
            z = torch.complex(x[..., even], x[..., odd]) * turn
            y = x.clone()
            y[..., even], y[..., odd] = z.real, z.imag
            outs.append(y)
        return tuple(outs)
    pi, cents = s["rotation"].double(), s["cents"].double()
    hkv, dim, group = c["hkv"], c["dim"], c["hq"] // c["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    byte = torch.arange(256, device="cuda")
    pair = torch.stack((cents[byte // 16], cents[byte % 16]), dim=1)  # the two centroids of a byte
    for i, n in enumerate(lens):
        r0, r1 = starts[i], starts[i + 1]
        base = n - (r1 - r0)
        p = torch.arange(n, device="cuda")
        held = s["cache"][s["table"][i, p // BLOCK].long(), p % BLOCK]
        at, vec = 0, []
        for _ in range(2):
            idx = held[:, at : at + hkv * dim // 2].reshape(n, hkv, dim // 2)
            at += hkv * dim // 2
            norm = held[:, at : at + 4 * hkv].contiguous().view(torch.float32).double()
            at += 4 * hkv
            vec.append(((pair[idx.long()].flatten(2)) @ pi) * norm[:, :, None])
        words = s["mask"][r0:r1].long() & 0xFFFFFFFF
        bits = (words[:, :, None] >> torch.arange(32, device="cuda") & 1).flatten(1).bool()[:, : r1 - r0]
        sees = torch.ones(r1 - r0, n, dtype=torch.bool, device="cuda")
        sees[:, base:] = bits
        if c["window"]:
            mine = base + bits.sum(dim=1) - 1  # a row's own position
            sees[:, :base] = p[None, :base] > mine[:, None] - c["window"]
        for h in range(hkv):
            q = s["q"][r0:r1, h * group : (h + 1) * group].double()
            a = torch.einsum("tgd,nd->tgn", q, vec[0][:, h]) / math.sqrt(dim)
            a = torch.softmax(a.masked_fill(~sees[:, None], -math.inf), dim=-1).nan_to_num(0.0)
            out[r0:r1, h * group : (h + 1) * group] = torch.einsum("tgn,nd->tgd", a, vec[1][:, h])
    return out
