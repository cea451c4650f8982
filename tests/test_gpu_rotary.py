"""Rotary positions against 64-bit arithmetic."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from turboquant_vllm.kernels import ops as _ops

    return _ops


def reference(x, positions, inv_freq, interleaved, factor=1.0, inverse=False):
    angle = positions.double()[:, None, None] * inv_freq.double() * (-1 if inverse else 1)
    rot = 2 * inv_freq.numel()
    y = x.double().clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = factor * (x[..., a].double() * angle.cos() - x[..., b].double() * angle.sin())
    y[..., b] = factor * (x[..., b].double() * angle.cos() + x[..., a].double() * angle.sin())
    return y


def tolerance(x, dtype, factor=1.0):
    """Cosine and sine to 2^-22 (the turn as a float: 2^-25 of a turn, pi 2^-24; the function's own 2 units; the factor), two products
    and a sum in fp32; then half a step of the output's type."""
    size = factor * x.double().abs().amax() * 2
    return float(size * (2 ** -22 + 3 * 2 ** -24 + torch.finfo(dtype).eps / 2))


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("t,hq,hkv,d,rot", [
    (1, 32, 8, 128, 128), (37, 28, 4, 128, 64), (300, 4, 1, 96, 96), (1500, 14, 2, 64, 64), (5, 8, 4, 256, 256), (9, 3, 3, 128, 6),
    (11, 2, 1, 80, 20), (1, 1, 1, 2, 2), (3, 1, 0, 128, 128), (4, 200, 8, 256, 64), (700, 2, 2, 10, 8), (2, 1, 1, 1024, 1024)])
def test_rotary(ops, dtype, interleaved, t, hq, hkv, d, rot):
    g = torch.Generator().manual_seed(t + d)
    x = [torch.randn(t, h, d, generator=g).to(DTYPES[dtype]) for h in (hq, hkv)]
    pos = torch.randint(0, 1 << 20, (t,), generator=g)
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    for positions in (pos, pos.int()):
        got = ops.tq4_rotary(x[0].cuda(), x[1].cuda() if hkv else None, positions.cuda(), freq.cuda(), interleaved=interleaved)
        for y, z in zip(got, x):
            if y is None:
                assert hkv == 0
                continue
            want = reference(z, pos, freq, interleaved)
            assert y.dtype == z.dtype and y.shape == z.shape
            assert (y.cpu().double() - want).abs().max() <= tolerance(z, z.dtype)
            assert torch.equal(y.cpu()[..., rot:], z[..., rot:])  # handed through


def test_far_negative_and_zero_positions(ops):
    """The angle is exact whatever the position: far ones lose nothing, and zero is the identity."""
    pos = torch.tensor([0, 1, -1, 131071, -131072, 10 ** 7, 2 ** 31 - 1, -(2 ** 31), 2 ** 40])
    x = torch.randn(len(pos), 2, 64, generator=torch.Generator().manual_seed(0))
    freq = 500000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    y, _ = ops.tq4_rotary(x.cuda(), None, pos.cuda(), freq.cuda())
    # 64-bit arithmetic itself is off by 2^-53 of the angle here: 2^40 * 2^-53 = 2^-13 at the last position
    for i, p in enumerate(pos.tolist()):
        want = reference(x[i : i + 1], pos[i : i + 1], freq, False)
        assert (y[i].cpu().double() - want[0]).abs().max() <= tolerance(x, x.dtype) + 8 * abs(p) * 2 ** -52, p
    assert torch.equal(y[0].cpu(), x[0])


def test_angles_against_whole_turns(ops):
    """Frequencies of 2 pi / n: position n is a whole turn, n / 2 a half one, by integer arithmetic."""
    n = torch.tensor([2, 3, 7, 64], dtype=torch.float64)
    freq = 2 * torch.pi / n
    x = torch.ones(1, 1, 8)
    for turns in (0, 1, 1000, 10 ** 6):
        pos = torch.tensor([2 * 3 * 7 * 64 * turns + 1])
        got = ops.tq4_rotary(x.cuda(), None, pos.cuda(), freq.cuda())[0].cpu().double()
        want = reference(x, torch.tensor([1]), freq, False)
        # (the frequency itself has a rounding of 2^-53 of it, which the position multiplies)
        assert (got - want).abs().max() <= tolerance(x, x.dtype) + 2 * float(pos) * float(freq.max()) * 2 ** -53


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_factor_float_frequencies_and_the_gradient(ops, interleaved):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(50, 4, 128, generator=g)
    pos = torch.randint(0, 5000, (50,), generator=g)
    freq = 10000.0 ** (-torch.arange(0, 96, 2, dtype=torch.float32) / 96)
    kw = dict(interleaved=interleaved, attention_factor=1.25)
    y, _ = ops.tq4_rotary(x.cuda(), None, pos.cuda(), freq.cuda(), **kw)
    assert (y.cpu().double() - reference(x, pos, freq, interleaved, 1.25)).abs().max() <= tolerance(x, x.dtype, 1.25)
    back, _ = ops.tq4_rotary(y, None, pos.cuda(), freq.cuda(), inverse=True, interleaved=interleaved, attention_factor=0.8)
    assert (back.cpu() - x).abs().max() <= 2 * tolerance(x, x.dtype, 1.25)
    # the gradient of the turn is the turn back: against the formula's
    z = x.double().clone().requires_grad_(True)
    out = torch.randn(50, 4, 128, generator=g)
    (reference_autograd(z, pos, freq, interleaved, 1.25) * out.double()).sum().backward()
    grad, _ = ops.tq4_rotary(out.cuda(), None, pos.cuda(), freq.cuda(), inverse=True, **kw)
    assert (grad.cpu().double() - z.grad).abs().max() <= tolerance(out, out.dtype, 1.25)


def reference_autograd(x, positions, inv_freq, interleaved, factor):
    angle = positions.double()[:, None, None] * inv_freq.double()
    rot = 2 * inv_freq.numel()
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
    u, v = factor * (a * angle.cos() - b * angle.sin()), factor * (b * angle.cos() + a * angle.sin())
    turned = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((turned, x[..., rot:]), dim=-1)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("pad", [0, 8, 3])
def test_in_place_on_parts_of_a_projection(ops, dtype, pad):
    """Queries and keys as views of one projection's output, rotated in place, and into rows of another buffer; values stay."""
    g = torch.Generator().manual_seed(5)
    full = torch.randn(70, 8 + 2 + 2, 128 + pad, generator=g).to(DTYPES[dtype]).cuda()
    before = full.clone()
    q, k = full[:, :8, :128], full[:, 8:10, :128]
    pos, freq = torch.arange(70).cuda() * 37, (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).cuda()
    want = ops.tq4_rotary(before[:, :8, :128].contiguous(), before[:, 8:10, :128].contiguous(), pos, freq)
    other = torch.full_like(full, 9.0)
    out = (other[:, :8, :128], other[:, 8:10, :128])
    assert ops.tq4_rotary(q, k, pos, freq, out=out) is not None
    assert torch.equal(full, before) and all(torch.equal(a, b) for a, b in zip(out, want))
    assert (other[:, 10:] == 9).all() and (other[:, :, 128:] == 9).all()
    got = ops.tq4_rotary(q, k, pos, freq, out=(q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(full[:, 10:], before[:, 10:]) and torch.equal(full[..., 128:], before[..., 128:])


def test_odd_addresses_equal_aligned_ones(ops):
    g = torch.Generator().manual_seed(6)
    x = torch.randn(33, 5, 128, generator=g).bfloat16().cuda()
    pos, freq = torch.arange(33).cuda(), (10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)).cuda()
    want, _ = ops.tq4_rotary(x, None, pos, freq)
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    odd = flat[1:].view(x.shape).copy_(x)
    assert torch.equal(ops.tq4_rotary(odd, None, pos, freq)[0], want)
    even = x.transpose(0, 1).contiguous().transpose(0, 1)  # heads outside tokens
    assert torch.equal(ops.tq4_rotary(even, None, pos, freq)[0], want)


def test_infinities_and_nan_stay_where_they_are(ops):
    x = torch.randn(4, 2, 64, generator=torch.Generator().manual_seed(1))
    x[1, 0, 3], x[2, 1, 40] = float("inf"), float("nan")
    freq = 10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    y, _ = ops.tq4_rotary(x.cuda(), None, torch.tensor([3, 5, 6, 7]).cuda(), freq.cuda())
    bad = ~torch.isfinite(y.cpu())
    assert bad.sum() == 4 and bad[1, 0, [3, 35]].all() and bad[2, 1, [8, 40]].all()
    freq[2] = float("inf")
    y, _ = ops.tq4_rotary(torch.ones(1, 1, 64).cuda(), None, torch.tensor([1]).cuda(), freq.cuda())
    assert torch.isnan(y[0, 0, [2, 34]]).all() and torch.isfinite(y).sum() == 62


def test_refusals(ops):
    q, k = torch.zeros(4, 2, 64, device="cuda"), torch.zeros(4, 1, 64, device="cuda")
    pos, freq = torch.arange(4).cuda(), torch.ones(32, dtype=torch.float64, device="cuda")

    def refused(error, match, *args, **kw):
        with pytest.raises(error, match=match):
            ops.tq4_rotary(*args, **kw)

    refused(RuntimeError, "CUDA", q.cpu(), k, pos, freq)
    refused(RuntimeError, "CUDA", q, k, pos.cpu(), freq)
    refused(TypeError, "float32/float16/bfloat16", q.double(), k.double(), pos, freq)
    refused(AssertionError, "same tokens", q, k.half(), pos, freq)
    refused(AssertionError, "same tokens", q, k[:3], pos, freq)
    refused(AssertionError, "positions", q, k, pos[:3], freq)
    refused(AssertionError, "positions", q, k, pos.float(), freq)
    refused(AssertionError, "inv_freq", q, k, pos, freq.half())
    refused(AssertionError, "inv_freq", q, k, pos, torch.ones(33, device="cuda"))
    refused(AssertionError, "inv_freq", q, k, pos, torch.ones(0, device="cuda"))
    refused(AssertionError, "out must be a pair", q, k, pos, freq, out=q)
    refused(AssertionError, "shape and type", q, k, pos, freq, out=(q.half(), k))
    refused(AssertionError, "input or not overlap", q[:3], None, pos[:3], freq, out=(q[1:], None))
    refused(AssertionError, "may not overlap", q, k, pos, freq, out=(q, q[:, :1]))
    refused(AssertionError, "may not be expanded", q, None, pos, freq, out=(torch.empty(1, 2, 64, device="cuda").expand(4, 2, 64), None))
    refused(NotImplementedError, "tq4_rotary", torch.zeros(1, 1, 2048, device="cuda"), None, pos[:1], torch.ones(600, device="cuda"))
    empty = ops.tq4_rotary(q[:0], k[:0], pos[:0], freq)
    assert empty[0].shape == (0, 2, 64) and empty[1].shape == (0, 1, 64)


def test_captured(ops):
    g = torch.Generator().manual_seed(9)
    q, k = (torch.randn(16, h, 128, generator=g).half().cuda() for h in (32, 8))
    pos, freq = torch.arange(16).cuda(), (10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)).cuda()
    out = torch.empty_like(q), torch.empty_like(k)
    ops.tq4_rotary(q, k, pos, freq, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.tq4_rotary(q, k, pos, freq, out=out)
    pos += 1000
    graph.replay()
    want = ops.tq4_rotary(q, k, pos, freq)
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_in_place_through_another_view_of_one_token(ops):
    """Strides of dimensions of one element say nothing: these are the same places."""
    x = torch.randn(1, 4, 128, generator=torch.Generator().manual_seed(2)).cuda()
    pos, freq = torch.tensor([7]).cuda(), (10000.0 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)).cuda()
    want, _ = ops.tq4_rotary(x, None, pos, freq)
    for shape, strides in (((1, 4, 128), (7, 128, 1)), ((4, 1, 128), (128, 3, 1))):
        mine = x.clone().view(shape)
        p = pos.expand(shape[0]).contiguous()
        out = mine.as_strided(shape, strides)
        assert ops.tq4_rotary(mine, None, p, freq, out=(out, None))[0] is out
        assert torch.equal(mine.view(1, 4, 128), want)
