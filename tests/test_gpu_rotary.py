"""Rotary embedding by position against a plain 64-bit counterpart."""
import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def tolerance(ref, x, dtype, mscale):
    """Result rounded to its type (half a step of it; fp16 also has a smallest step, 2^-24); sine and cosine are fp32
    values of a fraction of a turn that is itself rounded to fp32 (2^-25 turns = 2^-25 * 2 pi radians), two ulps of the
    function and one of the mscale product, and the two products and their sum round three times: 2^-20 of |a| + |b|."""
    size = np.abs(x).max(-1, keepdims=True) * 2 * abs(mscale)
    return HALF_STEP[dtype] * np.abs(ref) + 2.0 ** -20 * size + (2.0 ** -25 if dtype == torch.float16 else 0)


def check(x, pos, freq, layout, mscale=1.0, inverse=False, out=None):
    import magi_b200 as mb
    before = x.double().cpu().numpy()
    got = mb.rotary(x, pos, freq, layout=layout, mscale=mscale, inverse=inverse, out=out)
    ref = R.rotary(before, pos.cpu().numpy(), freq.cpu().numpy(), layout, mscale, inverse)
    assert (np.abs(got.double().cpu().numpy() - ref) <= tolerance(ref, before, x.dtype, mscale)).all()
    rot = 2 * freq.shape[0]
    assert np.array_equal(got.double().cpu().numpy()[..., rot:], before[..., rot:])
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(1, 1, 128, 128), (1, 48, 128, 96), (7, 3, 64, 64), (33, 5, 80, 32), (5, 2, 96, 50), (130, 8, 256, 256), (3, 1, 6, 2),
                                       (9, 4, 128, 0), (600, 1, 64, 16), (64, 56, 128, 128)])
def test_values(dtype, layout, T, H, D, rot):
    import magi_b200 as mb
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, H, D, generator=g).to(dtype).cuda()
    pos = torch.randint(0, 5000, (T,), generator=g).int().cuda()
    freq = mb.rotary_frequencies(rot)[0] if rot else torch.empty(0, dtype=torch.float64, device="cuda")
    for inverse in (False, True):
        check(x, pos, freq, layout, 1.1, inverse)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_alignment_and_in_place(layout):
    import magi_b200 as mb
    freq, _ = mb.rotary_frequencies(64)
    pos = torch.arange(21, device="cuda")  # int64
    big = torch.randn(21, 9, 200, device="cuda").to(torch.bfloat16)
    for view in (big[:, 1:7, 8:136], big[:, ::2, 3:131], big[:, :, :128].transpose(0, 1).contiguous().transpose(0, 1), big[::2, :, 1:101]):
        check(view, pos[:view.shape[0]].contiguous(), freq, layout)
    x = big[:, 2:5, 16:144]
    rest = big.clone()
    want = mb.rotary(x, pos, freq, layout=layout)
    assert mb.rotary(x, pos, freq, layout=layout, out=x) is x and torch.equal(x, want)
    rest[:, 2:5, 16:144] = want
    assert torch.equal(big, rest)  # nothing beside it was touched


def test_far_and_negative_positions():
    """At a million positions the phase of the fastest pair is still right to fp32's fraction of a turn."""
    import magi_b200 as mb
    x = torch.randn(6, 2, 128, device="cuda")
    for scaling in (dict(), dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0), dict(scaling="yarn", factor=16.0, original_context=4096)):
        freq, mscale = mb.rotary_frequencies(128, **scaling)
        check(x, torch.tensor([0, 1, 999_999, 2 ** 31 - 1, -5, 10 ** 6 + 7], dtype=torch.int64, device="cuda"), freq, "half", mscale)
        check(x, torch.tensor([0, 1, 999_999, 2 ** 31 - 1, -5, 10 ** 6 + 7], dtype=torch.int32, device="cuda"), freq, "interleaved", mscale)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_the_inverse_is_the_gradient(layout):
    """Against the formula (<R x, y> = <x, R^T y>) and against differences: R is linear, so a difference quotient of step 1
    is exact up to rounding."""
    import magi_b200 as mb
    freq, _ = mb.rotary_frequencies(48)
    pos = torch.tensor([3, 70000, 11, 0], dtype=torch.int32, device="cuda")
    x, y = torch.randn(2, 4, 3, 64, device="cuda")
    grad = mb.rotary(y, pos, freq, layout=layout, mscale=1.3, inverse=True)
    left = (mb.rotary(x, pos, freq, layout=layout, mscale=1.3).double() * y.double()).sum()
    assert abs(float(left - (x.double() * grad.double()).sum())) <= 2.0 ** -18 * float((x.abs() * y.abs()).sum()) * 2.6
    base = mb.rotary(x, pos, freq, layout=layout, mscale=1.3).double()
    for t, h, d in ((0, 0, 0), (1, 2, 5), (1, 1, 47), (2, 0, 30), (3, 2, 63), (1, 0, 24)):
        moved = x.clone()
        moved[t, h, d] += 1
        quotient = ((mb.rotary(moved, pos, freq, layout=layout, mscale=1.3).double() - base) * y.double()).sum()
        assert abs(float(quotient - grad[t, h, d].double())) <= 2.0 ** -18 * float(1 + x[t, h].abs().max()) * float(y[t, h].abs().sum())


def test_side_stream_and_graph():
    import magi_b200 as mb
    freq, _ = mb.rotary_frequencies(128)
    x = torch.randn(40, 6, 128, device="cuda").to(torch.bfloat16)
    pos = torch.arange(40, dtype=torch.int32, device="cuda")
    want = mb.rotary(x, pos, freq)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    got = mb.rotary(x, pos, freq, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = mb.rotary(x, pos, freq)
    pos += 1
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, mb.rotary(x, pos, freq))


def test_refusals():
    import magi_b200 as mb
    freq, _ = mb.rotary_frequencies(64)
    x, pos = torch.zeros(4, 2, 128, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    for bad in (lambda: mb.rotary(x.double(), pos, freq), lambda: mb.rotary(x.cpu(), pos, freq), lambda: mb.rotary(x[0], pos, freq),
                lambda: mb.rotary(x, pos[:3], freq), lambda: mb.rotary(x, pos.float(), freq), lambda: mb.rotary(x, pos.cpu(), freq),
                lambda: mb.rotary(x, pos, freq.float()), lambda: mb.rotary(x, pos, freq, layout="neox"), lambda: mb.rotary(x[..., :60], pos, freq),
                lambda: mb.rotary(x[..., ::2], pos, freq), lambda: mb.rotary(x, pos, freq, out=x.half()), lambda: mb.rotary(x, pos, freq, out=x[:3]),
                lambda: mb.rotary(x[:, :1].expand(4, 2, 128), pos, freq, out=x[:, :1].contiguous().expand(4, 2, 128)),
                lambda: mb.rotary(torch.zeros(3, 2, 128, device="cuda"), pos[:3], freq, out=torch.zeros(3, 2, 128, device="cuda").transpose(0, 1))):
        with pytest.raises(ValueError):
            bad()
    assert mb.rotary(x[:0], pos[:0], freq).shape == (0, 2, 128)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,H,D,rot", [(3, 57, 72, 24), (501, 7, 40, 40), (37, 113, 96, 64), (2003, 3, 10, 6), (5000, 1, 2, 2), (1, 300, 136, 128),
                                       (90, 11, 264, 16), (300, 5, 3, 2), (11, 2, 4096, 4096), (700, 1, 17, 0)])
def test_walks_over_odd_shapes(layout, T, H, D, rot):
    """Several batches per thread, steps that carry from pieces to heads to tokens, and x itself as the result."""
    import magi_b200 as mb
    pos = torch.arange(T, device="cuda", dtype=torch.int32) * 3
    freq = mb.rotary_frequencies(rot)[0] if rot else torch.empty(0, dtype=torch.float64, device="cuda")
    for dtype in HALF_STEP:
        x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(D)).to(dtype).cuda()
        want = check(x, pos, freq, layout, 0.9)
        assert mb.rotary(x, pos, freq, layout=layout, mscale=0.9, out=x) is x and torch.equal(x, want)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_results_that_share_memory_with_x(layout):
    """out may be x itself, or lie apart from it, between x's own heads too; any other view of its memory is refused."""
    import magi_b200 as mb
    freq, _ = mb.rotary_frequencies(64)
    pos = torch.arange(20, device="cuda")
    packed = torch.randn(21, 6, 200, device="cuda").to(torch.bfloat16)
    x = packed[:20, :2, :80]
    want = mb.rotary(x, pos, freq, layout=layout)
    for apart in (packed[:20, 2:4, :80], packed[:20, :2, 80:160], packed[:20, 4:, 100:180]):
        keep, rest = packed.clone(), packed.clone()
        assert torch.equal(mb.rotary(x, pos, freq, layout=layout, out=apart), want)
        there = apart.storage_offset()
        rest.as_strided(apart.shape, apart.stride(), there).copy_(want)
        assert torch.equal(packed, rest)
        packed.copy_(keep)
    before = packed.clone()
    for bad in (packed[1:, :2, :80], packed[:20, 1:3, :80], packed[:20, :2, 8:88], packed[:20, :2, 79:159], packed[1:, 1:3, 40:120],
                packed.view(-1)[8:].as_strided((20, 2, 80), (160, 80, 1), 8), packed.transpose(0, 1)[:2, :20].as_strided((20, 2, 80), (200, 4200, 1), 200)):
        with pytest.raises(ValueError):
            mb.rotary(x, pos, freq, layout=layout, out=bad)
    assert torch.equal(packed, before)
    one = packed[3:4, :2, :80]   # one token: its stride says nothing
    assert mb.rotary(one, pos[:1], freq, layout=layout, out=one) is one


def test_sizes_beyond_32_bits_do_not_wrap():
    import magi_b200 as mb
    none = torch.empty(0, dtype=torch.float64, device="cuda")
    x = torch.zeros(1, 1, 1, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="32-bit"):
        mb.rotary(x.expand(1, 2 ** 32 + 3, 1), torch.zeros(1, dtype=torch.int32, device="cuda"), none)
    with pytest.raises(ValueError, match="32-bit"):
        mb.rotary(x.expand(2 ** 31, 1, 1), torch.zeros(1, dtype=torch.int32, device="cuda"), none)
